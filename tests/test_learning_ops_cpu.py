"""What the learning operators' entry points refuse: the argument checks come before the context's and need no GPU."""
import ctypes
import math

import numpy as np
import pytest

from go_ai import _hip

P = ctypes.c_void_p
lib = _hip.lib


def err():
    return lib.goai_last_error().decode()


def logprobs(**k):
    a = dict(logits=64, elem=0, stride=82, valid=None, vstride=0, actions=64, t=1.0, top=0, logp=64, ent=64, lse=64, ta=None, tl=None, rows=4, cols=82,
             work=None, bytes=0)
    a.update(k)
    return lib.goai_action_logprobs(None, a["logits"], a["elem"], a["stride"], a["valid"], a["vstride"], a["actions"], a["t"], a["top"], a["logp"],
                                    a["ent"], a["lse"], a["ta"], a["tl"], a["rows"], a["cols"], a["work"], a["bytes"])


@pytest.mark.parametrize("bad,message", [
    (dict(), "ctx is NULL"), (dict(rows=-1), "rows"), (dict(cols=0), "cols"), (dict(cols=(1 << 30) + 1), "cols"), (dict(elem=3), "elem_type"),
    (dict(elem=-1), "elem_type"), (dict(t=0.0), "temperature"), (dict(t=math.nan), "temperature"), (dict(t=math.inf), "temperature"),
    (dict(t=-1.0), "temperature"), (dict(logits=None), "logits"), (dict(logits=66), "aligned"), (dict(logits=65, elem=1), "aligned"),
    (dict(stride=81), "stride"), (dict(stride=-82), "stride"), (dict(valid=64, vstride=5), "stride"), (dict(top=65), "top"), (dict(top=-1), "top"),
    (dict(top=3), "top_actions"), (dict(top=3, ta=64), "top_logp"), (dict(actions=None), "actions"), (dict(rows=0, logits=None), "ctx is NULL"),
    (dict(rows=3, cols=200_000, stride=200_000), "workspace"), (dict(rows=3, cols=200_000, stride=200_000, work=64, bytes=64), "workspace"),
    (dict(rows=3, cols=200_000, stride=200_000, work=72, bytes=1 << 30), "workspace"),
    (dict(rows=3, cols=200_000, stride=200_000, work=64, bytes=1 << 30), "ctx is NULL"),
])
def test_logprobs(bad, message):
    assert logprobs(**bad) == -1 and message in err()


def test_logprobs_workspace():
    f = lib.goai_action_logprobs_workspace
    assert f(5, 82, 64) == 0 and f(0, 1 << 30, 64) == 0 and f(1, 4096, 64) == 0
    for rows in (1, 3, 511, 512, 100_000):
        for cols in (1025, 4097, 70_001, 1 << 30):
            for top in (0, 64):
                need = f(rows, cols, top)
                assert 0 <= need <= rows * 64 * (16 + 8 * top) and (need == 0 or rows < 512)
    assert f(-1, 82, 0) == -1 and f(1, 0, 0) == -1 and f(1, 82, 65) == -1


def grad(**k):
    a = dict(logits=64, elem=0, stride=82, actions=64, t=1.0, lse=64, ent=64, g=64, h=64, d=64, ds=82, rows=4, cols=82)
    a.update(k)
    return lib.goai_action_logprobs_grad(None, a["logits"], a["elem"], a["stride"], None, 0, a["actions"], a["t"], a["lse"], a["ent"], a["g"], a["h"],
                                         a["d"], a["ds"], a["rows"], a["cols"])


@pytest.mark.parametrize("bad,message", [
    (dict(), "ctx is NULL"), (dict(lse=None), "lse"), (dict(d=None), "d_logits"), (dict(actions=None), "actions"), (dict(ent=None), "entropy"),
    (dict(ds=81), "d_stride"), (dict(ds=0), "d_stride"), (dict(d=66), "aligned"), (dict(t=0.0), "temperature"), (dict(logits=None), "logits"),
    (dict(ent=None, h=None), "ctx is NULL"), (dict(actions=None, g=None), "ctx is NULL"),
    # the logits at 1000 (4 rows of 82 float32) and a gradient that is on, beside or between them
    (dict(logits=1000, d=1000), "ctx is NULL"), (dict(logits=1000, d=1004), "overlaps"), (dict(logits=1004, d=1000), "overlaps"),
    (dict(logits=1000, d=1000, ds=83), "overlaps"), (dict(logits=1000, d=1000, stride=0), "overlaps"),
    (dict(logits=1000, d=1000 + 4 * 328), "ctx is NULL"), (dict(logits=1000 + 4 * 328, d=1000), "ctx is NULL"),
    (dict(logits=1000, d=996 + 4 * 328), "overlaps"), (dict(logits=1000, d=1000 + 4 * 82), "overlaps"),
    (dict(logits=1000, d=1000 + 4 * 82, stride=164, ds=164), "ctx is NULL"), (dict(logits=1000 + 4 * 82, d=1000, stride=164, ds=164), "ctx is NULL"),
    (dict(logits=1000, d=996 + 4 * 82, stride=164, ds=164), "overlaps"), (dict(logits=1000, d=1004 + 4 * 82, stride=164, ds=164), "overlaps"),
    (dict(logits=1000, d=1000, rows=1, stride=90), "ctx is NULL"), (dict(logits=1000, d=1004, rows=1), "overlaps"),
])
def test_gradient(bad, message):
    assert grad(**bad) == -1 and message in err()


def init(**k):
    a = dict(n=2, params=[256, 1024], pt=[0, 1], gt=[0, 1], numels=[10, 300], decays=[0.0, 0.1], bits=8, m=64, v=64, ms=64, vs=64)
    a.update(k)
    t = lambda c, x: None if x is None else (c * max(len(x), 1))(*x)  # noqa: E731
    out = P()
    return lib.goai_adamw_init(None, a["n"], t(P, a["params"]), t(ctypes.c_int32, a["pt"]), t(ctypes.c_int32, a["gt"]), t(ctypes.c_int64, a["numels"]),
                               t(ctypes.c_float, a["decays"]), a["bits"], a["m"], a["v"], a["ms"], a["vs"], ctypes.byref(out))


@pytest.mark.parametrize("bad,message", [
    (dict(), "ctx is NULL"), (dict(n=0), "no tensors"), (dict(params=None), "NULL table"), (dict(numels=None), "NULL table"),
    (dict(decays=None), "NULL table"), (dict(pt=None), "NULL table"), (dict(gt=None), "NULL table"), (dict(bits=16), "state_bits"),
    (dict(m=None), "moments"), (dict(v=None), "moments"), (dict(ms=None), "moments"), (dict(m=72), "16-byte"), (dict(pt=[0, 3]), "element type"),
    (dict(gt=[-1, 0]), "element type"), (dict(numels=[-1, 3]), "size"), (dict(decays=[0.0, -1.0]), "decay"), (dict(decays=[math.nan, 0.0]), "decay"),
    (dict(params=[None, 1024]), "NULL parameter"), (dict(params=[258, 1024]), "aligned"), (dict(params=[256, 1025]), "aligned"),
    (dict(params=[1020, 1024]), "overlap"), (dict(params=[256, 256]), "overlap"), (dict(params=[None, 1024], numels=[0, 300]), "ctx is NULL"),
    (dict(bits=32, ms=None, vs=None), "ctx is NULL"), (dict(numels=[1 << 39, 300], params=[1 << 41, 1024]), "too many"),
])
def test_adamw_init(bad, message):
    assert init(**bad) == -1 and message in err()


def test_adamw_state_elems():
    n = (ctypes.c_int64 * 5)(0, 1, 256, 257, 1 << 33)
    assert lib.goai_adamw_state_elems(5, n) == 256 + 256 + 512 + (1 << 33)
    assert lib.goai_adamw_state_elems(0, None) == 0
    assert lib.goai_adamw_state_elems(1, None) == -1
    assert lib.goai_adamw_state_elems(1, (ctypes.c_int64 * 1)(-5)) == -1


def test_adamw_calls():
    table = (P * 1)(64)
    step = lambda t=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, opt=64, g=table, m=0.0, c=None: lib.goai_adamw_step(None, opt, g, t, lr, b1, b2, eps, m, c, None)  # noqa: E731
    for bad, message in ((dict(t=0), "t = 1"), (dict(lr=-1.0), "lr"), (dict(lr=math.nan), "lr"), (dict(lr=math.inf), "lr"), (dict(b1=1.0), "betas"),
                         (dict(b2=-0.1), "betas"), (dict(b2=math.nan), "betas"), (dict(eps=0.0), "eps"), (dict(eps=math.nan), "eps"),
                         (dict(opt=None), "NULL"), (dict(g=None), "NULL"), (dict(m=-1.0), "max_norm"), (dict(m=math.nan), "max_norm"),
                         (dict(m=1.0), "norm_and_coef"), (dict(m=1.0, c=64), "ctx is NULL"), (dict(), "ctx is NULL")):
        assert step(**bad) == -1 and message in err(), bad
    norm = lambda m=1.0, opt=64, g=table, out=64: lib.goai_adamw_grad_norm(None, opt, g, m, out)  # noqa: E731
    for bad, message in ((dict(m=0.0), "max_norm"), (dict(m=-1.0), "max_norm"), (dict(m=math.nan), "max_norm"), (dict(opt=None), "NULL"),
                         (dict(g=None), "NULL"), (dict(out=None), "NULL"), (dict(), "ctx is NULL")):
        assert norm(**bad) == -1 and message in err(), bad
    assert lib.goai_adamw_load_moments(None, 64, None, 64) == -1 and lib.goai_adamw_moments(None, 64, 64, None) == -1
    assert lib.goai_adamw_destroy(None, None) == 0


def test_adamw_without_a_gpu_is_only_numbers():
    """Host parameters (RLNet.parameters) or none: the optimiser waits for the net it is handed to."""
    import torch
    from go_ai.models import AdamW
    for params in (None, [], [torch.zeros(3), torch.zeros(2, 2)]):
        opt = AdamW(params, lr=0.1, weight_decay=0.0)
        assert opt.params is None and opt.lr == 0.1
        with pytest.raises(RuntimeError, match="no parameters yet"):
            opt.step([])
    for bad in (dict(lr=-1), dict(betas=(0.9, 1.0)), dict(eps=0), dict(state_bits=4), dict(max_norm=-1)):
        with pytest.raises(ValueError):
            AdamW(None, **bad)


@pytest.mark.parametrize("dtype", ["int8", "uint8", "int16", "uint16", "int32", "uint32", "int64", "uint64", "float32", "bool", "complex64"])
def test_action_types(dtype):
    """Actions of every integer type mean what they say, or are refused: the largest of a type is not -1 (no action)."""
    import torch
    from go_ai.engine import Context
    c = object.__new__(Context)
    c._h, c.device = None, torch.device("cpu")
    kind = np.dtype(dtype)
    if kind.kind not in "iu" or dtype == "uint64":
        with pytest.raises(ValueError, match="actions"):
            c._per_row(np.zeros(2, kind), 2, torch.int32, "actions")
        return
    least, most = np.iinfo(kind).min, np.iinfo(kind).max
    got = c._per_row(np.array([least, 5, most], kind), 3, torch.int32, "actions").tolist()
    assert got == [max(least, -1) if kind.itemsize == 8 else least, 5, min(most, 0x7fffffff)]


def test_adamw_takes_no_host_tensors():
    from types import SimpleNamespace

    import torch
    from go_ai.models import AdamW
    with pytest.raises(ValueError, match="of one GPU"):
        AdamW().bind([torch.zeros(300)])
    with pytest.raises(ValueError, match="context"):
        AdamW().bind([torch.zeros(300)], SimpleNamespace(device=torch.device("cuda", 0)))


def test_adamw_copies():
    import copy
    import pickle
    from go_ai.models import AdamW
    opt = AdamW(None, lr=0.25, max_norm=2.0)
    for c in (copy.copy(opt), copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert c.lr == 0.25 and c.max_norm == 2.0 and c.params is None
