"""AdamW with max_norm: steps whose gradients' norm is not finite leave no trace, neither in the moments nor in the step's number that
corrects their bias, eager or captured."""
import ctypes
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(300,), (7, 1000), (1,)]
U = 2.0 ** -24


def tensors(seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).cuda() for s in SHAPES]


def spoil(grads, bad):
    out = [g.clone() for g in grads]
    out[1][3, 17] = bad
    return out


def same(a, b):
    torch.cuda.synchronize()
    return all(torch.equal(x, y) for x, y in zip(a, b))


# 22 good steps: 8-bit moments are rounded to the nearest for 16, then at random
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad_at", [{0: 10}, {3: 1, 19: 2}, {0: 1, 1: 1, 21: 3}])
def test_good_steps_alone(bits, bad_at):
    from go_ai.models import AdamW
    runs = []
    for with_bad in (False, True):
        p = tensors(1)
        opt = AdamW(p, lr=1e-2, state_bits=bits, max_norm=1.0)
        for k in range(22):
            if with_bad:
                for j in range(bad_at.get(k, 0)):
                    opt.step(spoil(tensors(50), (math.nan, math.inf, -math.inf)[j % 3]))
                    assert not math.isfinite(float(opt.norm))
            opt.step(tensors(100 + k))
        assert opt.steps == 22 and opt.state_dict()["steps"] == 22
        runs.append(p + list(opt.moments()))
    assert same(*runs)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_first_good_step_is_the_first_step(bits):
    """The size of the update behind ten skipped steps: lr / (1 + eps / |g|) for every element, as the first step's is."""
    from go_ai.models import AdamW
    p = [torch.zeros(5000, device="cuda")]
    opt = AdamW(p, lr=0.5, weight_decay=0.0, state_bits=bits, max_norm=1e9)
    g = torch.randn(5000, device="cuda", generator=torch.Generator("cuda").manual_seed(0)) + 3.0 * torch.tensor([1.0, -1.0], device="cuda").repeat(2500)
    bad = g.clone()
    bad[0] = math.nan
    for _ in range(10):
        opt.step([bad])
    opt.step([g])
    # 14 roundings of the quotient, the coefficients' two
    assert float((p[0].abs() - 0.5).abs().max()) <= 0.5 * (20 * U + 1e-8 / float(g.abs().min()))
    assert opt.steps == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_captured(bits):
    from go_ai.models import AdamW
    p = tensors(1)
    opt = AdamW(p, lr=1e-2, state_bits=bits, max_norm=1.0)
    static = tensors(2)
    opt.advance()
    torch.cuda.synchronize()
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            opt.step(static, captured=True)
    torch.cuda.synchronize()
    q = tensors(1)
    eager = AdamW(q, lr=1e-2, state_bits=bits, max_norm=1.0)
    first = True
    for k in range(22):
        for grads in ([spoil(tensors(50), math.nan)] if k in (0, 5, 18) else []) + [tensors(100 + k)]:
            for a, b in zip(static, grads):
                a.copy_(b)
            if not first:
                opt.advance()
            first = False
            graph.replay()
        eager.step(tensors(100 + k))
        assert same(p + list(opt.moments()), q + list(eager.moments())), k
        assert opt.steps == eager.steps == k + 1
    # eager steps behind the graph's, with and without clipping
    for max_norm in (1.0, 0.0):
        opt.max_norm = eager.max_norm = max_norm
        for o, m in ((opt, p), (eager, q)):
            o.step(tensors(300))
        assert same(p + list(opt.moments()), q + list(eager.moments()))
    assert opt.steps == eager.steps == 24


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_that_ends(bits):
    """Steps without max_norm behind skipped ones: number and rounding follow the applied ones (the correction of the 4th and 5th step
    with float64 powers of the GPU's or the host's: the last bit of a float32 at most)."""
    from go_ai.models import AdamW
    runs = []
    for bad in (0, 3):
        p = tensors(1)
        opt = AdamW(p, lr=1e-2, state_bits=bits, max_norm=1.0)
        for k in range(3):
            opt.step(tensors(100 + k))
            for _ in range(bad):
                opt.step(spoil(tensors(50), math.inf))
        opt.max_norm = 0.0
        for k in range(2):
            opt.step(tensors(200 + k))
        assert opt.steps == 5
        runs.append(p + list(opt.moments()))
    assert same(*runs)


@pytest.mark.parametrize("bits", [32, 8])
def test_loaded_moments_start_a_new_count(bits):
    from go_ai.models import AdamW
    p, q = tensors(1), tensors(1)
    opt, other = [AdamW(x, state_bits=bits, max_norm=1.0) for x in (p, q)]
    for _ in range(4):
        opt.step(spoil(tensors(50), math.nan))
    m, v = tensors(3), [x.square() for x in tensors(4)]
    for o in (opt, other):
        o.load_moments(m, v, 7)
        assert o.steps == 7
        for k in range(18):
            o.step(tensors(100 + k))
        assert o.steps == 25
    assert same(p + list(opt.moments()), q + list(other.moments()))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("t_first", [1, 20000])
def test_a_coefficient_of_the_callers(bits, t_first):
    """goai_adamw_grad_norm, then goai_adamw_step with its coefficient: the same as the step that does both; a NaN skips."""
    from go_ai import _hip
    from go_ai.models import AdamW
    p, q = tensors(1), tensors(1)
    both, apart = [AdamW(x, lr=1e-2, state_bits=bits, max_norm=0.5) for x in (p, q)]
    m, v = tensors(3), [x.square() for x in tensors(4)]
    for o in (both, apart):
        o.load_moments(m, v, t_first - 1)
    out = torch.zeros(2, device="cuda")
    h, ctx = apart._h, apart._ctx._h
    t = t_first
    for k, grads in enumerate([tensors(10), spoil(tensors(11), math.nan), tensors(12), [tensors(13)[0], None, tensors(13)[2]], tensors(14)]):
        both.step(grads)
        table = (ctypes.c_void_p * 3)(*[None if g is None else g.data_ptr() for g in grads])
        _hip.check(_hip.lib.goai_adamw_grad_norm(ctx, h, table, 0.5, out.data_ptr()))
        _hip.check(_hip.lib.goai_adamw_step(ctx, h, table, t, 1e-2, 0.9, 0.999, 1e-8, 0.0, out.data_ptr(), None))
        t += 1
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads if g is not None))
        torch.cuda.synchronize()
        if k == 1:
            assert not math.isfinite(float(out[0])) and math.isnan(float(out[1]))
        else:
            assert abs(float(out[0]) - norm) <= 2 * U * norm and abs(float(out[1]) - min(1.0, 0.5 / norm)) <= 2 * U
        assert same(p + list(both.moments()), q + list(apart.moments())), k
    skipped = ctypes.c_int64()
    _hip.check(_hip.lib.goai_adamw_skipped(ctx, h, ctypes.byref(skipped)))
    assert skipped.value == 1 and both.steps == t_first + 3
    # the norm alone
    _hip.check(_hip.lib.goai_adamw_grad_norm(ctx, h, table, math.inf, out.data_ptr()))
    assert float(out[1]) == 1.0 and abs(float(out[0]) - norm) <= 2 * U * norm
    # a coefficient that the caller made: gradients of half the size
    half = [g * 0.5 for g in tensors(15)]
    both.max_norm = 0.0
    both.step(half)
    out.copy_(torch.tensor([0.0, 0.5]))
    full = tensors(15)
    table = (ctypes.c_void_p * 3)(*[g.data_ptr() for g in full])
    _hip.check(_hip.lib.goai_adamw_step(ctx, h, table, t, 1e-2, 0.9, 0.999, 1e-8, 0.0, out.data_ptr(), None))
    assert same(p + list(both.moments()), q + list(apart.moments()))


def test_scalars():
    """What a captured step reads: float64, less the skipped steps."""
    from go_ai.models import AdamW
    p = tensors(1)
    opt = AdamW(p, lr=3e-3, betas=(0.8, 0.99), max_norm=1.0)
    for grads in (tensors(2), spoil(tensors(3), math.nan), tensors(4)):
        opt.step(grads)
    opt.advance()
    want = [3e-3, 1 / math.sqrt(1 - 0.99 ** 3), 3e-3 / (1 - 0.8 ** 3)]
    assert np.allclose(opt._scalars.cpu().numpy(), want, rtol=1e-14, atol=0) and opt.steps == 3


def test_the_count_outlives_the_context():
    """A net's training buffers are rebuilt under its optimiser: the number of steps can still be read."""
    from go_ai.engine import Context
    from go_ai.models import AdamW
    for bad in (0, 2):
        c = Context(9)
        p = tensors(1)
        opt = AdamW(p, max_norm=1.0, ctx=c)
        for _ in range(3):
            opt.step(tensors(2))
        for _ in range(bad):
            opt.step(spoil(tensors(3), math.nan))
        c.close()
        assert opt.steps == 3
        with pytest.raises(RuntimeError, match="closed"):
            opt.step(tensors(2))
        assert opt.steps == 3
