"""AdamW across interruptions: a net's optimiser resumed from its state_dict, moments kept when the training buffers grow, a bind() that
is refused."""
import io
import pickle
import warnings

import numpy as np
import pytest
import torch

from oracle import nn_ref

pytestmark = pytest.mark.gpu
SIZE = 5


def net_of(kind, sd, train_batch=8):
    from go_ai.models.ac_net import ActorCriticNet
    from go_ai.models.val_net import ValueNet
    net = (ActorCriticNet if kind == "ac" else ValueNet)(SIZE, n_blocks=1, max_batch=64, train_batch=train_batch)
    net.load_state_dict(sd)
    return net


def batch(n, seed):
    rng = np.random.default_rng(seed)
    return ((rng.random((n, 6, SIZE, SIZE)) < 0.3).astype(np.uint8), rng.integers(0, 26, n), np.zeros(n),
            (rng.random((n, 26, 6, SIZE, SIZE)) < 0.3).astype(np.uint8), np.zeros(n), rng.integers(-1, 2, n).astype(np.float32),
            rng.random((n, 26)).astype(np.float32))


def train(net, opt, seeds, n=6):
    for s in seeds:
        np.random.seed(s)                                    # the symmetries that train_step draws
        net.train_step(opt, *batch(n, s))


def through_a_file(x):
    f = io.BytesIO()
    torch.save(x, f)
    f.seek(0)
    return torch.load(f, weights_only=True)


def state_of(net, opt):
    m, v = opt.moments()
    names = opt._net_names
    return ({k: x.clone() for k, x in net.state_dict().items()}, dict(zip(names, [x.cpu().clone() for x in opt._split(m)])),
            dict(zip(names, [x.cpu().clone() for x in opt._split(v)])))


def equal(a, b):
    for x, y in zip(a, b):
        assert x.keys() == y.keys()
        assert all(torch.equal(x[k], y[k]) for k in x), [k for k in x if not torch.equal(x[k], y[k])]


@pytest.mark.parametrize("kind", ["ac", "val"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("turned", [False, True])
def test_resumed_run(kind, bits, turned):
    """Saved after three steps and resumed by another net and optimiser (its tensors in another order, too): the uninterrupted run's bits."""
    from go_ai.models import AdamW
    sd = nn_ref.make_state_dict(kind, SIZE, 5, layers=1)
    args = dict(lr=1e-2, weight_decay=0.05, state_bits=bits)
    net, opt = net_of(kind, sd), AdamW(**args)
    train(net, opt, (1, 2, 3))
    saved, weights = through_a_file(opt.state_dict()), through_a_file(net.state_dict())
    assert saved["steps"] == 3
    train(net, opt, (4, 5))
    net2 = net_of(kind, dict(reversed(weights.items())) if turned else weights)
    opt2 = AdamW(net2.parameters(), **args)
    opt2.load_state_dict(saved)
    assert opt2.steps == 3 and opt2.params is None
    train(net2, opt2, (4, 5))
    assert opt2.steps == opt.steps == 5
    equal(state_of(net2, opt2), state_of(net, opt))
    # and into an optimiser that the net has already
    opt2.load_state_dict(saved)
    assert opt2.steps == 3
    m = dict(zip(opt2._net_names, opt2._split(opt2.moments()[0])))
    for k, want in zip(saved["names"], saved["exp_avg"]):
        assert torch.equal(m[k].cpu(), want), k


@pytest.mark.parametrize("bits", [32, 8])
def test_resumed_policy_steps(bits):
    from go_ai.models import AdamW
    sd = nn_ref.make_state_dict("ac", SIZE, 5, layers=1)
    st = np.zeros((4, 6, SIZE, SIZE), np.uint8)
    st[1, 0, 2, 2] = st[1, 3, 2, 2] = 1
    step = lambda net, opt: net.policy_step(opt, st, [1, 2, 25, -1], [1.0, -0.5, 0.25, 0.0])  # noqa: E731
    net, opt = net_of("ac", sd), AdamW(lr=1e-2, state_bits=bits)
    for _ in range(2):
        step(net, opt)
    saved, weights = pickle.loads(pickle.dumps(opt.state_dict())), net.state_dict()
    net2, opt2 = net_of("ac", weights), AdamW(lr=1e-2, state_bits=bits)
    opt2.load_state_dict(saved)
    for n, o in ((net, opt), (net2, opt2)):
        step(n, o)
    assert opt.steps == opt2.steps == 3
    equal(state_of(net2, opt2), state_of(net, opt))


def test_a_state_of_the_other_bits():
    """32-bit moments for an 8-bit optimiser, rounded to their nearest codes, and back: the values that the codes stand for."""
    from go_ai.models import AdamW
    g = torch.Generator().manual_seed(1)
    p = [torch.randn(300, generator=g).cuda(), torch.randn(4, 5, generator=g).cuda()]
    full, short, again = AdamW(p, state_bits=32), AdamW(p, state_bits=8), AdamW(p, state_bits=32)
    full.step([torch.randn(x.shape, generator=g).cuda() for x in p])
    short.load_state_dict(full.state_dict())
    again.load_state_dict(short.state_dict())
    assert short.steps == again.steps == 1
    for name, most in (("exp_avg", 2.0 ** -4), ("exp_avg_sq", 2.0 ** -4 * (1 + 2.0 ** -6))):     # (1 + 2^-5)^2 of a root's half step
        for a, b, c in zip(*[o.state_dict()[name] for o in (full, short, again)]):
            assert torch.equal(b, c)
            off = (b.double() - a.double()).abs() - most * (1 + 1e-5) * a.double().abs()
            assert float(off.max()) <= 1.2 * 2.0 ** -16 * float(a.abs().max())                   # (smallest codes: 2^-9 / 448, 1.125 2^-16)


def test_a_state_that_waits():
    """For parameters given later: kept over copies, given out again, checked when they come, and used once."""
    from go_ai.models import AdamW
    g = torch.Generator().manual_seed(1)
    p = [torch.randn(300, generator=g).cuda(), torch.randn(4, 5, generator=g).cuda()]
    grads = [torch.randn(x.shape, generator=g).cuda() for x in p]
    q = [x.clone() for x in p]
    opt = AdamW(p)
    opt.step(grads)
    saved = opt.state_dict()
    for x, y in zip(q, p):
        x.copy_(y)
    late = AdamW()
    late.load_state_dict(saved)
    late = pickle.loads(pickle.dumps(late))
    assert late.steps == 1 and late.state_dict()["steps"] == 1 and torch.equal(late.state_dict()["exp_avg"][0], saved["exp_avg"][0])
    with pytest.raises(ValueError, match="loaded state"):
        late.bind([q[0]])
    with pytest.raises(ValueError, match="loaded state"):
        late.bind([q[0], q[1].view(5, 4)])
    assert late.params is None and late.steps == 1
    late.bind(q)
    for o in (opt, late):
        o.step(grads)
    assert late.steps == 2 and all(torch.equal(a, b) for a, b in zip(p + list(opt.moments()), q + list(late.moments())))
    late.bind(q)
    assert late.steps == 0 and not any(x.any() for x in late.moments())
    with pytest.raises(ValueError, match="steps"):
        AdamW().load_state_dict({**saved, "steps": -1})


def test_a_state_of_another_net_is_refused_first():
    from go_ai.models import AdamW
    sd = nn_ref.make_state_dict("ac", SIZE, 5, layers=1)
    net, opt, other = net_of("ac", sd), AdamW(), AdamW()
    train(net, opt, (1,))
    other.load_state_dict(opt.state_dict())
    val = net_of("val", nn_ref.make_state_dict("val", SIZE, 5, layers=1), train_batch=4)
    before = {k: x.clone() for k, x in val.state_dict().items()}
    with pytest.raises(ValueError, match="another net"):
        train(val, other, (1,))
    state = {k: v for k, v in opt.state_dict().items() if k != "names"}
    other.load_state_dict({**state, "exp_avg": state["exp_avg"][:-1]})
    with pytest.raises(ValueError, match="loaded state"):
        train(net, other, (2,))
    assert val.train_batch == 4 and all(torch.equal(before[k], v) for k, v in val.state_dict().items())


@pytest.mark.parametrize("bits", [32, 8])
def test_reserved_training_buffers_keep_the_moments(bits):
    """The run whose buffers are rebuilt on the way, and the one that had them from the start."""
    from go_ai.models import AdamW
    sd = nn_ref.make_state_dict("ac", SIZE, 5, layers=1)
    nets = [net_of("ac", sd, train_batch=b) for b in (6, 11)]
    opts = [AdamW(lr=1e-2, state_bits=bits, max_norm=1.0) for _ in nets]
    for net, opt in zip(nets, opts):
        train(net, opt, (1, 2, 3))
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        nets[0].reserve_train_batch(11, opts[0])
        assert nets[0].train_batch == 11 and opts[0].steps == 3
        assert all(torch.equal(a, b) for a, b in zip(opts[0].moments(), opts[1].moments()))
        nets[0].reserve_train_batch(5, opts[0])
        for net, opt in zip(nets, opts):
            train(net, opt, (4, 5), n=11)
    assert not any("AdamW" in str(w.message) for w in seen)
    equal(state_of(nets[0], opts[0]), state_of(nets[1], opts[1]))
    assert opts[0].steps == opts[1].steps == 5
    # buffers that a step itself has to rebuild: the moments start again, and it says so
    with pytest.warns(RuntimeWarning, match="reserve_train_batch"):
        train(nets[0], opts[0], (6,), n=12)
    assert opts[0].steps == 1
    fresh = net_of("ac", sd, train_batch=4)
    fresh.reserve_train_batch(9, AdamW())
    assert fresh.train_batch == 9
    with pytest.raises(ValueError, match="belongs"):
        fresh.reserve_train_batch(20, opts[0])
    assert fresh.train_batch == 9


def test_a_refused_bind_leaves_the_optimiser_as_it_was():
    from go_ai._hip import GoaiError
    from go_ai.models import AdamW
    net, opt = net_of("ac", nn_ref.make_state_dict("ac", SIZE, 5, layers=1)), AdamW()
    train(net, opt, (1,))
    before = [x.clone() for x in opt.moments()]
    x = torch.zeros(100).cuda()
    with pytest.raises(GoaiError, match="overlap"):
        opt.bind([x[:60], x[40:]])
    with pytest.raises(ValueError):
        opt.bind([x.cpu()])
    assert opt.steps == 1 and all(torch.equal(a, b) for a, b in zip(before, opt.moments()))
    train(net, opt, (2,))
    assert opt.steps == 2


def test_a_state_that_was_changed():
    """Values that were edited after they were saved are loaded, not the codes that were saved beside them."""
    from go_ai.models import AdamW
    g = torch.Generator().manual_seed(1)
    p = [torch.randn(700, generator=g).cuda(), torch.randn(4, 5, generator=g).cuda()]
    opt = AdamW(p, state_bits=8)
    for _ in range(3):
        opt.step([torch.randn(x.shape, generator=g).cuda() for x in p])
    saved = opt.state_dict()
    codes = [x.clone() for x in (opt._m, opt._v, opt._scales)]
    opt.step([torch.ones_like(x) for x in p])
    opt.load_state_dict(saved)
    assert all(torch.equal(a, b) for a, b in zip(codes, (opt._m, opt._v, opt._scales)))
    for name, other in (("exp_avg", "exp_avg_sq"), ("exp_avg_sq", "exp_avg")):
        state = opt.state_dict()
        state[name] = [state[name][0], torch.zeros(4, 5)]
        opt.load_state_dict(state)
        got = opt.state_dict()
        assert not got[name][1].any() and got[name][0].any() and got[other][1].any()
        opt.load_state_dict(saved)


def test_an_optimiser_that_was_closed():
    """A net takes its closed AdamW as one without moments, and says so."""
    from go_ai.models import Adam, AdamW
    net, opt = net_of("ac", nn_ref.make_state_dict("ac", SIZE, 5, layers=1)), AdamW()
    train(net, opt, (1, 2))
    opt.close()
    with pytest.warns(RuntimeWarning, match="reset"):
        train(net, opt, (3,))
    assert opt.steps == 1
    opt.close()
    net.reserve_train_batch(20, opt)
    net.reserve_train_batch(21, Adam())
    assert net.train_batch == 21
