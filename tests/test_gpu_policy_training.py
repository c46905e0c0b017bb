"""The learning operators together, as a training run uses them: the actor's logits, their log probabilities, the loss's gradient, the
backward pass and the AdamW step (ActorCriticNet.policy_step), AdamW in the reference's train_step / optimize, and the log
probabilities of played moves (ActorCriticNet.move_logprobs).  Against float64 autograd on the oracle's networks."""
import warnings

import numpy as np
import pytest
import torch

from helpers import random_positions
from oracle import nn_ref, nn_train_ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LOOSE = 1e-2        # of a gradient tensor's rms: one flipped ReLU mask moves a channel's gradients by about 1e-3 (tests/test_gpu_train.py)


def net_of(size, layers, seed=3, **kw):
    from go_ai.models.ac_net import ActorCriticNet
    net = ActorCriticNet(size, n_blocks=layers, max_batch=64, **kw)
    sd = nn_ref.make_state_dict("ac", size, seed, layers=layers)
    net.load_state_dict(sd)
    return net, {k: v.clone() for k, v in sd.items()}


def adamw64(p, g, m, v, t, lr, decay, b1=0.9, b2=0.999, eps=1e-8):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    upd = lr / (1 - b1 ** t) * m / (np.sqrt(v / (1 - b2 ** t)) + eps)
    return p * (1 - lr * decay) - upd, m, v, 24 * U * lr / (1 - b1 ** t) * (np.abs(m) + 3 * (1 - b1) * np.abs(g)) / (np.sqrt(v / (1 - b2 ** t)) + eps) + 4 * U * np.abs(p)


@pytest.mark.parametrize("size,layers,n,temperature", [(5, 0, 2, 1.0), (5, 1, 7, 0.8), (9, 1, 12, 1.0), (13, 2, 5, 1.5), (19, 1, 3, 1.0)])
def test_policy_step_against_autograd(size, layers, n, temperature):
    from go_ai.models import AdamW
    net, sd = net_of(size, layers)
    rng = np.random.default_rng(size + n)
    states = random_positions(size, n, seed=size, canonical=True, pass_prob=0.05)
    valid = np.concatenate([1 - states[:, 3].reshape(n, -1), np.ones((n, 1), states.dtype)], axis=1).astype(bool)
    actions = np.array([rng.choice(np.flatnonzero(v)) for v in valid])
    if n > 3:
        actions[1] = -1
    adv = rng.standard_normal(n)
    weight = 0.05
    opt = AdamW(None, lr=1e-2, weight_decay=0.1)
    got = net.policy_step(opt, states, actions, adv, entropy_weight=weight, temperature=temperature)

    d = {k: v.double() for k, v in sd.items()}
    keys = nn_train_ref.param_keys(d)
    for k in keys:
        d[k].requires_grad_(True)
    logits = nn_train_ref._actor_logits(d, torch.as_tensor(states).double())
    lp = torch.log_softmax((logits / temperature).masked_fill(~torch.from_numpy(valid), -np.inf), 1)
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, 0.0).nan_to_num(0.0).sum(1)
    act = torch.from_numpy(actions)
    logp = torch.where(act < 0, 0.0, lp.gather(1, act.clamp(min=0)[:, None])[:, 0])
    loss = -(torch.from_numpy(adv).float().double() * logp).mean() - weight * H.mean()
    # (autograd through p log p at p = 0 is NaN: the entropy's gradient by its own formula)
    g_logits = torch.autograd.grad(-(torch.from_numpy(adv).float().double() * logp).mean(), logits, retain_graph=True)[0]
    g_logits = g_logits + weight / n / temperature * torch.where(p > 0, p * (torch.where(p > 0, lp, 0.0) + H[:, None]), 0.0).detach()
    logits.backward(g_logits)
    assert abs(got[0] - loss.item()) < 1e-4 * (1 + abs(loss.item()))
    assert abs(got[1] - logp.mean().item()) < 1e-4 * (1 + abs(logp.mean().item())) and abs(got[2] - H.mean().item()) < 1e-4 * (1 + H.mean().item())
    grads = net._train.train_export({k: tuple(sd[k].shape) for k in keys}, net._train.TRAIN_GRADS)
    top = max(float(d[k].grad.square().mean().sqrt()) for k in keys if d[k].grad is not None)
    for k in keys:
        w = d[k].grad.numpy() if d[k].grad is not None else np.zeros(tuple(sd[k].shape))
        rms = max(np.sqrt(np.mean(w ** 2)), 1e-4 * top)               # (a convolution's bias in front of BatchNorm has no gradient but noise)
        assert np.sqrt(np.mean((grads[k] - w) ** 2)) <= LOOSE * rms, (k, np.abs(grads[k] - w).max(), rms)
    # the step on the GPU's own gradients; the critic's head has none and stays as it is
    after = net.state_dict()
    for k in keys:
        p0 = sd[k].double().numpy()
        if k.startswith("crit_head."):
            assert np.array_equal(after[k].numpy(), sd[k].numpy())
            continue
        want, _, _, tol = adamw64(p0, grads[k].astype(np.float64), 0.0, 0.0, 1, 1e-2, float(np.float32(0.1)))
        assert (np.abs(after[k].numpy() - want) <= tol).all(), k
    # the inference side sees the new weights
    logits_now = net.ctx.nn_forward(states)[0].cpu().numpy()
    want_now = nn_ref.forward(after, torch.as_tensor(states).float(), "ac")[0].detach().numpy()
    assert np.abs(logits_now - want_now).max() < 1e-3 * max(1.0, np.abs(want_now).max())


@pytest.mark.parametrize("kind", ["ac", "val"])
@pytest.mark.parametrize("bits", [32, 8])
def test_train_step_with_adamw(kind, bits):
    """train_step with an AdamW: goai_train_step's losses and gradients, bit for bit, then AdamW's update of them."""
    from go_ai.models import Adam, AdamW
    from go_ai.models.ac_net import ActorCriticNet
    from go_ai.models.val_net import ValueNet
    size, n, layers = 5, 6, 1
    rng = np.random.default_rng(1)
    A = size * size + 1
    nets = [(ActorCriticNet if kind == "ac" else ValueNet)(size, n_blocks=layers, max_batch=16) for _ in range(2)]
    sd = nn_ref.make_state_dict(kind, size, 5, layers=layers)
    for net in nets:
        net.load_state_dict(sd)
    keys = nn_train_ref.param_keys(sd)
    shapes = {k: tuple(sd[k].shape) for k in keys}
    opt = AdamW(nets[0].parameters(), lr=1e-2, weight_decay=0.05, state_bits=bits, max_norm=0.5)
    m = {k: 0.0 for k in keys}
    v = {k: 0.0 for k in keys}
    for t in (1, 2):
        batch = ((rng.random((n, 6, size, size)) < 0.3).astype(np.uint8), rng.integers(0, A, n), np.zeros(n),
                 (rng.random((n, A, 6, size, size)) < 0.3).astype(np.uint8), np.zeros(n), rng.integers(-1, 2, n).astype(np.float32),
                 rng.random((n, A)).astype(np.float32))
        before = {k: x.double().numpy() for k, x in nets[0].state_dict().items()}
        results = []
        for net, o in zip(nets, (opt, Adam(lr=0.0, weight_decay=0.0))):
            np.random.seed(7)                                            # the symmetries that train_step draws
            results.append(net.train_step(o, *batch))
        assert results[0] == results[1]
        grads = [net._train.train_export(shapes, net._train.TRAIN_GRADS) for net in nets]
        assert all(np.array_equal(grads[0][k], grads[1][k]) for k in keys)
        norm = np.sqrt(sum((grads[0][k].astype(np.float64) ** 2).sum() for k in keys))
        assert abs(float(opt.norm) - norm) <= 4 * U * norm
        after = nets[0].state_dict()
        for k in keys:
            g = grads[0][k].astype(np.float64) * min(1.0, 0.5 / norm)
            want, m1, v1, tol = adamw64(before[k], g, m[k], v[k], t, 1e-2, float(np.float32(0.05)))
            assert (np.abs(after[k].numpy() - want) <= tol).all(), (t, k)
        moments = opt.moments()
        for k, a, b in zip(opt._net_names, opt._split(moments[0]), opt._split(moments[1])):
            m[k], v[k] = a.double().cpu().numpy(), b.double().cpu().numpy()
        nets[1].load_state_dict(after)                                   # (lr = 0 moved nothing; the statistics moved alike)
    assert opt.steps == 2


def test_optimize_with_adamw_and_a_larger_batch():
    """The reference's optimize() with an AdamW; a batch beyond the training buffers rebuilds them, and the moments start again."""
    from go_ai.data import SoloComm
    from go_ai.models import AdamW
    net, _ = net_of(5, 1, train_batch=8)
    rng = np.random.default_rng(2)

    def batch(n):
        return ((rng.random((n, 6, 5, 5)) < 0.3).astype(np.uint8), rng.integers(0, 26, n), np.zeros(n),
                (rng.random((n, 26, 6, 5, 5)) < 0.3).astype(np.uint8), np.zeros(n), rng.integers(-1, 2, n).astype(np.float32),
                rng.random((n, 26)).astype(np.float32))
    opt = AdamW(net.parameters(), lr=1e-3, state_bits=8, max_norm=1.0)
    before = {k: v.clone() for k, v in net.state_dict().items()}
    metrics = net.optimize(SoloComm(), [batch(4), batch(8)], opt)
    assert np.isfinite([metrics.crit_loss, metrics.act_loss]).all() and opt.steps == 2
    after = net.state_dict()
    assert any(not torch.equal(before[k], after[k]) for k in before)
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        net.optimize(SoloComm(), [batch(11)], opt)
    assert any("AdamW's moments were reset" in str(w.message) for w in seen) and opt.steps == 1
    other, _ = net_of(5, 1)
    with pytest.raises(ValueError, match="belongs"):
        other.train_step(opt, *batch(4))
    with pytest.raises(ValueError, match="AdamW"):
        net.policy_step(object(), np.zeros((2, 6, 5, 5), np.uint8), [0, 1], [1.0, 1.0])
    opt2 = AdamW()
    for bad in (dict(actions=[0], advantages=[1.0, 1.0]), dict(actions=[0, 1], advantages=[1.0])):
        with pytest.raises(ValueError):
            net.policy_step(opt2, np.zeros((2, 6, 5, 5), np.uint8), **bad)
    with pytest.raises(ValueError, match="at least 2"):
        net.policy_step(opt2, np.zeros((1, 6, 5, 5), np.uint8), [0], [1.0])


def test_backward_leaves_parameters_and_adam_alone():
    from go_ai.engine import Context
    size, n = 5, 4
    rng = np.random.default_rng(0)
    sd = nn_ref.make_state_dict("ac", size, 1, layers=1)
    shapes = {k: tuple(sd[k].shape) for k in nn_train_ref.param_keys(sd)}
    batch = ((rng.random((n, 6, size, size)) < 0.3).astype(np.uint8), (rng.random((n, 6, size, size)) < 0.3).astype(np.uint8),
             rng.integers(-1, 2, n).astype(np.float32), rng.random((n, 26)).astype(np.float32))
    a, b = Context(size), Context(size)
    for c in (a, b):
        c.train_init(Context.NET_AC, 1, 8)
        c.train_load(sd)
    first = a.train_backward(*batch)
    again = a.train_backward(*batch)                     # replayed; the batch statistics do not depend on the running ones
    assert first == again
    g = a.train_export(shapes, a.TRAIN_GRADS)
    assert all(np.array_equal(a.train_export(shapes)[k], sd[k].numpy()) for k in shapes)
    assert all((a.train_export(shapes, what)[k] == 0).all() for what in (a.TRAIN_ADAM_M, a.TRAIN_ADAM_V) for k in shapes)
    assert b.train_step(*batch) == first
    gb = b.train_export(shapes, b.TRAIN_GRADS)
    assert all(np.array_equal(g[k], gb[k]) for k in shapes)
    # and a step behind it is the first step
    assert a.train_step(*batch) == first
    pa, pb = a.train_export(shapes), b.train_export(shapes)
    assert all(np.array_equal(pa[k], pb[k]) for k in shapes)
    flat = a.train_grads().cpu().numpy()
    for k in shapes:
        off, numel = a.train_parameter(k)
        assert np.array_equal(flat[off:off + numel], g[k].reshape(-1))


def test_call_sequence():
    from go_ai import _hip
    from go_ai.engine import Context
    c = Context(5)
    st = np.zeros((3, 6, 5, 5), np.uint8)
    with pytest.raises(_hip.GoaiError, match="train_init"):
        c.train_actor_forward(st)
    with pytest.raises(_hip.GoaiError, match="train_init"):
        c.train_grads()
    c.train_init(Context.NET_AC, 1, 8)
    c.train_load(nn_ref.make_state_dict("ac", 5, 1, layers=1))
    with pytest.raises(_hip.GoaiError, match="must follow"):
        c.train_actor_backward(torch.zeros(3, 26).cuda())
    for n in (1, 9):
        with pytest.raises(_hip.GoaiError, match="batch size"):
            c.train_actor_forward(np.zeros((n, 6, 5, 5), np.uint8))
    logits = c.train_actor_forward(st)
    assert logits.shape == (3, 26)
    with pytest.raises(_hip.GoaiError, match="must follow"):
        c.train_actor_backward(torch.zeros(2, 26).cuda())
    c.train_actor_backward(torch.zeros(3, 26).cuda())
    assert not c.train_grads().any()
    with pytest.raises(_hip.GoaiError, match="must follow"):
        c.train_actor_backward(torch.zeros(3, 26).cuda())
    c.train_actor_forward(st)
    c.train_backward(st, st, np.zeros(3, np.float32), np.ones((3, 26), np.float32))
    with pytest.raises(_hip.GoaiError, match="must follow"):
        c.train_actor_backward(torch.zeros(3, 26).cuda())
    for name in ("main.1.running_mean", "nothing"):
        with pytest.raises(_hip.GoaiError, match="no parameter"):
            c.train_parameter(name)
    v = Context(5)
    v.train_init(Context.NET_VAL, 1, 8)
    with pytest.raises(_hip.GoaiError, match="no policy head"):
        v.train_actor_forward(st)


@pytest.mark.parametrize("size", [5, 9, 13, 19])
def test_move_logprobs(size):
    net, sd = net_of(size, 1)
    n = 7
    states = random_positions(size, n, seed=3, canonical=True, pass_prob=0.05)
    valid = np.concatenate([1 - states[:, 3].reshape(n, -1), np.ones((n, 1), states.dtype)], axis=1).astype(bool)
    actions = np.array([int(np.flatnonzero(v)[-1]) for v in valid])
    r = net.move_logprobs(states, actions, top=5, temperature=0.7)
    logits = net.ctx.nn_forward(states)[0].double().cpu().numpy()
    s = np.where(valid, logits / 0.7, -np.inf)
    lp = s - s.max(1, keepdims=True)
    lp = lp - np.log(np.exp(lp).sum(1, keepdims=True))
    tol = U * (16 * np.abs(logits).max() / 0.7 + 64)
    assert np.abs(r.logp.cpu().numpy() - lp[np.arange(n), actions]).max() <= tol
    order = np.argsort(-np.where(valid, logits, -np.inf), axis=1, kind="stable")[:, :5]
    best = np.take_along_axis(lp, order, 1)
    there = np.isfinite(best)
    assert np.array_equal(r.top_actions.cpu().numpy(), np.where(there, order, -1))
    assert np.abs(r.top_logp.cpu().numpy()[there] - best[there]).max() <= tol
    assert net.move_logprobs(states).logp is None


def test_loaded_parameters_end_an_actor_pass():
    from go_ai import _hip
    from go_ai.engine import Context
    c = Context(5)
    c.train_init(Context.NET_AC, 1, 8)
    sd = nn_ref.make_state_dict("ac", 5, 1, layers=1)
    c.train_load(sd)
    c.train_actor_forward(np.zeros((3, 6, 5, 5), np.uint8))
    c.train_load(sd)
    with pytest.raises(_hip.GoaiError, match="must follow"):
        c.train_actor_backward(torch.zeros(3, 26).cuda())


def test_policy_step_checks_its_actions():
    from go_ai.models import AdamW
    net, _ = net_of(5, 1)
    opt, st = AdamW(), np.zeros((2, 6, 5, 5), np.uint8)
    before = {k: v.clone() for k, v in net.state_dict().items()}
    for actions in ([0, 26], [0, 1 << 32], [0.0, 1.0], [True, False], torch.tensor([0, 26]).cuda(), torch.tensor([0.5, 1.0]).cuda()):
        with pytest.raises(ValueError, match="actions"):
            net.policy_step(opt, st, actions, [1.0, 1.0])
    assert opt.params is None and all(torch.equal(before[k], v) for k, v in net.state_dict().items())
    loss, _, _ = net.policy_step(opt, st, torch.tensor([-1, 25], dtype=torch.int8), [1.0, 1.0])
    assert np.isfinite(loss) and opt.steps == 1


def test_an_optimiser_bound_elsewhere_is_not_a_nets():
    """Bound by hand to other tensors, with the net's own context even, it has none of the net's gradients."""
    from go_ai.models import AdamW
    net, _ = net_of(5, 1)
    st = np.zeros((2, 6, 5, 5), np.uint8)
    opt = AdamW()
    net.policy_step(opt, st, [0, 1], [1.0, 1.0])
    for ctx in (net._train, None):
        opt.bind([torch.zeros(10).cuda()], ctx)
        with pytest.raises(ValueError, match="belongs"):
            net.policy_step(opt, st, [0, 1], [1.0, 1.0])
