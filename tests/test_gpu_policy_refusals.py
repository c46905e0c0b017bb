"""What policy_step, train_step and optimize refuse, and that a refused call leaves everything as it was: parameters, BatchNorm statistics, the
optimiser's moments and step number, the training buffers and the moments of the reference's Adam in them."""
import math
import warnings

import numpy as np
import pytest
import torch

from oracle import nn_ref

pytestmark = pytest.mark.gpu
SIZE = 5


def net_of(train_batch=4):
    from go_ai.models.ac_net import ActorCriticNet
    net = ActorCriticNet(SIZE, n_blocks=1, max_batch=64, train_batch=train_batch)
    net.load_state_dict(nn_ref.make_state_dict("ac", SIZE, 3, layers=1))
    return net


def empty(n):
    return np.zeros((n, 6, SIZE, SIZE), np.uint8)


def occupied(n):
    """A black stone on point 7 of the last position, where nobody may play."""
    st = empty(n)
    st[n - 1, 0, 1, 2] = st[n - 1, 3, 1, 2] = 1
    return st


def batch(n, seed=0):
    rng = np.random.default_rng(seed)
    return ((rng.random((n, 6, SIZE, SIZE)) < 0.3).astype(np.uint8), rng.integers(0, 26, n), np.zeros(n),
            (rng.random((n, 26, 6, SIZE, SIZE)) < 0.3).astype(np.uint8), np.zeros(n), rng.integers(-1, 2, n).astype(np.float32),
            rng.random((n, 26)).astype(np.float32))


class Unchanged:
    """The net, its Adam and an AdamW of its own: the same before and behind a refused call."""

    def __init__(self, net, opt):
        self.net, self.opt, self.train, self.capacity = net, opt, net._train, net.train_batch
        self.seen = self.look()

    def look(self):
        net, opt = self.net, self.opt
        shapes = net._tensor_shapes()
        params = {k: s for k, s in shapes.items() if not k.endswith(("running_mean", "running_var"))}
        parts = [net._train.train_export(shapes)] + [net._train.train_export(params, what) for what in (net._train.TRAIN_ADAM_M, net._train.TRAIN_ADAM_V)]
        arrays = [a for p in parts for a in p.values()]
        if opt is not None and opt.params is not None:
            arrays += [m.cpu().numpy().copy() for m in opt.moments()] + [np.array(opt.steps)]
        return arrays

    def check(self):
        assert self.net._train is self.train and self.net.train_batch == self.capacity
        assert all(np.array_equal(a, b) for a, b in zip(self.seen, self.look()))


def trained():
    from go_ai.models import Adam, AdamW
    net, opt = net_of(), AdamW(lr=1e-2)
    net.train_step(Adam(), *batch(4))
    net.policy_step(opt, empty(3), [0, 25, -1], [1.0, -1.0, 0.5])
    return net, opt


# six positions are more than the training buffers hold, and have to be refused before they grow
@pytest.mark.parametrize("n", [3, 6])
@pytest.mark.parametrize("change,message", [
    (dict(states=occupied), "not legal"), (dict(actions=26), "beyond"), (dict(actions=2 ** 31 - 1), "beyond"), (dict(actions=0.5), "actions"),
    (dict(advantages=math.nan), "finite"), (dict(advantages=math.inf), "finite"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=math.nan), "temperature"), (dict(temperature=1e5), "temperature"), (dict(entropy_weight=math.inf), "entropy_weight"),
    (dict(n_actions=-1), "shape"), (dict(n_advantages=1), "shape"), (dict(board=7), "shape")])
def test_a_refused_policy_step(n, change, message):
    net, opt = trained()
    kept = Unchanged(net, opt)
    states = change.get("states", empty)(n)
    if "board" in change:
        states = np.zeros((n, 6, 7, 7), np.uint8)
    actions, adv = [7] * (n + change.get("n_actions", 0)), [1.0] * (n + change.get("n_advantages", 0))
    if "actions" in change:
        actions[-1] = change["actions"]
    if "advantages" in change:
        adv[-1] = change["advantages"]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(ValueError, match=message):
            net.policy_step(opt, states, actions, adv, change.get("entropy_weight", 0.01), change.get("temperature", 1.0))
    kept.check()


def test_an_illegal_action_of_no_weight_is_refused_too():
    net, opt = trained()
    kept = Unchanged(net, opt)
    with pytest.raises(ValueError, match="not legal"):
        net.policy_step(opt, occupied(2), [0, 7], [1.0, 0.0])
    kept.check()
    # the stone's position with a legal action, or without one, is fine
    assert np.isfinite(net.policy_step(opt, occupied(2), [7, 8], [1.0, 1.0])).all()
    assert np.isfinite(net.policy_step(opt, occupied(2), [7, -1], [1.0, 1.0])).all()
    assert opt.steps == 3


@pytest.mark.parametrize("n", [3, 6])
def test_an_optimiser_that_is_not_the_nets(n):
    from go_ai.models import AdamW
    net, opt = trained()
    other, elsewhere = net_of(), AdamW([torch.zeros(10).cuda()])
    others = AdamW()
    other.policy_step(others, empty(3), [0, 1, 2], [1.0, 1.0, 1.0])
    kept = Unchanged(net, opt)
    for bad, message in ((elsewhere, "belongs"), (others, "belongs"), (AdamW(grad_dtype=torch.bfloat16), "float32"),
                         (AdamW(grad_dtype=[torch.float16] * 26), "float32")):
        with pytest.raises(ValueError, match=message):
            net.policy_step(bad, empty(n), [0] * n, [1.0] * n)
        with pytest.raises(ValueError, match=message):
            net.train_step(bad, *batch(n))
        with pytest.raises(ValueError, match=message):
            net.optimize(None, [batch(n)], bad)
    kept.check()
