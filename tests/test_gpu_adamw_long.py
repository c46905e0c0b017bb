"""AdamW's moments in 8 bits over thousands of steps, against AdamW in float64: they follow their gradients, though a step moves a
root by far less than half a code.

A root r that a step moves by d, less than its code's step s <= r / 16, stays or moves by s: unbiased, with a variance of at most |d| s.  Here
d = a r |g^2 / v - 1| with a = (1 - beta2) / 2, and r forgets at the rate a, so its own scatter has a variance of at most |d| s / (2 a) =
r^2 / 32 E|g^2 / v - 1|, for normal gradients (0.174 r)^2 (SD).  The mean of n elements is off by SD / sqrt(n) and by terms of the second order
(SD^2 = 0.03, also of the updates, which go with 1 / r).  To the nearest, the same runs give 9 times the root (half fall), 0.36
times (the largest falls silent), 1.16 times (all alike)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SD = 0.174


class Float64:
    """AdamW's moments and update in float64."""

    def __init__(self, n, b1=0.9, b2=0.999, eps=1e-8):
        self.m = torch.zeros(n, dtype=torch.float64, device="cuda")
        self.v = self.m.clone()
        self.b, self.eps, self.t = (b1, b2), eps, 0

    def step(self, g):
        b1, b2 = self.b
        self.t += 1
        g = g.double()
        self.m.mul_(b1).add_(g, alpha=1 - b1)
        self.v.mul_(b2).addcmul_(g, g, value=1 - b2)
        return self.m / (1 - b1 ** self.t) / ((self.v / (1 - b2 ** self.t)).sqrt() + self.eps)


def run(grad, n, steps, b1=0.9, b2=0.999, look=500, captured=False, lr=1e-6, start=None):
    """`steps` steps; the optimiser, the float64 one, and the sums of both's updates over the last `look` steps (in units of lr)."""
    from go_ai.models import AdamW
    g = torch.Generator("cuda").manual_seed(5)
    p = torch.zeros(n, device="cuda")
    opt, ref = AdamW([p], lr=lr, betas=(b1, b2), weight_decay=0.0, state_bits=8), Float64(n, b1, b2)
    if start is not None:
        opt.load_moments([start[0]], [start[1]], start[2])
        ref.m, ref.v, ref.t = start[0].double(), start[1].double(), start[2]
    total = torch.zeros(n, dtype=torch.float64, device="cuda")
    buf = torch.empty(n, device="cuda")
    graph = None
    if captured:
        opt.advance()
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s):
            with torch.cuda.graph(graph, stream=s):
                opt.step([buf], captured=True)
        torch.cuda.synchronize()
    for k in range(steps):
        if k == steps - look:
            p.zero_()
        buf.copy_(grad(k, g))
        if captured:
            if k:
                opt.advance()
            graph.replay()
        else:
            opt.step([buf])
        u = ref.step(buf)
        if k >= steps - look:
            total -= u
    torch.cuda.synchronize()
    return opt, ref, p.double() / lr, total


def root_ratio(opt, ref, where):
    return (opt.moments()[1][:ref.v.numel()].double().sqrt() / ref.v.sqrt())[where].cpu().numpy()


def holds(ratio, got, want):
    n = ratio.size
    assert abs(ratio.mean() - 1) <= 5 * SD / math.sqrt(n) + SD ** 2, ratio.mean()
    lo, hi = np.quantile(ratio, [0.01, 0.99])
    # 1 % of a normal scatter is beyond 2.33 deviations
    assert 1 - 3 * SD <= lo and hi <= 1 + 3 * SD, (lo, hi)
    slope = float((got * want).sum() / (want * want).sum())
    assert abs(slope - 1) <= SD ** 2 + 5 * SD / math.sqrt(n) + 0.01, slope


N = 256 * 40


def normal(k, g):
    return torch.randn(N, generator=g, device="cuda")


def halves(k, g):
    x = normal(k, g).view(-1, 256)
    if k >= 3000:
        x[:, 128:] *= 0.1
    return x.view(-1)


def silent(k, g):
    x = normal(k, g).view(-1, 256)
    x[:, 0] *= 5 if k < 3000 else 0
    return x.view(-1)


WITHIN = torch.arange(N) % 256


@pytest.mark.parametrize("name,grad,steps,where", [("alike", normal, 3000, WITHIN >= 0), ("half fall", halves, 10000, WITHIN >= 128),
                                                   ("the largest falls silent", silent, 6000, WITHIN >= 1)])
def test_moments_follow(name, grad, steps, where):
    opt, ref, got, want = run(grad, N, steps)
    where = where.cuda()
    holds(root_ratio(opt, ref, where), got[where], want[where])


def test_captured_moments_follow():
    """The replays of one captured step draw other numbers each (its number is counted on the GPU)."""
    opt, ref, got, want = run(halves, N, 10000, captured=True)
    where = (WITHIN >= 128).cuda()
    holds(root_ratio(opt, ref, where), got[where], want[where])


def test_loaded_moments_follow():
    """From moments of a long run, as a training run resumes."""
    g = torch.Generator("cuda").manual_seed(1)
    start = (0.1 * torch.randn(N, generator=g, device="cuda"), 1 + 0.1 * torch.randn(N, generator=g, device="cuda"), 20000)
    opt, ref, got, want = run(lambda k, g: 0.1 * normal(k, g), N, 5000, start=start)
    holds(root_ratio(opt, ref, WITHIN.cuda() >= 0), got, want)


@pytest.mark.parametrize("b1", [0.9, 0.98])
def test_elements_without_gradients_come_to_rest(b1):
    """Half of each block has no gradients after step 300: their first moments are 0 after 3000 steps (expected size m0 b1^n, under
    2^-60 of e4m3's smallest), not four of its smallest steps for ever, and the parameters stay where they are."""
    from go_ai.models import AdamW
    g = torch.Generator("cuda").manual_seed(3)
    p = torch.zeros(N, device="cuda")
    opt = AdamW([p], betas=(b1, 0.999), weight_decay=0.0, state_bits=8)
    dead = (WITHIN >= 128).cuda()
    for k in range(3000):
        x = normal(k, g)
        if k >= 300:
            x[dead] = 0
        opt.step([x])
    assert not opt.moments()[0][dead].any()
    before = p.clone()
    for k in range(20):
        opt.step([torch.where(dead, 0.0, normal(k, g))])
    assert torch.equal(before[dead], p[dead]) and not torch.equal(before, p)


@pytest.mark.parametrize("b1", [0.9, 0.98])
def test_constant_gradients_that_fall(b1):
    """First moments of constant gradients end on one of the two codes around them (2^-3), also after a fall by a third of half the elements,
    though at beta1 = 0.98 a step moves them by less than half a code.  A code that is met exactly comes back some 2^-22 off, and one in
    some 3e5 steps then falls by one more: a few of 10240 elements are on their way back at any time."""
    w = torch.linspace(0.3, 1, 256).repeat(N // 256).cuda()
    third = torch.where(WITHIN.cuda() >= 128, 2 / 3, 1.0)
    opt, ref, _, _ = run(lambda k, g: w if k < 500 else w * third, N, 1500, b1=b1)
    ratio = (opt.moments()[0][:N].double() / ref.m).cpu().numpy()
    off = np.abs(ratio - 1)
    assert np.quantile(off, 0.998) <= 2.0 ** -3 + 1e-3 and off.max() <= 2.0 ** -2 + 1e-3 and abs(ratio.mean() - 1) <= 0.02, (off.max(), ratio.mean())


def steps_of(n_steps, seed=7):
    from go_ai.models import AdamW
    g = torch.Generator("cuda").manual_seed(seed)
    p = [torch.zeros(5000, device="cuda"), torch.zeros(3, 300, device="cuda")]
    opt = AdamW(p, state_bits=8)
    for _ in range(n_steps):
        opt.step([torch.randn(x.shape, generator=g, device="cuda") for x in p])
    return p + list(opt.moments())


def test_same_steps_same_bits():
    assert all(torch.equal(a, b) for a, b in zip(steps_of(60), steps_of(60)))


def test_a_step_of_random_rounding():
    """Codes on either side of the value, and right on average: one step behind 20 of zero gradients, of values between two codes."""
    from go_ai.models import AdamW
    n = 256 * 400
    p = torch.zeros(n, device="cuda")
    opt = AdamW([p], betas=(0.5, 0.5), weight_decay=0.0, state_bits=8)
    for _ in range(20):
        opt.step([torch.zeros(n, device="cuda")])
    assert not any(x.any() for x in opt.moments())
    x = torch.rand(n, device="cuda", generator=torch.Generator("cuda").manual_seed(2)) * 1.5 + 0.5
    x[::256] = 2.0
    opt.step([x])
    m, v = opt.moments()
    for got, want, step in ((m.double(), 0.5 * x.double(), 2.0 ** -3), (v.double().sqrt(), (0.5 * x.double() ** 2).sqrt(), 2.0 ** -4)):
        off = (got / want - 1).cpu().numpy()
        assert np.abs(off).max() <= step * (1 + 1e-5) and np.abs(off).max() >= 0.6 * step         # beyond half a step: not the nearest
        assert abs(off.mean()) <= 5 * 0.5 * step / math.sqrt(n)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_gradient_that_is_not_finite(bad):
    """Spoils its block, as with rounding to the nearest, and no other."""
    from go_ai.models import AdamW
    n = 256 * 3
    p = torch.zeros(n, device="cuda")
    opt = AdamW([p], weight_decay=0.0, state_bits=8)
    g = torch.ones(n, device="cuda")
    for _ in range(20):
        opt.step([g])
    g[300] = bad
    opt.step([g])
    m, v = opt.moments()
    fine = torch.ones(n, dtype=torch.bool, device="cuda")
    fine[256:512] = False
    assert torch.isnan(m[300]) and torch.isnan(p[300]) and torch.isfinite(m[fine]).all() and torch.isfinite(v[fine]).all()
    assert torch.isfinite(p[fine]).all() and (m[fine] > 0).all()
