"""AdamW's parts by themselves: the gradients' norm without a step, and the kernel's square root on every significand."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_grad_norm(dtype):
    """Float64 sums in a fixed order, rounded once; parameters, moments and the step's number stay."""
    from go_ai.models import AdamW
    g = torch.Generator("cuda").manual_seed(2)
    shapes = [(1,), (0,), (300,), (7, 1001), (70001,)] + [(3,)] * 300                 # two launches
    p = [torch.randn(s, generator=g, device="cuda").to(dtype) for s in shapes]
    grads = [torch.randn(s, generator=g, device="cuda").to(dtype) for s in shapes]
    opt = AdamW(p)
    before = [x.clone() for x in p]
    norm = lambda gs: math.sqrt(sum(float(x.double().square().sum()) for x in gs if x is not None))  # noqa: E731
    want = norm(grads)
    first = opt.grad_norm(grads)
    assert abs(float(first) - want) <= 2 * U * want and torch.equal(first, opt.grad_norm(grads))
    some = [None if i % 3 == 0 else x for i, x in enumerate(grads)]
    assert abs(float(opt.grad_norm(some)) - norm(some)) <= 2 * U * want
    assert float(opt.grad_norm([None] * len(p))) == 0.0
    grads[4][70000] = math.inf
    assert float(opt.grad_norm(grads)) == math.inf
    grads[4][70000] = math.nan
    assert math.isnan(float(opt.grad_norm(grads)))
    with pytest.raises(ValueError):
        opt.grad_norm(grads[:-1])
    assert opt.steps == 0 and all(torch.equal(a, b) for a, b in zip(before, p)) and not any(m.any() for m in opt.moments())


def roots(x):
    """The kernel's square roots of x, squared: a block of 256 with one number that is not 0 has its root as its scale, and that root's
    square comes back.  (Two neighbouring roots' float32 squares differ: they are two steps of a root apart, relative to them.)"""
    from go_ai.models import AdamW
    n = x.numel()
    p = torch.zeros(256 * n, dtype=torch.bfloat16, device="cuda")
    opt = AdamW([p], state_bits=8)
    spread = torch.zeros((n, 256), device="cuda")
    spread[:, 37] = x.cuda()
    opt.load_moments([spread.view(-1)], [spread.view(-1)], 0)
    got = opt.moments()[1].view(n, 256)
    assert not got[:, :37].any() and not got[:, 38:].any()
    return got[:, 37].cpu()


@pytest.mark.parametrize("part", range(8))
def test_square_root_of_every_significand(part):
    """[1, 4): the powers of two between which a root and its steps only change by their exponents."""
    first = 0x3f800000 + part * (1 << 21)
    x = torch.arange(first, first + (1 << 21), dtype=torch.int32).view(torch.float32)
    want = torch.from_numpy(np.sqrt(x.numpy()))                  # (correctly rounded)
    assert torch.equal(roots(x), want * want)


def test_square_root_over_the_range():
    """Every exponent, on either side of 2^-102 where the kernel's own root ends (below 2^-126 after the root: held as zeros)."""
    rng = np.random.default_rng(0)
    bits = rng.integers(0, 1 << 23, (254, 64), dtype=np.int64) + (np.arange(1, 255, dtype=np.int64)[:, None] << 23)
    x = torch.from_numpy(bits.astype(np.int32).reshape(-1)).view(torch.float32)
    want = torch.from_numpy(np.sqrt(x.numpy()))
    got, square = roots(x), want * want
    assert torch.equal(got[square >= 2.0 ** -126], square[square >= 2.0 ** -126])
    assert float((got - x).abs().max() / x.max()) < 4 * U and torch.isfinite(got[x < 3e38]).all()
