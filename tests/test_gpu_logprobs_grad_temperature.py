"""The gradient's 1 / T is the forward pass's: rows where one column has all the probability have no gradient, however large logit / T is."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from go_ai.engine import Context
    c = Context(9)
    yield c
    c.close()


@pytest.mark.parametrize("temperature", [0.7, 1.3, 1e-3, 3e-4, 77.0])
@pytest.mark.parametrize("cols", [1, 26, 82, 362, 1500, 9000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_only_column(ctx, cols, dtype, temperature):
    """log p = x / T - lse is 0 for it: the same product, the same rounding."""
    n = 64
    g = torch.Generator("cuda").manual_seed(cols)
    x = (torch.rand((n, cols), generator=g, device="cuda") * 2000 - 1000).to(dtype)
    a = torch.randint(0, cols, (n,), generator=g, device="cuda", dtype=torch.int32)
    valid = torch.zeros((n, cols), dtype=torch.uint8, device="cuda").scatter_(1, a.long()[:, None], 1)
    r = ctx.action_logprobs(x, a, valid=valid, temperature=temperature)
    assert not r.logp.any() and not r.entropy.any()
    one = torch.ones(n, device="cuda")
    d = ctx.action_logprobs_grad(x, a, r.lse, r.entropy, one, one, valid=valid, temperature=temperature)
    assert not d.any()


@pytest.mark.parametrize("temperature", [0.7, 1.3])
def test_two_equal_columns(ctx, temperature):
    """p = 1/2 up to lse's own rounding: lse = x / T + log 2 rounds once (U |lse|), log 2 and its sum with x / T add 2 U."""
    n = 4096
    x = torch.linspace(-3000, 3000, n, device="cuda")[:, None].repeat(1, 2)
    a = torch.zeros(n, dtype=torch.int32, device="cuda")
    r = ctx.action_logprobs(x, a, temperature=temperature)
    d = ctx.action_logprobs_grad(x, a, r.lse, d_logp=torch.ones(n, device="cuda"), temperature=temperature)
    off = (d.double() * temperature - torch.tensor([0.5, -0.5], device="cuda")).abs()
    tol = 0.5 * U * (2 * r.lse.double().abs() + 12)
    assert (off <= tol[:, None]).all()
