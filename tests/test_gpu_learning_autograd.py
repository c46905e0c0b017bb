"""The learning operators beside autograd: what it cannot see is refused, and what they change in place it notices."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from go_ai.engine import Context
    c = Context(9)
    yield c
    c.close()


def test_logits_that_require_a_gradient(ctx):
    x = torch.randn(5, 82, device="cuda", requires_grad=True)
    a = torch.zeros(5, dtype=torch.int32, device="cuda")
    for logits in (x, x * 2, x.double(), x.t().contiguous().t()):
        with pytest.raises(ValueError, match="detach"):
            ctx.action_logprobs(logits, a)
        with pytest.raises(ValueError, match="detach"):
            ctx.action_logprobs_grad(logits, a, torch.zeros(5, device="cuda"), d_logp=torch.ones(5, device="cuda"))
    r = ctx.action_logprobs(x.detach(), a)
    with torch.no_grad():
        assert torch.equal(ctx.action_logprobs(x, a).logp, r.logp)
    with torch.inference_mode():
        assert torch.equal(ctx.action_logprobs(x, a).logp, r.logp)
    # the way through: the gradient of sum(logp) handed to autograd
    d = ctx.action_logprobs_grad(x.detach(), a, r.lse, d_logp=torch.ones(5, device="cuda"))
    x.backward(d)
    y = x.detach().double().requires_grad_(True)
    torch.log_softmax(y, 1).gather(1, a.long()[:, None]).sum().backward()
    assert float((x.grad.double() - y.grad).abs().max()) < 1e-6


def test_a_gradient_written_over_saved_logits(ctx):
    w = torch.randn(5, 82, device="cuda", requires_grad=True)
    x = torch.randn(5, 82, device="cuda")
    saved = (w * x).sum()                                    # w's gradient needs x
    a = torch.zeros(5, dtype=torch.int32, device="cuda")
    r = ctx.action_logprobs(x, a)
    d = ctx.action_logprobs_grad(x, a, r.lse, d_logp=torch.ones(5, device="cuda"), out=x)
    assert d is x
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    with pytest.raises(ValueError, match="in place"):
        ctx.action_logprobs_grad(x.clone(), a, r.lse, d_logp=torch.ones(5, device="cuda"), out=w)


@pytest.mark.parametrize("views", [False, True])
@pytest.mark.parametrize("parameter", [False, True])
def test_a_step_over_saved_parameters(views, parameter):
    """A graph that was recorded before the step must not run backward with the parameters behind it."""
    from go_ai.models import AdamW
    base = torch.randn(500, device="cuda")
    p = [base[3:203], base[203:403]] if views else [torch.randn(200, device="cuda"), torch.randn(200, device="cuda")]
    if parameter and not views:
        p = [torch.nn.Parameter(x) for x in p]
    g = [torch.ones(200, device="cuda") for _ in p]
    opt = AdamW(p)
    x = torch.randn(200, device="cuda", requires_grad=True)
    before = (x * p[1]).sum()
    opt.step(g)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        before.backward()
    (x * p[1]).sum().backward()
    assert torch.equal(x.grad, p[1].detach())
    opt.step(g)


def test_a_training_loop_with_autograd():
    """Forward, backward and step over torch parameters, as torch.optim.AdamW is used."""
    from go_ai.models import AdamW
    torch.manual_seed(0)
    net = torch.nn.Linear(7, 3).cuda()
    other = torch.nn.Linear(7, 3).cuda()
    other.load_state_dict(net.state_dict())
    opt, theirs = AdamW(net.parameters(), lr=1e-2), torch.optim.AdamW(other.parameters(), lr=1e-2)
    for k in range(5):
        x = torch.randn(11, 7, device="cuda", generator=torch.Generator("cuda").manual_seed(k))
        net.zero_grad()
        net(x).square().mean().backward()
        opt.step([p.grad for p in net.parameters()])
        theirs.zero_grad()
        other(x).square().mean().backward()
        theirs.step()
    for a, b in zip(net.parameters(), other.parameters()):
        assert np.allclose(a.detach().cpu().numpy(), b.detach().cpu().numpy(), rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("number", [np.float32, np.float64, torch.tensor, int])
def test_numbers_of_other_types(ctx, number):
    """Temperatures and learning rates as numpy or torch numbers, or whole ones."""
    from go_ai.models import AdamW
    from go_ai.models.ac_net import ActorCriticNet
    x = torch.randn(5, 82, device="cuda")
    a = torch.zeros(5, dtype=torch.int32, device="cuda")
    want = ctx.action_logprobs(x, a, temperature=2.0)
    assert torch.equal(ctx.action_logprobs(x, a, temperature=number(2)).logp, want.logp)
    g = torch.ones(5, device="cuda")
    assert torch.equal(ctx.action_logprobs_grad(x, a, want.lse, d_logp=g, temperature=number(2)),
                       ctx.action_logprobs_grad(x, a, want.lse, d_logp=g, temperature=2.0))
    p, q = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    opt, other = AdamW([p]), AdamW([q])
    opt.lr, other.lr = number(2), 2.0
    for o in (opt, other):
        o.step([torch.ones(300, device="cuda")])
    assert torch.equal(p, q) and p.any()
    net, loss = ActorCriticNet(5, n_blocks=0, max_batch=4, train_batch=4), []
    st = np.zeros((2, 6, 5, 5), np.uint8)
    opt = AdamW(lr=0.0)
    for t in (number(2), 2.0):
        loss.append(net.policy_step(opt, st, [0, 1], [1.0, 1.0], entropy_weight=number(1), temperature=t))
    assert loss[0] == loss[1]
