"""A call works on its context's GPU and leaves the caller on its own."""
import gc

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def calls(device):
    from go_ai.engine import Context
    from go_ai.models import AdamW
    now = torch.cuda.current_device()
    c = Context(9, device)
    assert torch.cuda.current_device() == now
    x = torch.randn(5, 82, device=f"cuda:{device}")
    a = torch.zeros(5, dtype=torch.int32, device=f"cuda:{device}")
    r = c.action_logprobs(x, a, top=3)
    d = c.action_logprobs_grad(x, a, r.lse, d_logp=torch.ones(5, device=f"cuda:{device}"))
    assert torch.cuda.current_device() == now and r.lse.device == d.device == x.device
    c.transition(np.zeros((2, 6, 9, 9), np.uint8), [0, 1])
    opt = AdamW([x], max_norm=1.0, state_bits=8)
    opt.step([torch.ones_like(x)])
    assert opt.steps == 1 and torch.cuda.current_device() == now
    want = torch.log_softmax(x.double(), 1)
    del opt, c
    gc.collect()
    assert torch.cuda.current_device() == now and torch.isfinite(want).all()
    torch.cuda.synchronize(device)


def test_on_the_current_device():
    calls(torch.cuda.current_device())


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
@pytest.mark.parametrize("now,other", [(0, 1), (1, 0)])
def test_on_another_device(now, other):
    with torch.cuda.device(now):
        calls(other)
        assert torch.zeros(1, device="cuda").device.index == now
