"""Many rows of more than 384 columns: from 2048 rows on a wavefront takes a row, tile by tile, where fewer rows take four or are split.
Against float64 on the GPU, with bounds that do not grow with the length of a row: its sums carry their roundings from tile to tile."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ctx():
    from go_ai.engine import Context
    c = Context(9)
    yield c
    c.close()


class Exact:
    """The definition in float64, and bounds of a float32 computation's error.

    A power 2^t is off by 2 U of |t| in t (difference and product) and by its own step 2 U; with A = sum p |s - max s| that is U (2 A + 2) of the
    sum.  Then the additions: 16 columns four ways 5 U, tiles with carry 2 U, three joins (lanes, wavefronts, segments) of 6 additions and a
    raise of 5 U each, 33 U.  A raise from tile to tile multiplies what was summed before by a factor that is off by 5 U: in a row in random
    order ten of them at most weigh anything (`raises`).  The logarithm, max s and their sum: 2 U log l, 2 U |max s|, U |lse|."""

    def __init__(self, x, valid=None, temperature=1.0, raises=10):
        self.x = x
        there = x > -math.inf
        if valid is not None:
            there = there & (valid != 0)
        s = torch.where(there, x.double() / temperature, -math.inf)
        self.there, self.some = there, there.any(1)
        peak = torch.where(self.some, s.amax(1), 0.0)
        off = torch.where(there, s - peak[:, None], 0.0)
        e = torch.where(there, off.exp(), 0.0)
        total = e.sum(1)
        logl = torch.where(self.some, total, 1.0).log()
        self.s = s
        self.lse = torch.where(self.some, peak + logl, -math.inf)
        p = e / torch.where(self.some, total, 1.0)[:, None]
        A, A2 = (p * off.abs()).sum(1), (p * off * off).sum(1)
        self.entropy = torch.where(self.some, logl + A, 0.0)
        self.rel = U * (2 * A + 2 + 7 + 33 + 5 * raises)
        self.lse_tol = self.rel + U * (2 * logl + 2 * peak.abs() + torch.where(self.some, self.lse, 0.0).abs())
        self.entropy_tol = self.rel + U * 2 * logl + A * (self.rel + 8 * U) + 2 * U * A2 + U * (logl + A)
        self.peak = peak

    def logp(self, a):
        m = self.x.shape[1]
        lp = self.s.gather(1, a.long().clamp(0, m - 1)[:, None])[:, 0] - torch.where(self.some, self.lse, 0.0)
        lp = torch.where(self.some, lp, -math.inf)
        return torch.where(a < 0, 0.0, torch.where(a >= m, math.nan, lp))

    def logp_tol(self, lp):
        f = torch.where(torch.isfinite(lp), lp.abs(), 0.0)
        return self.rel + U * (2 * (self.lse - self.peak).abs().nan_to_num(0.0, 0.0, 0.0) + 4 * f + 4 * (self.lse - self.peak).abs().nan_to_num(0.0, 0.0, 0.0))

    def best(self, top):
        order, at = torch.sort(self.s, dim=1, descending=True, stable=True)
        order, at = order[:, :top], at[:, :top]
        none = order == -math.inf
        lp = torch.where(none, -math.inf, order - torch.where(self.some, self.lse, 0.0)[:, None])
        return at.masked_fill(none, -1).int(), lp


def same(got, want, tol, what):
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine].nan_to_num(5.0, 6.0, 7.0), want[~fine].nan_to_num(5.0, 6.0, 7.0)), what
    off = ((got - want).abs() - tol)[fine]
    assert torch.isfinite(got[fine]).all() and (not off.numel() or float(off.max()) <= 0), (what, float(off.max()))


def check(ctx, x, a, valid=None, temperature=1.0, top=0, raises=10):
    r = ctx.action_logprobs(x, a, valid=valid, temperature=temperature, top=top)
    e = Exact(x, valid, temperature, raises)
    same(r.lse, e.lse, e.lse_tol, "lse")
    same(r.entropy, e.entropy, e.entropy_tol, "entropy")
    lp = e.logp(a)
    same(r.logp, lp, e.logp_tol(lp), "logp")
    if top:
        at, best = e.best(top)
        assert torch.equal(r.top_actions, at)
        m = best.shape[1]
        tol = torch.stack([e.logp_tol(best[:, k]) for k in range(m)], 1)
        same(r.top_logp, best, tol, "top")
    return r, e


def make(rows, cols, dtype, seed, masked):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (3 * torch.randn((rows, cols), generator=g, device="cuda")).to(dtype)
    valid = None
    if masked:
        valid = (torch.rand((rows, cols), generator=g, device="cuda") < 0.5).to(torch.uint8)
        valid[::7] = 0                                                           # rows without an allowed column
        valid[5::7, : cols // 2] = 0
        x[valid == 0] = float("nan")                                             # (what is masked is never used)
        x[3::11] = torch.where(torch.rand((len(range(3, rows, 11)), cols), generator=g, device="cuda") < 0.3, -math.inf, x[3::11].float()).to(dtype)
    a = torch.randint(-1, cols + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return x, valid, a


def clean(x, valid):
    return x if valid is None else torch.where(valid != 0, x, torch.zeros_like(x))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(2048, 385), (2051, 1025), (2049, 5003), (2048, 30001), (700, 5003), (60, 30001)])
@pytest.mark.parametrize("top,masked,temperature", [(0, False, 1.0), (1, True, 0.7), (20, False, 1.5), (64, True, 1.0)])
def test_forward(ctx, rows, cols, dtype, top, masked, temperature):
    x, valid, a = make(rows, cols, dtype, rows + cols, masked)
    r = ctx.action_logprobs(x, a, valid=valid, temperature=temperature, top=top)
    e = Exact(clean(x, valid), valid, temperature)
    same(r.lse, e.lse, e.lse_tol, "lse")
    same(r.entropy, e.entropy, e.entropy_tol, "entropy")
    lp = e.logp(a)
    same(r.logp, lp, e.logp_tol(lp), "logp")
    if top:
        at, best = e.best(top)
        assert torch.equal(r.top_actions, at)
        for k in range(top):
            same(r.top_logp[:, k], best[:, k], e.logp_tol(best[:, k]), k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(2048, 3001), (2048, 30001), (3, 30001)])
@pytest.mark.parametrize("kind", ["rising", "falling", "equal", "few values", "late"])
def test_orders_and_ties(ctx, rows, cols, dtype, kind):
    """Rows whose every tile enters the list, or none behind the first; equal columns; the best at the end.  (A rising row raises from
    tile to tile: as many raises as tiles.)"""
    g = torch.Generator("cuda").manual_seed(cols)
    j = torch.arange(cols, device="cuda", dtype=torch.float32)
    row = {"rising": j / cols * 20, "falling": -j / cols * 20, "equal": 0 * j + 1.25, "late": torch.where(j >= cols - 40, j / cols, -3.0),
           "few values": torch.randint(0, 4, (cols,), generator=g, device="cuda").float()}[kind]
    x = row.repeat(rows, 1)
    x[1::2] += 0.5
    x = x.to(dtype)
    a = torch.randint(0, cols, (rows,), generator=g, device="cuda", dtype=torch.int32)
    for top in (1, 20, 64):
        check(ctx, x, a, top=top, raises=10 if kind != "rising" else cols // 1024 + 2)


@pytest.mark.parametrize("rows", [2048, 600, 2])
@pytest.mark.parametrize("cols", [30001, 128001, 200000])
def test_long_rows_of_equal_columns(ctx, rows, cols):
    """Equal logits below larger ones in the first tiles (a lane that has seen nothing larger adds ones): equal terms round the same way
    again and again, 2000 of them up to 3e-5 of their sum one by one, and the bound does not know the length."""
    rows = min(rows, 2048 if cols < 100000 else 2100)
    x = torch.empty((rows, cols), device="cuda")
    for k, v in enumerate((0.0, -0.3, -1.7, -2.9)):
        x[k::4] = v + 0.37
    x[:, :4096] += torch.linspace(0.1, 0.9, rows, device="cuda")[:, None]
    a = torch.full((rows,), 5, device="cuda", dtype=torch.int32)
    if rows * cols <= 2048 * 130000:
        check(ctx, x, a, raises=1)
    else:
        for part in range(0, 4):
            r = ctx.action_logprobs(x, a)
            e = Exact(x[part:part + 8], raises=1)
            same(r.lse[part:part + 8], e.lse, e.lse_tol, "lse")
            same(r.entropy[part:part + 8], e.entropy, e.entropy_tol, "entropy")


@pytest.mark.parametrize("cols", [385, 1025, 5003])
def test_nan_and_infinity(ctx, cols):
    rows = 2048
    x, _, a = make(rows, cols, F32, 1, False)
    a = a.clamp(0, cols - 2)
    x[::3, cols - 1] = math.nan
    x[1::3, cols // 2] = math.inf
    x[2::6] = -math.inf
    r = ctx.action_logprobs(x, a, top=3)
    for v in (r.lse, r.entropy, r.logp):
        assert torch.isnan(v[::3]).all() and torch.isnan(v[1::3])[a[1::3] != cols // 2].all()
    assert (r.lse[2::6] == -math.inf).all() and (r.entropy[2::6] == 0).all() and (r.logp[2::6] == -math.inf).all()
    assert (r.top_actions[2::6] == -1).all() and (r.top_logp[2::6] == -math.inf).all()
    assert not (r.top_actions[::3] == cols - 1).any()
    e = Exact(x[5::6])
    same(r.lse[5::6], e.lse, e.lse_tol, "lse")


def test_strided_and_shared_rows(ctx):
    """A column range of a wider array at an odd offset, one mask for all rows, one row for all."""
    rows, cols = 2050, 3003
    for dtype in (F32, F16):
        g = torch.Generator("cuda").manual_seed(4)
        wide = torch.randn((rows, cols + 9), generator=g, device="cuda").to(dtype)
        x = wide[:, 3:3 + cols]
        valid = (torch.rand((1, cols), generator=g, device="cuda") < 0.7).to(torch.uint8).expand(rows, cols)
        a = torch.randint(0, cols, (rows,), generator=g, device="cuda", dtype=torch.int32)
        lp_masked = ~(valid.gather(1, a.long()[:, None])[:, 0] != 0)
        r = ctx.action_logprobs(x, a, valid=valid, top=20)
        e = Exact(x, valid)
        same(r.lse, e.lse, e.lse_tol, "lse")
        assert (r.logp[lp_masked] == -math.inf).all() and torch.equal(r.top_actions, e.best(20)[0])
        one = x[:1].expand(rows, cols)
        r = ctx.action_logprobs(one, a, top=5)
        e = Exact(one[:1].contiguous())
        assert torch.equal(r.lse, r.lse[:1].expand(rows)) and torch.equal(r.top_actions, r.top_actions[:1].expand(rows, 5))
        same(r.lse[:1], e.lse, e.lse_tol, "lse")
