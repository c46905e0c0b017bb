"""Log probabilities of actions and their gradient (Context.action_logprobs / action_logprobs_grad) against their definitions in
float64 on the host.  They have no counterpart in the reference beyond the cross entropy of one greedy target
(go_ai/models/__init__.py:175-184)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                    # half a float32 step, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}     # below: flushed, or half a subnormal step
FMAX = float(np.finfo(np.float32).max)


@pytest.fixture(scope="module")
def ctx():
    from go_ai.engine import Context
    c = Context(9)
    yield c
    c.close()


def definition(logits, valid=None, actions=None, temperature=1.0, top=0):
    x = logits.double().cpu().numpy()
    n, m = x.shape
    there = x > -np.inf
    if valid is not None:
        there &= valid.cpu().numpy().astype(bool)
    s = np.where(there, np.where(there, x, 0.0) / temperature, -np.inf)
    some = there.any(1)
    peak = np.where(some, s.max(1, initial=-np.inf), 0.0)[:, None]
    e = np.where(there, np.exp(s - peak), 0.0)
    logl = np.log(np.where(some, e.sum(1), 1.0))[:, None]
    lse = np.where(some, (peak + logl)[:, 0], -np.inf)
    lp = np.where(there, s - peak - logl, -np.inf)
    p = np.exp(lp)
    entropy = -np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0).sum(1)
    r = dict(there=there, lp=lp, p=p, lse=lse, entropy=entropy, s=np.where(there, s, 0.0))
    if actions is not None:
        a = actions.cpu().numpy()
        r["logp"] = np.where(a < 0, 0.0, lp[np.arange(n), np.clip(a, 0, m - 1)])
        r["logp"][a >= m] = np.nan
    if top:
        order = np.argsort(np.where(there, -x, np.inf), axis=1, kind="stable")[:, :top]
        none = ~np.take_along_axis(there, order, 1)
        best, best_lp = np.where(none, -1, order), np.where(none, -np.inf, np.take_along_axis(lp, order, 1))
        short = top - best.shape[1]
        r["top_actions"] = np.pad(best, ((0, 0), (0, max(short, 0))), constant_values=-1)
        r["top_logp"] = np.pad(best_lp, ((0, 0), (0, max(short, 0))), constant_values=-np.inf)
    return r


def bounds(want, cols):
    """Absolute error bounds of lse, entropy, log p.  A power 2^t carries 2 roundings of t (relative 2 U |t|, |t| ln 2 in the power)
    and the power's own step 2 U; weighted by the probabilities, |t| averages to at most log2(cols).  A lane adds at most
    cols / 16 + 16 numbers one after the other (a wavefront per row or more); the rest are the last operations' roundings."""
    size = np.abs(want["s"]).max(1, initial=0.0)
    with np.errstate(invalid="ignore"):
        lse = U * (4 * math.log2(cols + 1) + cols / 16 + 32 + 4 * np.where(np.isfinite(want["lse"]), np.abs(want["lse"]), 0) + 4 * size)
    return lse, 2 * lse * (1 + math.log(cols)), lambda lp: lse + 4 * U * (np.where(np.isfinite(lp), np.abs(lp), 0) + size)


def same(got, want, tol):
    got, want = got.double().cpu().numpy(), np.asarray(want)
    tol = np.broadcast_to(tol, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
    assert np.isfinite(got[fine]).all()
    off = np.abs(got[fine] - want[fine]) - tol[fine]
    assert off.max(initial=-1.0) <= 0, (got[fine][off.argmax()], want[fine][off.argmax()], tol[fine][off.argmax()])


def check(ctx, logits, valid=None, actions=None, temperature=1.0, top=0, vals=None):
    r = ctx.action_logprobs(logits, actions, valid=valid, temperature=temperature, top=top)
    torch.cuda.synchronize()
    want = definition(logits, valid, actions, temperature, top)
    lse, ent, lp = bounds(want, logits.shape[1])
    same(r.lse, want["lse"], lse)
    same(r.entropy, want["entropy"], ent)
    if actions is not None:
        same(r.logp, want["logp"], lp(want["logp"]))
    else:
        assert r.logp is None
    if top:
        assert np.array_equal(r.top_actions.cpu().numpy(), want["top_actions"])
        lse2 = lse[:, None]
        size = np.abs(want["s"]).max(1, initial=0.0)[:, None]
        f = np.where(np.isfinite(want["top_logp"]), np.abs(want["top_logp"]), 0)
        same(r.top_logp, want["top_logp"], lse2 + 4 * U * (f + size))
    else:
        assert r.top_actions is None and r.top_logp is None
    return r, want


def check_grad(ctx, logits, actions, g, h, valid=None, temperature=1.0, out=None):
    want = definition(logits, valid, actions, temperature)
    n, m = logits.shape
    lse = torch.from_numpy(want["lse"]).float().cuda()
    ent = torch.from_numpy(want["entropy"]).float().cuda()
    x = logits.clone() if out is logits else logits
    got = ctx.action_logprobs_grad(logits, actions, lse, ent, g, h, valid=valid, temperature=temperature, out=out)
    torch.cuda.synchronize()
    a = actions.cpu().numpy() if actions is not None else np.full(n, -1)
    gg = np.where(a < 0, 0.0, g.double().cpu().numpy()) if g is not None else np.zeros(n)
    hh = h.double().cpu().numpy() if h is not None else np.zeros(n)
    p, there = want["p"], want["there"]
    lp = np.where(p > 0, np.where(there, want["lp"], 0.0), 0.0)
    hot = np.arange(m)[None, :] == a[:, None]
    H = want["entropy"][:, None]
    d = np.where(there, (gg[:, None] * (hot - p) - hh[:, None] * p * (lp + H)) / temperature, 0.0)
    # log p is off by the roundings of x / T (2), of lse (1) and of their difference, p by ln 2 (log p's error and its own step);
    # then four operations on the terms, and the rounding to the logits' type
    dlp = U * (4 * np.abs(want["s"]) + 3 * np.where(np.isfinite(want["lse"]), np.abs(want["lse"]), 0)[:, None] + 3 * np.abs(lp) + 4)
    terms = (np.abs(gg)[:, None] * (p * (dlp + 8 * U) + hot * 4 * U) + np.abs(hh)[:, None] * p * (np.abs(lp + H) * (dlp + 8 * U) + dlp + 4 * U * (np.abs(lp) + H + 1)))
    tol = terms / temperature
    tol = tol + HALF[x.dtype] * (np.abs(d) + tol) + TINY[x.dtype]
    same(got, d, tol)
    return got, d


def make(rows, cols, dtype, seed, masked=False, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (scale * torch.randn((rows, cols), generator=g)).to(dtype).cuda()
    valid = None
    if masked:
        valid = (torch.rand((rows, cols), generator=g) < 0.5).to(torch.uint8)
        valid[::5] = 0
        valid = valid.cuda()
    a = torch.randint(-1, cols, (rows,), generator=g, dtype=torch.int32).cuda()
    return x, valid, a


SIZES = [(1, 1), (3, 2), (5, 26), (2, 50), (4, 63), (4, 64), (4, 65), (33, 82), (9, 127), (9, 128), (9, 129), (5, 170), (65, 362), (7, 511),
         (7, 512), (7, 513), (3, 1000), (3, 1023), (3, 1024), (3, 1025), (5, 2047), (2, 4097), (3, 8191), (1, 50021), (300, 3001), (2, 200003)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_forward(ctx, rows, cols, dtype):
    for masked, top, temperature in ((False, 0, 1.0), (True, 5, 1.0), (False, 64, 0.7), (True, 1, 1.5)):
        x, valid, a = make(rows, cols, dtype, rows * 7 + cols, masked)
        check(ctx, x, valid, a, temperature, top)


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradient(ctx, rows, cols, dtype):
    for masked, temperature in ((False, 1.0), (True, 0.7)):
        x, valid, a = make(rows, cols, dtype, rows + 3 * cols, masked)
        g, h = torch.randn(rows).cuda(), torch.randn(rows).cuda()
        check_grad(ctx, x, a, g, h, valid, temperature)


def test_many_rows(ctx):
    for rows, cols in ((100_003, 26), (40_001, 82), (5_000, 362)):
        x, valid, a = make(rows, cols, torch.float32, rows, True)
        check(ctx, x, valid, a, 1.0, 3)
        check_grad(ctx, x, a, torch.randn(rows).cuda(), torch.randn(rows).cuda(), valid)


def test_no_rows(ctx):
    x = torch.empty((0, 82)).cuda()
    r = ctx.action_logprobs(x, torch.empty(0, dtype=torch.int32).cuda(), top=3)
    assert r.logp.shape == (0,) and r.top_actions.shape == (0, 3)
    assert ctx.action_logprobs_grad(x, None, r.lse).shape == (0, 82)


@pytest.mark.parametrize("cols", [1, 26, 82, 362, 1500, 9001])
def test_what_is_masked_is_never_used(ctx, cols):
    """NaN, infinities and the types' lowest values behind the mask; rows without anything; -inf among the allowed."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x, valid, a = make(40, cols, dtype, cols, True)
        bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min, torch.finfo(dtype).max]).to(dtype).cuda()
        fill = bad[torch.arange(cols).cuda() % 5].expand(40, cols)
        x = torch.where(valid.bool(), x, fill)
        x[7] = -math.inf
        valid[7] = 1
        r, want = check(ctx, x, valid, a, 1.0, min(8, cols))
        assert float(r.entropy[0]) == 0.0 and float(r.lse[0]) == -math.inf and int(r.top_actions[0, 0]) == -1
        check_grad(ctx, x, a, torch.randn(40).cuda(), torch.randn(40).cuda(), valid)


@pytest.mark.parametrize("cols", [26, 82, 362, 5000])
def test_rows_of_the_lowest_value(ctx, cols):
    """A row full of the mask value of the numpy shim (float32's lowest) is uniform; one other column takes all."""
    for dtype in (torch.float32, torch.bfloat16):
        low = torch.finfo(dtype).min
        x = torch.full((4, cols), low, dtype=dtype).cuda()
        x[1, cols // 2] = 0.0
        x[2, cols - 1] = torch.finfo(dtype).max
        for temperature in (1.0, 0.5, 2.0):
            r = ctx.action_logprobs(x, torch.full((4,), cols // 2, dtype=torch.int32).cuda(), temperature=temperature, top=3)
            got = [t.cpu().numpy() for t in r]
            tol = 64 * U * (1 + math.log(cols))
            assert abs(got[1][0] - math.log(cols)) <= tol and abs(got[0][0] + math.log(cols)) <= tol
            assert got[0][1] == 0.0 and got[1][1] == 0.0 and got[3][1].tolist() == [cols // 2, 0, 1]
            assert got[0][2] == -math.inf and got[1][2] == 0.0 and got[3][2, 0] == cols - 1
            assert got[3][0].tolist() == [0, 1, 2] and np.isfinite(got[2]).all()


def test_nan_and_infinity_among_the_allowed(ctx):
    for cols in (30, 400, 7000):
        x = torch.randn(4, cols).cuda()
        x[0, 3] = math.nan
        x[1, 5] = math.inf
        r = ctx.action_logprobs(x, torch.full((4,), 7, dtype=torch.int32).cuda(), top=2)
        for t in (r.logp, r.entropy, r.lse):
            assert torch.isnan(t[:2]).all() and torch.isfinite(t[2:]).all()
        assert int(r.top_actions[1, 0]) == 5 and not (r.top_actions[0] == 3).any()
        d = ctx.action_logprobs_grad(x, torch.full((4,), 7, dtype=torch.int32).cuda(), r.lse, r.entropy, torch.ones(4).cuda(), torch.ones(4).cuda())
        assert torch.isnan(d[:2]).all() and torch.isfinite(d[2:]).all()


@pytest.mark.parametrize("cols", [26, 64, 82, 362, 1024, 1200, 20000])
@pytest.mark.parametrize("top", [1, 7, 64])
def test_ties_go_to_the_lower_column(ctx, cols, top):
    g = torch.Generator().manual_seed(cols)
    for dtype in (torch.float32, torch.bfloat16):
        few = torch.randint(0, 3, (6, cols), generator=g).to(dtype)          # three values: ties everywhere
        few[1] = 0.0
        few[2] = torch.where(torch.arange(cols) % 2 == 0, 0.0, -0.0)         # -0 equals 0
        few[3] = torch.arange(cols).to(dtype) / cols                         # each column better than the last
        few[4] = -torch.arange(cols).to(dtype) / cols
        check(ctx, few.cuda(), None, None, 1.0, top)
        valid = (torch.rand((6, cols), generator=g) < 0.5).to(torch.uint8).cuda()
        check(ctx, few.cuda(), valid, None, 0.01, top)                       # scaling merges none and ranks the logits themselves


def test_actions_out_of_range(ctx):
    x = torch.randn(5, 82).cuda()
    valid = torch.ones((5, 82), dtype=torch.bool).cuda()
    valid[3, 10] = False
    a = torch.tensor([-1, -2 ** 31, 82, 10, 2 ** 31 - 1], dtype=torch.int32).cuda()
    r = ctx.action_logprobs(x, a, valid=valid)
    assert r.logp[:2].tolist() == [0.0, 0.0] and torch.isnan(r.logp[[2, 4]]).all() and float(r.logp[3]) == -math.inf
    d = ctx.action_logprobs_grad(x, a, r.lse, d_logp=torch.ones(5).cuda(), valid=valid)
    assert (d[:2] == 0).all() and torch.isnan(d[2]).all() and torch.isnan(d[4][valid[4]]).all() and float(d[3, 10]) == 0.0
    p = torch.softmax(x[3].masked_fill(~valid[3], -math.inf), 0)
    assert torch.allclose(d[3], -p, atol=1e-6)


def strided_views(rows, cols, dtype):
    """The same matrix as the API may meet it: padded rows, an odd offset, every second row, columns first, one row for all."""
    big = torch.randn(2 * rows + 1, cols + 5).to(dtype).cuda()
    yield big[:rows, :cols]
    yield big[:rows, 3:cols + 3]
    yield big[1::2][:rows, 1:cols + 1]
    yield torch.randn(cols, rows).to(dtype).cuda().t()
    yield big[0, :cols].expand(rows, cols)
    flat = torch.randn(rows * cols + 1).to(dtype).cuda()
    yield flat[1:].view(rows, cols)


@pytest.mark.parametrize("rows,cols", [(1, 82), (9, 82), (9, 363), (5, 1001), (3, 5003), (2, 70001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strides_and_alignment(ctx, rows, cols, dtype):
    masks = [None, (torch.rand(rows, cols + 3) < 0.6).cuda()[:, 1:cols + 1], (torch.rand(cols) < 0.6).cuda().expand(rows, cols)]
    for i, x in enumerate(strided_views(rows, cols, dtype)):
        valid = masks[i % 3]
        a = torch.randint(0, cols, (rows,), dtype=torch.int32).cuda()
        check(ctx, x, valid, a, 1.0, 4)
        wide = torch.full((rows, cols + 7), 5.0, dtype=dtype).cuda()
        check_grad(ctx, x, a, torch.randn(rows).cuda(), torch.randn(rows).cuda(), valid, out=wide[:, 2:cols + 2])
        assert (wide[:, :2] == 5).all() and (wide[:, cols + 2:] == 5).all()


def test_gradient_in_place(ctx):
    for rows, cols in ((9, 82), (4, 5001)):
        x = torch.randn(rows, cols).cuda()
        check_grad(ctx, x, torch.zeros(rows, dtype=torch.int32).cuda(), torch.randn(rows).cuda(), torch.randn(rows).cuda(), out=x)


def test_gradient_parts(ctx):
    x, valid, a = make(9, 82, torch.float32, 1, True)
    g, h = torch.randn(9).cuda(), torch.randn(9).cuda()
    check_grad(ctx, x, a, g, None, valid)
    check_grad(ctx, x, None, None, h, valid)
    r = ctx.action_logprobs(x, a, valid=valid)
    assert (ctx.action_logprobs_grad(x, None, r.lse, valid=valid) == 0).all()


def test_gradient_against_differences(ctx):
    """Central differences of the loss sum(g log p) + sum(h H) in float64 at every logit of a few rows."""
    rows, cols, step = 3, 26, 1e-5
    x, valid, a = make(rows, cols, torch.float32, 4, False)
    a = a.clamp(min=0)
    g, h = torch.randn(rows).cuda(), torch.randn(rows).cuda()
    got = check_grad(ctx, x, a, g, h, None, 0.8)[0].double().cpu().numpy()
    base = x.double()

    def loss(v):
        w = definition(v, None, a, 0.8)
        return g.double().cpu().numpy() * w["logp"] + h.double().cpu().numpy() * w["entropy"]
    for j in range(cols):
        e = torch.zeros_like(base)
        e[:, j] = step
        slope = (loss(base + e) - loss(base - e)) / (2 * step)
        # second-order error: step^2 times a third derivative below 10 (|g| + |h| cols) / T^3; rounding: eps / step
        assert np.abs(slope - got[:, j]).max() < 1e-6, j


def test_long_offsets(ctx):
    """Rows whose offsets pass 2^31 elements (and 2^32 bytes)."""
    rows, cols, stride = 5, 82, 600_000_000
    x = torch.empty(4 * stride + cols, dtype=torch.float16, device="cuda")
    view = x.as_strided((rows, cols), (stride, 1))
    view.copy_(torch.randn(rows, cols))
    a = torch.randint(0, cols, (rows,), dtype=torch.int32).cuda()
    check(ctx, view, None, a, 1.0, 4)
    check_grad(ctx, view, a, torch.randn(rows).cuda(), torch.randn(rows).cuda(), out=None)
    out = torch.empty(4 * stride + cols, dtype=torch.float16, device="cuda").as_strided((rows, cols), (stride, 1))
    check_grad(ctx, view, a, torch.randn(rows).cuda(), torch.randn(rows).cuda(), out=out)


def test_two_streams_and_a_graph():
    from go_ai.engine import Context
    one, two = Context(9), Context(19)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    inputs = [make(3, 150_001, torch.float32, s, False) for s in (1, 2)]
    alone = [c.action_logprobs(x, a, top=20) for c, (x, _, a) in zip((one, two), inputs)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, s, (x, _, a) in zip((one, two), streams, inputs):
            with torch.cuda.stream(s):
                got.append(c.action_logprobs(x, a, top=20))
        torch.cuda.synchronize()
        for r, w in zip(got, alone):
            assert all(torch.equal(p, q) for p, q in zip(r, w))
    # captured: two graphs of one context, replayed in turn and with eager calls between them
    s = streams[0]
    graphs, outs, static = [], [], [x.clone() for x, _, _ in inputs]
    for x, (_, _, a) in zip(static, inputs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            one.action_logprobs(x, a, top=20)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                r = one.action_logprobs(x, a, top=20)
                d = one.action_logprobs_grad(x, a, r.lse, r.entropy, torch.ones(3, device="cuda"), None)
        graphs.append(graph)
        outs.append((r, d))
    for k in range(3):
        fresh = [torch.randn_like(x) for x in static]
        for x, f in zip(static, fresh):
            x.copy_(f)
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (r, d), f, (_, _, a) in zip(outs, fresh, inputs):
            w = one.action_logprobs(f, a, top=20)
            assert all(torch.equal(p, q) for p, q in zip(r, w))
            assert torch.equal(d, one.action_logprobs_grad(f, a, w.lse, w.entropy, torch.ones(3, device="cuda"), None))
    one.close()
    two.close()


@pytest.mark.parametrize("rows,cols", [(67_200_003, 3), (4_194_310, 1025)])
def test_more_rows_than_one_launch_takes(ctx, rows, cols):
    x = torch.zeros((rows, cols), dtype=torch.float16, device="cuda")
    far = torch.randn(20, cols).half().cuda()
    x[-20:] = far
    a = torch.zeros(rows, dtype=torch.int32, device="cuda")
    a[-20:] = torch.arange(20).cuda() % cols
    r = ctx.action_logprobs(x, a, top=2)
    want = definition(far, None, a[-20:], 1.0, 2)
    lse, ent, lp = bounds(want, cols)
    same(r.logp[-20:], want["logp"], lp(want["logp"]))
    same(r.lse[-20:], want["lse"], lse)
    same(r.entropy[-20:], want["entropy"], ent)
    assert np.array_equal(r.top_actions[-20:].cpu().numpy(), want["top_actions"])
    head = r.lse[:-20]
    assert (head - math.log(cols)).abs().max() <= 64 * U * (1 + math.log(cols)) and (r.top_actions[:-20] == torch.arange(2).cuda()).all()
    g = torch.ones(rows, device="cuda")
    d = ctx.action_logprobs_grad(x, a, r.lse, r.entropy, g, None)
    p = torch.from_numpy(want["p"])
    hot = torch.nn.functional.one_hot(a[-20:].long().cpu(), cols)
    assert (d[-20:].double().cpu() - (hot - p)).abs().max() <= 2.0 ** -11 + 1e-5
    assert (d[:-20, 0].float() - (1 - 1 / cols)).abs().max() <= 2.0 ** -11 + 1e-5
    assert (d[:-20, 1:].float() + 1 / cols).abs().max() <= 2.0 ** -11 / cols + 2.0 ** -24


def test_mask_bytes_and_action_types(ctx):
    """Any byte but 0 allows; actions of other integer types, values beyond 32 bits included, mean what they say."""
    x, valid, a = make(9, 82, torch.float32, 2, True)
    want = ctx.action_logprobs(x, a, valid=valid, top=4)
    for scaled in (valid * 255, valid * 128, valid.bool(), valid * torch.arange(1, 83, dtype=torch.uint8).cuda()):
        got = ctx.action_logprobs(x, a, valid=scaled, top=4)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert all(torch.equal(p, q) for p, q in zip(ctx.action_logprobs(x, a.long(), valid=valid, top=4), want))
    far = torch.tensor([2 ** 32 + 5, -2 ** 33, 3]).cuda()
    r = ctx.action_logprobs(x[:3], far)
    assert torch.isnan(r.logp[0]) and float(r.logp[1]) == 0.0 and float(r.logp[2]) < 0
    for bad in (torch.ones(9), torch.ones(9, dtype=torch.bool)):
        with pytest.raises(ValueError, match="integers"):
            ctx.action_logprobs(x, bad.cuda())


def test_same_bits_twice(ctx):
    for rows, cols in ((50, 362), (4, 150_001), (300, 9001)):
        x, valid, a = make(rows, cols, torch.bfloat16, 3, True)
        first = ctx.action_logprobs(x, a, valid=valid, top=30)
        for _ in range(3):
            again = ctx.action_logprobs(x, a, valid=valid, top=30)
            assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_refusals(ctx):
    x = torch.randn(3, 82).cuda()
    for bad, match in ((dict(top=65), "top"), (dict(top=-1), "top"), (dict(valid=torch.ones(3, 81).cuda() > 0), "valid"),
                       (dict(valid=torch.ones(3, 82).cuda()), "valid"), (dict(actions=[1, 2]), "actions")):
        with pytest.raises(ValueError, match=match):
            ctx.action_logprobs(x, **bad)
    with pytest.raises(ValueError, match="logits"):
        ctx.action_logprobs(x.int())
    with pytest.raises(ValueError, match="logits"):
        ctx.action_logprobs(x[0])
    from go_ai._hip import GoaiError
    for t in (0.0, -1.0, math.nan, 1e9):
        with pytest.raises(GoaiError, match="temperature"):
            ctx.action_logprobs(x, temperature=t)
    r = ctx.action_logprobs(x)
    with pytest.raises(GoaiError, match="needs actions"):
        ctx.action_logprobs_grad(x, None, r.lse, d_logp=torch.ones(3).cuda())
    with pytest.raises(GoaiError, match="needs entropy"):
        ctx.action_logprobs_grad(x, None, r.lse, d_entropy=torch.ones(3).cuda())
    with pytest.raises(ValueError, match="out"):
        ctx.action_logprobs_grad(x, None, r.lse, out=torch.empty(3, 82).half().cuda())
    with pytest.raises(ValueError, match="lse"):
        ctx.action_logprobs_grad(x, None, r.lse[:2])


def test_host_arrays(ctx):
    x = np.random.default_rng(0).standard_normal((4, 26))
    r = ctx.action_logprobs(x, np.array([0, 1, 2, 25]), valid=np.ones((4, 26), bool), top=2)
    want = definition(torch.from_numpy(x).float(), None, torch.tensor([0, 1, 2, 25]), 1.0, 2)
    assert np.allclose(r.logp.cpu().numpy(), want["logp"], atol=1e-5) and np.array_equal(r.top_actions.cpu().numpy(), want["top_actions"])
