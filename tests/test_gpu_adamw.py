"""go_ai.models.AdamW (goai_adamw_*): a step over many tensors at once, moments in 32 and in 8 bits, against the update's
definition in float64.  The reference trains with torch.optim.Adam (train.py:52), which goai_train_step keeps."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SHAPES = [(1,), (3,), (255,), (256,), (257,), (0,), (2048,), (2049,), (7, 13), (5000,), (1, 1), (64, 33, 3, 3), (70001,)]


def tensors(shapes, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    dtypes = dtype if isinstance(dtype, list) else [dtype] * len(shapes)
    return [(scale * torch.randn(s, generator=g)).to(d).cuda() for s, d in zip(shapes, dtypes)]


def f64(xs):
    return [x.detach().double().cpu().numpy() for x in xs]


def reference(p, g, m, v, t, lr, b1, b2, eps, decay, max_norm):
    """One step in float64 over lists; also the bound of a float32 step's error in p, m, v."""
    norm = math.sqrt(sum(float((x * x).sum()) for x in g if x is not None))
    k = min(1.0, max_norm / norm) if max_norm and norm > 0 else 1.0
    out = []
    for p0, g0, m0, v0, d in zip(p, g, m, v, decay):
        if g0 is None:
            out.append((p0, m0, v0, 0 * p0, 0 * m0, 0 * v0))
            continue
        gk = k * g0
        m1 = b1 * m0 + (1 - b1) * gk
        # float32 holds squares up to 2^128 (its largest number and half a step): a |g| from 2^64 on has an infinite one, and the
        # update is m / inf = 0
        square = gk * gk
        square[square >= 2.0 ** 128 * (1 - 2.0 ** -25)] = math.inf
        v1 = b2 * v0 + (1 - b2) * square
        den = np.sqrt(v1 / (1 - b2 ** t)) + eps
        upd = lr / (1 - b1 ** t) * m1 / den
        # each product and sum rounds once, the constants once, the coefficient once
        dm = 5 * U * (np.abs(b1 * m0) + np.abs((1 - b1) * gk))
        dv = np.where(np.isinf(v1), 0, 7 * U * v1) + 2.0 ** -140
        # the root halves v's relative error, one rounding each for root, correction, product, eps, sum, quotient, product
        dupd = lr / (1 - b1 ** t) * (dm / den + np.abs(m1) / den * 14 * U)
        dp = dupd + 3 * U * (np.abs(p0) + np.abs(upd)) + 2.0 ** -140
        out.append((p0 * (1 - lr * d) - upd, m1, v1, dp, dm + 2.0 ** -140, dv))
    return norm, out


def close(got, want, tol, what=""):
    got, tol = got.double().cpu().numpy(), np.broadcast_to(tol, want.shape)
    there = np.isfinite(want)
    assert np.array_equal(got[~there], want[~there]), what
    off = np.abs(got[there] - want[there]) - tol[there]
    assert not np.isnan(off).any() and off.max(initial=-1) <= 0, (what, off.max())


def unpack(opt):
    m, v = opt.moments()
    return opt._split(m), opt._split(v)


def mean_bound(m, dm):
    """An e4m3 code of a block: half a step is 2^-4 of the value, or half of the smallest step 2^-9 of scale = largest / 448."""
    flat = m.reshape(-1)
    n = -(-flat.size // 256) * 256
    big = np.abs(np.pad(flat, (0, n - flat.size)).reshape(-1, 256)).max(1, initial=0).repeat(256)[:flat.size].reshape(m.shape)
    return dm + np.maximum(2.0 ** -4 * np.abs(m), 2.0 ** -10 / 448 * big) * (1 + 2.0 ** -18) + 8 * U * np.abs(m) + np.where(big < 2.0 ** -99, big, 0)


def root_bound(v, dv):
    """A code of the root: half a step 2^-5 of it, at least code 1 = 1.125 * 2^-16 of the block's largest when it is not zero."""
    r = np.sqrt(v)
    flat = r.reshape(-1)
    n = -(-flat.size // 256) * 256
    big = np.pad(flat, (0, n - flat.size)).reshape(-1, 256).max(1, initial=0).repeat(256)[:flat.size].reshape(r.shape)
    dr = np.where(r > 0, dv / np.maximum(2 * r, 1e-300) + 8 * U * r, 0) + 2.0 ** -5 * r * (1 + 2.0 ** -18)
    return np.maximum(dr, np.where((r > 0) & (r < 1.2 * 2.0 ** -16 * big), 1.2 * 2.0 ** -16 * big, 0)) + np.where(big < 2.0 ** -99, big, 0)


def run_steps(params, grads_of, steps, *, bits, max_norm=0.0, decay=0.01, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, start=None, opt=None, **kw):
    from go_ai.models import AdamW
    n = len(params)
    opt = opt or AdamW(params, lr=lr, betas=betas, eps=eps, weight_decay=decay, state_bits=bits, max_norm=max_norm, **kw)
    if start is not None:
        opt.load_moments(*start)
    decays = np.float32(decay if isinstance(decay, list) else [decay] * n).astype(np.float64)
    for k in range(steps):
        grads = grads_of(k)
        p0 = f64(params)
        m0, v0 = [f64(x) for x in unpack(opt)]
        g0 = [None if g is None else g.double().cpu().numpy() for g in grads]
        opt.step(grads)
        torch.cuda.synchronize()
        norm, want = reference(p0, g0, m0, v0, opt.steps, lr, betas[0], betas[1], eps, decays, max_norm)
        if max_norm:
            assert abs(float(opt.norm) - norm) <= 2 * U * norm
        m1, v1 = unpack(opt)
        for i, (p, m, v, dp, dm, dv) in enumerate(want):
            if g0[i] is None:
                assert np.array_equal(f64([params[i]])[0], p) and np.array_equal(f64([m1[i]])[0], m)
                continue
            dt = params[i].dtype
            close(params[i], p, dp + HALF[dt] * (np.abs(p) + dp) + TINY[dt], ("p", i))
            if bits == 32:
                close(m1[i], m, dm, ("m", i))
                close(v1[i], v, dv, ("v", i))
            else:
                close(m1[i], m, mean_bound(m, dm), ("m", i))
                # a scale is the largest root of its block: an infinite one makes the block's other roots that are not zero infinite
                blocks = np.pad(v.reshape(-1), (0, -v.size % 256)).reshape(-1, 256)
                blocks[np.isinf(blocks).any(1, keepdims=True) & (blocks > 0)] = math.inf
                v = blocks.reshape(-1)[:v.size].reshape(v.shape)
                close(v1[i].sqrt(), np.sqrt(v), root_bound(v, dv), ("r", i))
                # no root becomes 0 but those whose square float32 cannot hold: below 2^-150, half its smallest number (the
                # products g g (1 - beta2) may lose a factor of two on the way there)
                assert ((v1[i] > 0).cpu().numpy() | (v <= 2.0 ** -148)).all()
    return opt


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,gdtype", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (BF16, F16), (F16, F16), (F16, F32),
                                          (F16, BF16)])
def test_steps(bits, dtype, gdtype):
    params = tensors(SHAPES, dtype, 1, 0.1)
    run_steps(params, lambda k: tensors(SHAPES, gdtype, 10 + k), 3, bits=bits, grad_dtype=gdtype, max_norm=1.0 if dtype == F32 else 0.0,
              decay=[0.05 if len(s) > 1 else 0.0 for s in SHAPES])


@pytest.mark.parametrize("bits", [32, 8])
def test_mixed_types_and_late_steps(bits):
    dtypes = [(F32, BF16, F16)[i % 3] for i in range(len(SHAPES))]
    gdtypes = [(F32, F16, F32, BF16)[i % 4] for i in range(len(SHAPES))]
    params = tensors(SHAPES, dtypes, 2, 0.1)
    m = tensors(SHAPES, F32, 3, 1e-3)
    v = [x.square() for x in tensors(SHAPES, F32, 4, 1e-2)]
    run_steps(params, lambda k: tensors(SHAPES, gdtypes, 20 + k, 1e-2), 2, bits=bits, grad_dtype=gdtypes, start=(m, v, 20000), max_norm=0.5,
              betas=(0.95, 0.99), eps=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_wide_range_of_gradients(bits):
    """Sizes over many decades within a block, zeros, subnormals, blocks that are all zero or below the smallest scale."""
    g = torch.Generator().manual_seed(9)
    n = 256 * 9 + 17
    x = torch.randn(n, generator=g) * torch.exp(6 * torch.randn(n, generator=g))
    x[:256] = 0
    x[256:512] = torch.randn(256, generator=g) * 2.0 ** -110
    x[512:768] *= 2.0 ** -100
    x[768:1024:3] = 0
    x[1024:1280] = torch.randn(256, generator=g) * 2.0 ** -140
    x[1280:1536] *= 1e15
    run_steps([torch.randn(n, generator=g).cuda()], lambda k: [x.cuda()], 3, bits=bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_against_torch(bits):
    """Against torch.optim.AdamW itself in float64 over five steps (32 bits; with 8 the first step, which starts from zeros)."""
    shapes = SHAPES[:6] + SHAPES[7:]
    params = tensors(shapes, F32, 5)
    theirs = [p.double().cpu().clone().requires_grad_(True) for p in params]
    other = torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.1)
    from go_ai.models import AdamW
    opt = AdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits)
    for k in range(5 if bits == 32 else 1):
        grads = tensors(shapes, F32, 50 + k)
        opt.step(grads)
        for t, g in zip(theirs, grads):
            t.grad = g.double().cpu()
        other.step()
        for p, t in zip(params, theirs):
            # per step 16 roundings of the update (lr) and 3 of the parameter; float32(0.1) for the decay
            assert torch.allclose(p.double().cpu(), t.detach(), rtol=4e-7 * (k + 1), atol=1e-2 * 4e-6 * (k + 1))


def test_unaligned_views_and_their_neighbours():
    """Parameters and gradients as views of one buffer at odd offsets; the numbers between them are nobody's."""
    for dtype in (F32, BF16):
        sizes = [1, 5, 300, 2047, 6001, 2]
        buf = torch.full((sum(sizes) + 3 * len(sizes) + 1,), 7.0, dtype=dtype).cuda()
        gbuf = torch.randn(len(buf)).to(dtype).cuda()
        at, views, grads, inside = 1, [], [], torch.zeros(len(buf), dtype=torch.bool)
        for s in sizes:
            views.append(buf[at:at + s])
            grads.append(gbuf[at:at + s])
            inside[at:at + s] = True
            at += s + 3
        for bits in (32, 8):
            run_steps(views, lambda k: grads, 2, bits=bits, max_norm=1.0)
        assert (buf.cpu()[~inside] == 7.0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients(bits):
    shapes = [(300,), (5000,), (7,)]
    params = tensors(shapes, F32, 1)
    some = tensors(shapes, F32, 2)
    run_steps(params, lambda k: [some[0], None, some[2]] if k % 2 else [None, some[1], some[2]], 4, bits=bits, max_norm=0.1)
    opt = run_steps(params, lambda k: [None, None, None], 1, bits=bits, max_norm=0.1)
    assert float(opt.norm) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_norm_that_is_not_finite_skips_the_step(bits, bad):
    from go_ai.models import AdamW
    params, grads = tensors([(300,), (9000,)], F32, 1), tensors([(300,), (9000,)], F32, 2)
    opt = AdamW(params, state_bits=bits, max_norm=1.0)
    opt.step(grads)
    before = [x.clone() for x in params] + [x.clone() for x in opt.moments()]
    grads[1][8999] = bad
    opt.step(grads)
    after = params + list(opt.moments())
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    assert not math.isfinite(float(opt.norm))


def test_norms_of_huge_gradients_are_finite():
    from go_ai.models import AdamW
    p = [torch.zeros(1000).cuda()]
    opt = AdamW(p, max_norm=1.0, weight_decay=0.0)
    g = torch.full((1000,), 3e37).cuda()
    opt.step([g])
    assert abs(float(opt.norm) / (3e37 * math.sqrt(1000)) - 1) < 1e-6 or float(opt.norm) == math.inf
    assert torch.isfinite(p[0]).all() and (p[0] < 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_launch_takes(bits):
    shapes = [(1 + 37 * i % 700,) for i in range(600)]
    run_steps(tensors(shapes, F32, 1), lambda k: tensors(shapes, F32, 2 + k), 2, bits=bits, max_norm=0.3)


def test_codes_and_their_values():
    """Every code comes back as the value it was made from; values between two codes go to the nearer one, ties to the even."""
    from go_ai.models import AdamW
    m_codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    m_codes = torch.where(torch.isnan(m_codes), 448.0, m_codes)
    r_codes = ((torch.arange(256) + 1777) << 19).to(torch.int32).view(torch.float32)
    r_codes[0] = 0
    for scale in (1.0, 2.0 ** -40, 2.0 ** 30):                # powers of two: scaling is exact
        opt = AdamW([torch.zeros(256).cuda()], state_bits=8)
        # codes of the root as v = r^2 with an exact root: r has 5 significant bits, r^2 ten
        opt.load_moments([(m_codes * scale).cuda()], [(r_codes * scale).square().cuda()], 3)
        m, v = opt.moments()
        close(m, (m_codes * scale).double().numpy(), 2 * U * np.abs(m_codes.numpy()) * scale)
        assert torch.equal(v.cpu().sqrt(), r_codes * scale) and opt.steps == 3
    mid = (r_codes[1:255] + r_codes[2:256]) / 2
    opt = AdamW([torch.zeros(256).cuda()], state_bits=8)
    r = torch.cat([mid, torch.ones(2)])
    opt.load_moments([torch.zeros(256).cuda()], [r.square().cuda()], 0)
    got = opt.moments()[1].cpu().sqrt()
    even = torch.where(torch.arange(1, 255) % 2 == 1, r_codes[2:256], r_codes[1:255])       # 1777 is odd: an odd code's bits are even ...
    even = torch.where((torch.arange(1, 255) + 1777) % 2 == 0, r_codes[1:255], r_codes[2:256])
    assert torch.equal(got[:254], even)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict(bits):
    from go_ai.models import AdamW
    params = tensors(SHAPES, F32, 1)
    opt = AdamW(params, state_bits=bits)
    for k in range(2):
        opt.step(tensors(SHAPES, F32, 5 + k))
    saved = opt.state_dict()
    copies = [p.clone() for p in params]
    again = AdamW(copies, state_bits=bits)
    again.load_state_dict(saved)
    assert again.steps == 2
    for a, b in zip(again.moments(), opt.moments()):
        if bits == 32:
            assert torch.equal(a, b)
        else:                                       # a code's value over a block's scale rounds to that code again
            assert torch.allclose(a, b, rtol=8 * U, atol=0)
    g = tensors(SHAPES, F32, 9)
    opt.step(g)
    again.step(g)
    for a, b in zip(copies, params):
        assert torch.equal(a, b) if bits == 32 else torch.allclose(a, b, rtol=1e-6, atol=1e-8)


@pytest.mark.parametrize("bits", [32, 8])
def test_same_bits_on_another_stream(bits):
    from go_ai.models import AdamW
    grads = [tensors(SHAPES, F32, 5 + k) for k in range(3)]
    runs = []
    for s in (None, torch.cuda.Stream(), None):
        params = tensors(SHAPES, F32, 1)
        torch.cuda.synchronize()
        opt = AdamW(params, state_bits=bits, max_norm=0.7)
        with torch.cuda.stream(s if s is not None else torch.cuda.current_stream()):
            for g in grads:
                opt.step(g)
        torch.cuda.synchronize()
        runs.append(params + list(opt.moments()))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits):
    from go_ai.models import AdamW
    shapes = SHAPES
    grads = [tensors(shapes, F32, 5 + k) for k in range(5)]
    eager_p, graph_p = tensors(shapes, F32, 1), tensors(shapes, F32, 1)
    eager, opt = [AdamW(p, state_bits=bits, max_norm=0.7) for p in (eager_p, graph_p)]
    static = [g.clone() for g in grads[0]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    opt.advance()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            opt.step(static, captured=True)
    assert opt.steps == 1
    torch.cuda.synchronize()
    for k, g in enumerate(grads):
        if k:
            opt.lr = eager.lr = 1e-3 * (k + 1)
            opt.advance()
        for a, b in zip(static, g):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager.step(g)
        torch.cuda.synchronize()
        assert opt.steps == eager.steps == k + 1
        assert all(torch.equal(a, b) for a, b in zip(eager_p + list(eager.moments()), graph_p + list(opt.moments()))), k


def test_a_capture_without_scalars_is_refused():
    from go_ai._hip import GoaiError
    from go_ai.models import AdamW
    p, g = tensors([(300,)], F32, 1), tensors([(300,)], F32, 2)
    before = p[0].clone()
    opt = AdamW(p)
    with pytest.raises(RuntimeError, match="advance"):
        opt.step(g, captured=True)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            with pytest.raises(GoaiError, match="scalars"):
                opt.step(g)
            g[0] + 1
    assert opt.steps == 0 and torch.equal(p[0], before)


@pytest.mark.parametrize("bits,dtype", [(8, BF16), (32, F32)])
def test_long_tensors(bits, dtype):
    """Offsets beyond 2^31 elements: the far end is updated, and by the right gradient."""
    from go_ai.models import AdamW
    n = 2 ** 31 + 1500
    p = [torch.zeros(n, dtype=dtype, device="cuda"), torch.zeros(700, dtype=dtype, device="cuda")]
    g = [torch.zeros(n, dtype=dtype, device="cuda"), torch.ones(700, dtype=dtype, device="cuda")]
    g[0][-1000:] = torch.arange(1000).to(dtype).cuda() + 1
    g[0][:100] = -1.0
    opt = AdamW(p, lr=0.5, weight_decay=0.0, state_bits=bits)
    opt.step(g)
    tol = 0.5 * (HALF[dtype] + 32 * U)
    assert (p[0][-1000:].float() + 0.5).abs().max() <= tol and (p[0][:100].float() - 0.5).abs().max() <= tol
    assert (p[1].float() + 0.5).abs().max() <= tol
    assert not p[0][100:-1000].any()
    m, v = opt.moments()
    far = m[n - 1000:n].double().cpu().numpy()
    want = 0.1 * (np.arange(1000) + 1) if dtype == F32 else 0.1 * (torch.arange(1000).to(dtype).double().numpy() + 1)
    want = 0.1 * g[0][-1000:].double().cpu().numpy()
    assert (np.abs(far - want) <= 2.0 ** -4 * want + 1000 / 448 * 2.0 ** -10 * 0.1).all()
    assert not m[100:n - 1000].any() and not m[n:opt.offsets[1]].any()


def test_refusals():
    from go_ai._hip import GoaiError
    from go_ai.models import AdamW
    p = tensors([(4, 6), (30,)], F32, 1)
    for bad in (dict(lr=-1.0), dict(lr=math.nan), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=0.0), dict(state_bits=16),
                dict(max_norm=-1.0), dict(max_norm=math.nan), dict(weight_decay=[0.1]), dict(grad_dtype=torch.float64),
                dict(grad_dtype=[F32])):
        with pytest.raises(ValueError):
            AdamW(p, **bad)
    with pytest.raises(GoaiError, match="weight decay"):
        AdamW(p, weight_decay=-0.5)
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([p[0].t()])
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([torch.zeros(3, dtype=torch.float64).cuda()])
    with pytest.raises(ValueError, match="host"):
        AdamW([p[0], torch.zeros(3)])
    with pytest.raises(GoaiError, match="overlap"):
        AdamW([p[1][:20], p[1][10:]])
    with pytest.raises(GoaiError, match="overlap"):
        AdamW([p[1], p[1]])
    opt = AdamW(p)
    for g in ([p[0]], [p[0], p[1][:29]], [p[0].half(), p[1]], [p[0], p[1].cpu()], [torch.zeros(6, 4).cuda().t(), p[1]], [p[1], p[0]]):
        with pytest.raises(ValueError):
            opt.step(g)
    with pytest.raises(ValueError):
        opt.load_moments([p[0]], [p[0]], 1)
    with pytest.raises(ValueError):
        opt.load_moments(p, p, -1)
    assert opt.steps == 0
    loose = AdamW(None)
    with pytest.raises(RuntimeError, match="no parameters yet"):
        loose.step([])


def test_parameters_of_another_device_than_the_context():
    """The second GPU need not exist: a context that says it is there is enough."""
    from types import SimpleNamespace
    from go_ai.models import AdamW
    p = tensors([(300,)], F32, 1)
    with pytest.raises(ValueError, match="context"):
        AdamW(p, ctx=SimpleNamespace(device=torch.device("cuda", 1)))
    with pytest.raises(ValueError, match="context"):
        AdamW().bind([torch.zeros(300)], SimpleNamespace(device=torch.device("cuda", 0)))
    with pytest.raises(ValueError, match="GPU"):
        AdamW().bind([torch.zeros(300)])


def test_a_bound_optimiser_is_not_copied():
    import copy
    import pickle
    from go_ai.models import AdamW
    p = tensors([(300,), (7,)], F32, 1)
    opt = AdamW(p)
    for f in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="state_dict"):
            f(opt)


def test_replaced_parameter_memory():
    from go_ai.models import AdamW
    p, g = tensors([(300,), (7,)], F32, 1), tensors([(300,), (7,)], F32, 2)
    opt = AdamW(p)
    opt.step(g)
    old = p[0].data
    p[0].data = old.clone()
    before = old.clone()
    with pytest.raises(RuntimeError, match="replaced"):
        opt.step(g)
    assert opt.steps == 1 and torch.equal(old, before) and torch.equal(p[0], before)
    p[0].data = old
    opt.step(g)
    assert opt.steps == 2 and not torch.equal(p[0], before)
    opt.bind(p)
    assert opt.steps == 0 and not any(m.any() for m in opt.moments())
