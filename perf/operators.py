"""The workloads of the learning operators: log probabilities of given actions (with entropy and the best alternatives), their
gradient, and the AdamW step over many tensors with its moments in 32 or in 8 bits.

Each case is one call as a user's program makes it.  Where `own` is false, `run` computes it from elementary torch operations
in 32 bits (the gradient's norm in 64); where it is true, it calls go_ai.engine.Context and go_ai.models.AdamW.
`exact` computes the same from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256                # elements that share one scale of an 8-bit moment; tensors start at multiples of it
SMALLEST = 2.0 ** -100     # a block of moments below this is held as zeros
LEVEL0 = 1777              # 8-bit code c of a root second moment, c = 1..255: the float32 with the bits (c + LEVEL0) << 19


# ---- cases ----------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one lock-step move of 1024 self-play games on 9x9: the played moves' log probabilities, five alternatives each
        dict(name="logprobs 1024 x 82", op="logprobs", rows=1024, cols=82, dtype="f32", masked=True, temperature=1.0, top=5),
        # a single 19x19 position under analysis: only latency counts
        dict(name="logprobs 1 x 362", op="logprobs", rows=1, cols=362, dtype="f32", masked=True, temperature=1.0, top=10),
        # a replay of 19x19 positions evaluated at once, logits kept in bfloat16
        dict(name="logprobs 65536 x 362", op="logprobs", rows=65536, cols=362, dtype="bf16", masked=True, temperature=1.0, top=8),
        # a few rows over a large vocabulary: one decoding step
        dict(name="logprobs 5 x 128001", op="logprobs", rows=5, cols=128001, dtype="f16", masked=False, temperature=0.7, top=20),
        # many rows over a large vocabulary: scoring given text
        dict(name="logprobs 1500 x 50021", op="logprobs", rows=1500, cols=50021, dtype="f32", masked=False, temperature=1.0, top=1),
        # the reference's training batch of 32 positions on 9x9
        dict(name="logprobs_grad 32 x 82", op="logprobs_grad", rows=32, cols=82, dtype="f32", masked=True, temperature=1.0),
        # a large batch of 19x19 positions
        dict(name="logprobs_grad 32768 x 362", op="logprobs_grad", rows=32768, cols=362, dtype="bf16", masked=True, temperature=1.0),
        # a training batch over a large vocabulary
        dict(name="logprobs_grad 2000 x 32003", op="logprobs_grad", rows=2000, cols=32003, dtype="f32", masked=False, temperature=1.3),
        # the 9x9 actor-critic net of three blocks (42 tensors, 1 M parameters), one step
        dict(name="adamw 9x9 net, 32 bits", op="adamw", board=9, blocks=3, tensors=0, small=0, large=0, dtype="f32", grad_dtype="f32",
             bits=32, max_norm=0.0, t=1),
        # the 19x19 net of ten blocks, moments in 8 bits, gradients clipped by their global norm
        dict(name="adamw 19x19 net, 8 bits", op="adamw", board=19, blocks=10, tensors=0, small=0, large=0, dtype="f32",
             grad_dtype="f32", bits=8, max_norm=1.0, t=1000),
        # large models: tensors of 257 to 25 M elements
        dict(name="adamw 97 M, 32 bits", op="adamw", board=0, blocks=0, tensors=24, small=257, large=40000001, dtype="f32",
             grad_dtype="f32", bits=32, max_norm=1.0, t=20000),
        dict(name="adamw 250 M, 8 bits", op="adamw", board=0, blocks=0, tensors=40, small=129, large=75000001, dtype="bf16",
             grad_dtype="bf16", bits=8, max_norm=0.0, t=20000),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_grad", "adamw", "adamw"])
    if op != "adamw":
        if rng.random() < 0.5:                                   # the policies of the five board sizes
            cols = rng.choice([26, 50, 82, 170, 362])
            rows = _spread(rng, 1, 25_000_000 // cols)
        else:
            cols = _spread(rng, 1, 200_000)
            rows = _spread(rng, 1, max(1, min(100_000, 60_000_000 // cols)))
        case = dict(op=op, rows=rows, cols=cols, dtype=rng.choice(list(TYPES)), masked=rng.random() < 0.6,
                    temperature=rng.choice([1.0, 1.0, 0.5, 0.8, 1.5]))
        if op == "logprobs":
            case["top"] = min(cols, rng.choice([0, 1, 3, 5, 10, 20, 64]))
        return case
    if rng.random() < 0.4:
        board, blocks, tensors, small, large = rng.choice([5, 7, 9, 13, 19]), rng.randint(1, 12), 0, 0, 0
    else:
        board, blocks, tensors, small = 0, 0, rng.randint(1, 60), _spread(rng, 1, 3000)
        large = small + _spread(rng, 1, 20_000_000 // max(1, tensors // 4))
    return dict(op=op, board=board, blocks=blocks, tensors=tensors, small=small, large=large, dtype=rng.choice(["f32", "f32", "bf16", "f16"]),
                grad_dtype=rng.choice(["f32", "bf16", "f16"]), bits=rng.choice([8, 32]), max_norm=rng.choice([0.0, 1.0]),
                t=rng.choice([1, 10, 1000, 100000]))


def _shapes(case):
    """The tensors of an AdamW case: an actor-critic net's, or a geometric run of sizes, matrices and vectors in turn."""
    if case["board"]:
        cells, c = case["board"] ** 2, 128
        norm = lambda n: [(n,), (n,), (n,)]  # noqa: E731   (convolution bias, BatchNorm weight and bias)
        return ([(c, 6, 3, 3)] + norm(c) + ([(c, c, 3, 3)] + norm(c)) * (2 * case["blocks"]) + [(2, c, 1, 1)] + norm(2)
                + [(cells + 1, 2 * cells), (cells + 1,), (1, c, 1, 1)] + norm(1) + [(256, cells), (256,), (1, 256), (1,)])
    n, a, b = case["tensors"], case["small"], case["large"]
    sizes = [int(round(a * (b / a) ** (i / max(1, n - 1)))) for i in range(n)]
    return [(s,) if i % 2 else (1, s) for i, s in enumerate(sizes)]


def work(case):
    if case["op"] != "adamw":
        cells, e = case["rows"] * case["cols"], TYPES[case["dtype"]].itemsize
        mask = cells if case["masked"] else 0
        if case["op"] == "logprobs":
            return dict(bytes=cells * e + mask + case["rows"] * (16 + 8 * case["top"]), flops=6 * cells)
        return dict(bytes=2 * cells * e + mask + 20 * case["rows"], flops=8 * cells)
    n = sum(math.prod(s) for s in _shapes(case))
    pe, ge = TYPES[case["dtype"]].itemsize, TYPES[case["grad_dtype"]].itemsize
    # parameter, gradient, two moments; moments in 8 bits also come back as the values they stand for
    state = 16 if case["bits"] == 32 else 4 + 8
    return dict(bytes=n * (2 * pe + ge + state), flops=14 * n)


# ---- inputs ---------------------------------------------------------------------------------------------------------------

def _policy_inputs(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    rows, cols = case["rows"], case["cols"]
    logits = (3 * torch.randn((rows, cols), generator=g, device=DEV)).to(TYPES[case["dtype"]])
    valid = None
    actions = torch.randint(0, cols, (rows,), generator=g, device=DEV, dtype=torch.int32)
    if case["masked"]:
        valid = (torch.rand((rows, cols), generator=g, device=DEV) < 0.6).to(torch.uint8)
        valid[:, -1] = 1                                                          # passing is always allowed
        # a played action is a legal one: the next legal column at or after a random one
        at = torch.arange(cols, device=DEV, dtype=torch.int32)
        legal = torch.where(valid.bool(), at, cols - 1)
        actions = torch.where(at >= actions[:, None], legal, cols - 1).amin(1).to(torch.int32)
        if rows > 50:
            valid[::97] = 0                                                       # slots without a game: nothing is legal
    if rows > 50:
        actions[::61] = -1                                                        # positions without a recorded action
    return g, logits, valid, actions


def prepare(case, seed):
    s = {"case": case}
    if own:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-ai_amd"))
        from go_ai.engine import Context
        from go_ai.models import AdamW
    if case["op"] != "adamw":
        g, s["logits"], s["valid"], s["actions"] = _policy_inputs(case, seed)
        if case["op"] == "logprobs_grad":
            # what the forward pass left, and a policy-gradient loss with an entropy bonus
            _, s["entropy"], s["lse"] = _log_probs(s["logits"], s["valid"], s["actions"], case["temperature"])[:3]
            s["d_logp"] = -torch.randn(case["rows"], generator=g, device=DEV) / case["rows"]
            s["d_entropy"] = torch.full((case["rows"],), -0.01 / case["rows"], device=DEV)
        if own:
            s["ctx"] = Context(9, 0)
        return s
    g = torch.Generator(DEV).manual_seed(seed)
    shapes = _shapes(case)
    sizes = [math.prod(x) for x in shapes]
    blocks = [-(-n // BLOCK) for n in sizes]
    total = sum(blocks) * BLOCK
    starts = [BLOCK * sum(blocks[:i]) for i in range(len(sizes))]
    decays = [0.01 if len(x) > 1 else 0.0 for x in shapes]
    count = torch.tensor(blocks, device=DEV)
    # elements behind a tensor's end, up to the next one's start, belong to nobody: zeros
    ends = torch.repeat_interleave(torch.tensor([a + n for a, n in zip(starts, sizes)], device=DEV), count)
    inside = torch.arange(total, device=DEV).view(-1, BLOCK) < ends[:, None]
    rand = lambda: torch.randn((total // BLOCK, BLOCK), generator=g, device=DEV) * inside  # noqa: E731
    # blocks of gradients differ in size by some decades, as layers do
    size = torch.exp(2 * torch.randn((total // BLOCK, 1), generator=g, device=DEV)) * 1e-3
    s["p"] = (rand() * 0.05).to(TYPES[case["dtype"]])
    s["g"] = (rand() * size).to(TYPES[case["grad_dtype"]])
    first = case["t"] == 1
    m = torch.zeros((total // BLOCK, BLOCK), device=DEV) if first else rand() * size * 0.3
    v = torch.zeros((total // BLOCK, BLOCK), device=DEV) if first else (rand() * size).square() + (size * 0.1).square() * inside
    views = lambda flat: [flat.view(-1)[a:a + n].view(x) for a, n, x in zip(starts, sizes, shapes)]  # noqa: E731
    if own:
        s["grads"] = views(s["g"])
        s["opt"] = AdamW(views(s["p"]), lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=decays, state_bits=case["bits"],
                         max_norm=case["max_norm"], grad_dtype=TYPES[case["grad_dtype"]])
        s["opt"].load_moments(views(m), views(v), steps=case["t"] - 1)
        return s
    s["t"] = case["t"] - 1
    s["decay"] = torch.repeat_interleave(torch.tensor(decays, device=DEV), count)[:, None]
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        s["m"], s["m_scale"] = _pack_mean(m)
        s["v"], s["v_scale"] = _pack_root(v.sqrt())
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------------

def _log_probs(logits, valid, actions, temperature, top=0):
    """log p of the given actions, entropy, log of the sum, and the `top` best columns (ties: the lower one) with their log p.
    Columns that are not valid, or whose logit is -inf, do not exist; a row without any has entropy 0, log p -inf and no
    alternatives (-1)."""
    x = logits.float()
    x = x.masked_fill(valid == 0, -math.inf) if valid is not None else x
    some = (x > -math.inf).any(1)
    s = x * (1 / temperature)
    peak = torch.where(some, s.amax(1), 0.0)[:, None]
    e = torch.exp(s - peak)
    total = e.sum(1)
    lse = torch.log(total) + peak[:, 0]
    off = torch.where(e > 0, s - peak, 0.0)
    entropy = torch.where(some, torch.log(total) - (e * off).sum(1) / total, 0.0)
    lp = lambda v: torch.where(some[:, None], v - peak - torch.log(total)[:, None], -math.inf)  # noqa: E731
    given = lp(s.gather(1, actions.clamp(min=0).long()[:, None]))[:, 0]
    given = torch.where(actions < 0, 0.0, given)
    if not top:
        return given, entropy, lse, None, None
    order, at = torch.sort(x, dim=1, descending=True, stable=True)
    none = order[:, :top] == -math.inf
    return given, entropy, lse, at[:, :top].masked_fill(none, -1).to(torch.int32), lp(order[:, :top] * (1 / temperature))


def _log_probs_grad(s):
    """d / d logits of sum(d_logp * log p[action]) + sum(d_entropy * entropy)."""
    case, logits, actions = s["case"], s["logits"], s["actions"]
    x = logits.float()
    x = x.masked_fill(s["valid"] == 0, -math.inf) if s["valid"] is not None else x
    some = (x > -math.inf).any(1, keepdim=True)
    lp = x * (1 / case["temperature"]) - torch.where(some, s["lse"][:, None], 0.0)
    p = torch.exp(lp)
    given = torch.where(actions < 0, 0.0, s["d_logp"])[:, None]
    at = torch.arange(case["cols"], device=DEV)
    d = given * ((at == actions[:, None]).float() - p)
    d = d - s["d_entropy"][:, None] * p * (torch.where(p > 0, lp, 0.0) + s["entropy"][:, None])
    return torch.where(x > -math.inf, d * (1 / case["temperature"]), 0.0).to(logits.dtype)


def _pack_mean(m):
    """First moments in 8 bits: e4m3 codes of m / scale, scale = largest of the block / 448."""
    big = m.abs().amax(1, keepdim=True)
    held = big >= SMALLEST
    code = (m * torch.where(held, big.reciprocal() * 448.0, 0.0)).to(torch.float8_e4m3fn)
    return code, torch.where(held, big * (1 / 448.0), 0.0)


def _pack_root(r):
    """Roots of second moments in 8 bits: four exponent and four fraction bits below the block's largest, rounded to the nearest
    (ties to even); what is not zero stays above zero."""
    big = r.amax(1, keepdim=True)
    held = big >= SMALLEST
    bits = (r * torch.where(held, big.reciprocal(), 0.0)).view(torch.int32)
    code = ((bits + 0x3FFFF + ((bits >> 19) & 1)) >> 19) - LEVEL0
    code = torch.where((r > 0) & held, code.clamp(1, 255), 0).to(torch.uint8)
    return code, torch.where(held, big, 0.0)


def _mean_of(code, scale):
    return code.float() * scale


def _root_of(code, scale):
    return torch.where(code > 0, (code.to(torch.int32) + LEVEL0) << 19, 0).view(torch.float32) * scale


def _adamw(s):
    case = s["case"]
    s["t"] += 1
    lr, b1, b2, eps = 1e-3, 0.9, 0.999, 1e-8
    g, p = s["g"].float(), s["p"].float()
    norm = None
    if case["max_norm"]:
        norm = s["g"].double().square().sum().sqrt()
        g = g * torch.clamp(case["max_norm"] / norm, max=1.0).float()
    if case["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m, v = _mean_of(s["m"], s["m_scale"]), _root_of(s["v"], s["v_scale"]).square()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    root = v.sqrt()
    p = p * (1 - lr * s["decay"].double()).float() - (m / (root * (1 / math.sqrt(1 - b2 ** s["t"])) + eps)) * (lr / (1 - b1 ** s["t"]))
    s["p"].copy_(p)
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"params": s["p"], "exp_avg": s["m"], "exp_avg_sq": s["v"], "norm": None if norm is None else norm.float()}
    s["m"], s["m_scale"] = _pack_mean(m)
    s["v"], s["v_scale"] = _pack_root(root)
    return {"params": s["p"], "exp_avg": _mean_of(s["m"], s["m_scale"]), "exp_avg_sq": _root_of(s["v"], s["v_scale"]).square(),
            "norm": None if norm is None else norm.float()}


def run(s):
    case = s["case"]
    if case["op"] == "logprobs":
        if own:
            r = s["ctx"].action_logprobs(s["logits"], s["actions"], valid=s["valid"], temperature=case["temperature"], top=case["top"])
            return dict(logp=r.logp, entropy=r.entropy, lse=r.lse, top_actions=r.top_actions, top_logp=r.top_logp)
        return dict(zip(("logp", "entropy", "lse", "top_actions", "top_logp"),
                        _log_probs(s["logits"], s["valid"], s["actions"], case["temperature"], case["top"])))
    if case["op"] == "logprobs_grad":
        if own:
            return s["ctx"].action_logprobs_grad(s["logits"], s["actions"], s["lse"], s["entropy"], s["d_logp"], s["d_entropy"],
                                                 valid=s["valid"], temperature=case["temperature"])
        return _log_probs_grad(s)
    if own:
        s["opt"].step(s["grads"])
        m, v = s["opt"].moments()
        return {"params": s["p"], "exp_avg": m.view(-1, BLOCK), "exp_avg_sq": v.view(-1, BLOCK), "norm": s["opt"].norm if case["max_norm"] else None}
    return _adamw(s)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def _exact_rows(logits, valid, actions, temperature):
    """Softmax of the existing columns of some rows: (existing, p, log p, log of the sum, entropy)."""
    there = logits.double() > -math.inf
    if valid is not None:
        there = there & (valid != 0)
    z = torch.where(there, logits.double() / temperature, -math.inf)
    lse = torch.logsumexp(z, 1)
    lp = torch.where(there, z - torch.where(there.any(1), lse, 0.0)[:, None], -math.inf)
    p = lp.exp()
    return there, p, lp, lse, -torch.xlogy(p, p).sum(1)


def exact(case, seed):
    global own
    own = False                                        # the inputs alone
    s = prepare(case, seed)
    if case["op"] == "adamw":
        b1, b2, lr, t = 0.9, 0.999, 1e-3, case["t"]
        g, p = s["g"].double(), s["p"].double()
        norm = None
        if case["max_norm"]:
            norm = torch.linalg.vector_norm(g)
            if float(norm) > case["max_norm"]:
                g *= case["max_norm"] / norm
        if case["bits"] == 8:
            m = s["m"].double() * s["m_scale"].double()
            c = s["v"].long()
            unit = torch.where(c > 0, 2.0 ** (((c + LEVEL0) >> 4) - 127).double() * (1 + ((c + LEVEL0) & 15).double() / 16), 0.0)
            v = (unit * s["v_scale"].double()) ** 2
        else:
            m, v = s["m"].double(), s["v"].double()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g ** 2
        p = p - lr * s["decay"].double() * p - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + 1e-8)
        # a moment in 8 bits is its code's value: which of two neighbouring codes, is a matter of the last bit of the 32
        return {"params": p, "exp_avg": m if case["bits"] == 32 else None, "exp_avg_sq": v if case["bits"] == 32 else None, "norm": norm}
    rows, step = case["rows"], max(1, 40_000_000 // case["cols"])
    if case["op"] == "logprobs_grad":
        out = []
        for a in range(0, rows, step):
            cut = slice(a, a + step)
            act = s["actions"][cut].long()
            there, p, lp, _, entropy = _exact_rows(s["logits"][cut], None if s["valid"] is None else s["valid"][cut], act, case["temperature"])
            gl = s["d_logp"][cut].double() * (act >= 0)
            d = -gl[:, None] * p
            hot = torch.nn.functional.one_hot(act.clamp(min=0), case["cols"]).bool()
            d = torch.where(hot, d + gl[:, None], d)
            d -= s["d_entropy"][cut].double()[:, None] * (torch.xlogy(p, p) + p * entropy[:, None])
            out.append(torch.where(there, d / case["temperature"], 0.0))
        return torch.cat(out)
    got = []
    for a in range(0, rows, step):
        cut = slice(a, a + step)
        act = s["actions"][cut].long()
        _, _, lp, lse, entropy = _exact_rows(s["logits"][cut], None if s["valid"] is None else s["valid"][cut], act, case["temperature"])
        given = torch.where(act < 0, 0.0, lp[torch.arange(len(act), device=DEV), act.clamp(min=0)])
        best = torch.topk(lp, case["top"], 1).values if case["top"] else None
        got.append((given, entropy, lse, best))
    cat = lambda i: torch.cat([x[i] for x in got])  # noqa: E731
    return dict(logp=cat(0), entropy=cat(1), lse=cat(2), top_actions=None, top_logp=cat(3) if case["top"] else None)
