"""The steps from the residual stream to the next token with 8-bit activations, whose speed is measured:
the norm with the residual's addition and an FP8 output, rows and gated activations to FP8, the matrix
product of FP8 rows and weights with a scale for each block of 128, and the draw of a token.

``run`` computes a case in plain torch operations, in 32 bits (the draw in 64) and rounded once at the end,
or (``own``) through the framework's entry points. ``exact`` restates each case in 64 bits.

Shapes are the repository's own configurations (hidden 7168 / intermediate 2048, 5120 / 2304, 2560 / 640; a
vocabulary of 129,280) and, in ``draw``, any size of the ranges they span.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

VOCAB = 129280
EPS = 1e-6
BLOCK = 128
TOP = 448.0          # the largest E4M3 value
TINY = 2.0 ** -126   # the least scale


# ------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decode token between a block and the next projection: nothing but latency
        {"name": "norm-decode-1", "kind": "norm", "tokens": 1, "hidden": 7168, "residual": "fp32", "x": False, "offset": 0.0},
        # a ragged prompt chunk with a bf16 residual, whose x the router reads as well
        {"name": "norm-prompt-4001", "kind": "norm", "tokens": 4001, "hidden": 5120, "residual": "bf16", "x": True, "offset": 0.0},
        # a batch of decode requests between the two products of an MLP
        {"name": "swiglu-batch-64", "kind": "rows", "swiglu": True, "tokens": 64, "width": 2048, "type": "bf16", "limit": 0.0,
         "up_first": False, "pow2": False},
        # a long prompt's attention output on its way to the next projection, scales as powers of two
        {"name": "rows-prompt-16384", "kind": "rows", "swiglu": False, "tokens": 16384, "width": 7168, "type": "bf16", "limit": 0.0,
         "up_first": False, "pow2": True},
        # one decode token through a shared expert's gate and up
        {"name": "linear-decode-1", "kind": "linear", "tokens": 1, "k": 7168, "n": 4096, "out": "bf16", "add": False},
        # a verify round's six rows through the head, to fp32 logits
        {"name": "linear-head-6", "kind": "linear", "tokens": 6, "k": 7168, "n": VOCAB, "out": "fp32", "add": False},
        # a batch of decode requests
        {"name": "linear-batch-96", "kind": "linear", "tokens": 96, "k": 5120, "n": 4608, "out": "bf16", "add": False},
        # a ragged prompt onto an fp32 stream, outputs that are no multiple of anything
        {"name": "linear-ragged-1501", "kind": "linear", "tokens": 1501, "k": 2560, "n": 1283, "out": "fp32", "add": True},
        # a long prompt through a shared expert's gate and up
        {"name": "linear-prompt-16384", "kind": "linear", "tokens": 16384, "k": 7168, "n": 4096, "out": "bf16", "add": False},
        # the next token of one request, nucleus of what top-k leaves
        {"name": "sample-decode-1", "kind": "sample", "rows": 1, "vocab": VOCAB, "type": "fp32", "top_k": True, "top_p": True,
         "min_p": False, "mask": False},
        # a few requests that sample from the whole nucleus, under a grammar's mask
        {"name": "sample-nucleus-5", "kind": "sample", "rows": 5, "vocab": VOCAB, "type": "fp32", "top_k": False, "top_p": True,
         "min_p": False, "mask": True},
        # a large batch with every rule, some rows greedy
        {"name": "sample-batch-192", "kind": "sample", "rows": 192, "vocab": VOCAB, "type": "bf16", "top_k": True, "top_p": True,
         "min_p": True, "mask": False},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    w, form = _log(rng, low, high), rng.random()
    return w if form < 0.25 else min(high, -(-w // 128) * 128)


def draw(rng):
    kind = rng.choice(["norm", "rows", "linear", "linear", "sample"])
    if kind == "norm":
        H = _width(rng, 96, 16384)
        return {"kind": kind, "tokens": _log(rng, 1, min(20000, 16384 * 7168 // H)), "hidden": H,
                "residual": rng.choice(["fp32", "bf16"]), "x": rng.random() < 0.3, "offset": rng.choice([0.0, 0.0, 1.0])}
    if kind == "rows":
        W, swiglu = _width(rng, 64, 16384), rng.random() < 0.5
        return {"kind": kind, "swiglu": swiglu, "tokens": _log(rng, 1, min(20000, 8192 * 7168 // W)), "width": W,
                "type": rng.choice(["bf16", "bf16", "fp32"]), "limit": rng.choice([0.0, 10.0]) if swiglu else 0.0,
                "up_first": swiglu and rng.random() < 0.3, "pow2": not swiglu and rng.random() < 0.5}
    if kind == "linear":
        K = -(-_width(rng, 128, 8192) // 16) * 16
        N = rng.choice([_width(rng, 32, 16384), _width(rng, 512, 8192)])
        M = _log(rng, 1, min(16384, 16384 * 7168 * 4096 // (K * N)))
        return {"kind": kind, "tokens": M, "k": K, "n": N, "out": rng.choice(["bf16", "bf16", "fp32"]), "add": rng.random() < 0.3}
    V = rng.choice([VOCAB, rng.randint(500, 160000), rng.randint(20000, 160000)])
    return {"kind": kind, "rows": _log(rng, 1, min(256, 192 * VOCAB // V)), "vocab": V, "type": rng.choice(["fp32", "bf16"]),
            "top_k": rng.random() < 0.5, "top_p": rng.random() < 0.6, "min_p": rng.random() < 0.3, "mask": rng.random() < 0.3}


# ------------------------------------------------------------------------------- inputs

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _stored_weights(w):
    """A checkpoint's FP8 weights: a scale for each 128 x 128 block."""
    N, K = w.shape
    n, k = -(-N // BLOCK), -(-K // BLOCK)
    blocks = torch.nn.functional.pad(w, (0, k * BLOCK - K, 0, n * BLOCK - N)).view(n, BLOCK, k, BLOCK)
    s = blocks.abs().amax((1, 3)) / TOP
    q = (blocks / s[:, None, :, None]).to(torch.float8_e4m3fn).view(n * BLOCK, k * BLOCK)[:N, :K]
    return q.contiguous(), s


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = SimpleNamespace(case=dict(case))
    if kind == "norm":
        T, H, off = case["tokens"], case["hidden"], case["offset"]
        loud = torch.exp(torch.randn(H, device="cuda", generator=g) * 0.5)  # channels of uneven size, as a residual has
        s.residual = (torch.randn(T, H, device="cuda", generator=g) * loud * 2).to(_TYPES[case["residual"]])
        s.y = _randn(g, T, H, std=0.5, dtype=torch.bfloat16)
        s.weight = (1 - off + torch.randn(H, device="cuda", generator=g) * 0.1).to(torch.bfloat16)
    elif kind == "rows":
        T, W = case["tokens"], case["width"]
        s.x = _randn(g, T, 2 * W if case["swiglu"] else W, std=3.0 if case["limit"] else 1.0, dtype=_TYPES[case["type"]])
    elif kind == "linear":
        T, K, N = case["tokens"], case["k"], case["n"]
        x = _randn(g, T, K)
        s.scales = torch.stack([b.abs().amax(1) for b in x.split(BLOCK, 1)], 1) / TOP
        s.x = (x / s.scales.repeat_interleave(BLOCK, 1)[:, :K]).to(torch.float8_e4m3fn)
        s.weight, s.weight_scales = _stored_weights(_randn(g, N, K, std=K ** -0.5))
        s.add = _randn(g, T, N, dtype=_TYPES[case["out"]]) if case["add"] else None
    else:
        R, V = case["rows"], case["vocab"]
        rand = lambda *shape: torch.rand(*shape, device="cuda", generator=g)  # noqa: E731
        # a head's logits: a few tokens far above a long tail
        rank = torch.stack([torch.randperm(V, device="cuda", generator=g) for _ in range(R)]).float()
        s.logits = (_randn(g, R, V, std=1.5) - 1.6 * torch.log1p(rank)).to(_TYPES[case["type"]])
        if case["mask"]:
            s.logits[rand(R, V) < 0.4] = -math.inf
        s.uniforms = rand(R)
        s.temperature = 0.4 + 1.2 * rand(R)
        if R > 1:
            s.temperature[rand(R) < 0.1] = 0.0  # greedy
        s.top_k = torch.randint(0, 200, (R,), device="cuda", generator=g, dtype=torch.int32) if case["top_k"] else None  # 0: off
        s.top_p = 0.5 + 0.5 * rand(R) if case["top_p"] else None
        s.min_p = 0.1 * rand(R) if case["min_p"] else None
    return s


# ------------------------------------------------------------------------------- one pass

def _to_fp8(x, pow2=False):
    """fp32 rows to E4M3 with a scale for each 128 values."""
    T, W = x.shape
    b = -(-W // BLOCK)
    blocks = torch.nn.functional.pad(x, (0, b * BLOCK - W)).view(T, b, BLOCK)
    s = (blocks.abs().amax(2) / TOP).clamp(min=TINY)
    if pow2:
        m, e = torch.frexp(s)
        s = torch.ldexp(torch.ones_like(s), e - (m == 0.5).int())
    return (blocks / s[..., None]).view(T, b * BLOCK)[:, :W].to(torch.float8_e4m3fn), s


def _run_norm(s):
    c = s.case
    if own:
        import whallm_amd as wa
        got = wa.norm_fp8(s.residual, s.y, s.weight, eps=EPS, weight_offset=c["offset"], with_x=c["x"])
        return dict(zip(("q", "scales", "residual", "x"), got))
    r = (s.residual.float() + s.y.float()).to(s.residual.dtype)
    v = r.float()
    x = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * (s.weight.float() + c["offset"])
    q, scales = _to_fp8(x)
    return {"q": q, "scales": scales, "residual": r, **({"x": x.to(torch.bfloat16)} if c["x"] else {})}


def _run_rows(s):
    c = s.case
    if own:
        import whallm_amd as wa
        if c["swiglu"]:
            return wa.swiglu_fp8(s.x, limit=c["limit"], up_first=c["up_first"], pow2_scales=c["pow2"])
        return wa.quantize_fp8(s.x, pow2_scales=c["pow2"])
    x = s.x.float()
    if c["swiglu"]:
        a, b = x.chunk(2, 1)
        gate, up = (b, a) if c["up_first"] else (a, b)
        if c["limit"]:
            gate, up = gate.clamp(max=c["limit"]), up.clamp(-c["limit"], c["limit"])
        x = gate * torch.sigmoid(gate) * up
    return _to_fp8(x, c["pow2"])


def _run_linear(s):
    dt = _TYPES[s.case["out"]]
    if own:
        import whallm_amd as wa
        return wa.linear_fp8(s.x, s.scales, s.weight, s.weight_scales, out_dtype=dt, add=s.add)
    N, K = s.weight.shape
    x = s.x.float() * s.scales.repeat_interleave(BLOCK, 1)[:, :K]
    w = s.weight_scales.repeat_interleave(BLOCK, 1)[:, :K].repeat_interleave(BLOCK, 0)[:N] * s.weight.float()
    y = x @ w.t()
    return (y if s.add is None else y + s.add.float()).to(dt)


def _run_sample(s):
    if own:
        import whallm_amd as wa
        tokens, logp = wa.sample_logits(s.logits, s.uniforms, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p,
                                        min_p=s.min_p)
        return {"tokens": tokens, "logp": logp}
    R, V = s.logits.shape
    l, order = torch.sort(s.logits.double(), dim=1, descending=True, stable=True)
    t = s.temperature.double()[:, None]
    greedy = t == 0
    p = torch.exp((l - l[:, :1]) / torch.where(greedy, 1.0, t))
    at = torch.arange(V, device=l.device)
    keep = torch.isfinite(l)
    if s.top_k is not None:
        keep &= (s.top_k[:, None] <= 0) | (at < s.top_k[:, None])
    if s.top_p is not None:
        kept = torch.where(keep, p, 0.0)
        before = torch.cumsum(kept, 1) - kept
        keep &= (before < s.top_p.double()[:, None] * kept.sum(1, keepdim=True)) | (s.top_p[:, None] >= 1)
    if s.min_p is not None:
        keep &= p >= s.min_p.double()[:, None]
    keep &= ~greedy | (at == 0)
    p = torch.zeros_like(p).scatter(1, order, torch.where(keep, p, 0.0))  # by token id
    running = torch.cumsum(p, 1)
    token = (running <= s.uniforms.double()[:, None] * running[:, -1:]).sum(1, keepdim=True)
    return {"tokens": token[:, 0].int(), "logp": torch.log(p.gather(1, token) / running[:, -1:])[:, 0].float()}


def run(s):
    return {"norm": _run_norm, "rows": _run_rows, "linear": _run_linear, "sample": _run_sample}[s.case["kind"]](s)


# ------------------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "norm":
        T, H, r = case["tokens"], case["hidden"], 4 if case["residual"] == "fp32" else 2
        return {"bytes": T * (H * (2 * r + 3 + (2 if case["x"] else 0)) + 4 * -(-H // BLOCK)) + 2 * H, "flops": 8 * T * H}
    if kind == "rows":
        T, W, size = case["tokens"], case["width"], 2 if case["type"] == "bf16" else 4
        return {"bytes": T * (W * (size * (2 if case["swiglu"] else 1) + 1) + 4 * -(-W // BLOCK)),
                "flops": T * W * (10 if case["swiglu"] else 3)}
    if kind == "linear":
        T, K, N, size = case["tokens"], case["k"], case["n"], 2 if case["out"] == "bf16" else 4
        b = -(-K // BLOCK)
        return {"bytes": T * (K + 4 * b) + N * K + 4 * b * -(-N // BLOCK) + T * N * size * (2 if case["add"] else 1),
                "flops": 2 * T * N * K}
    R, V = case["rows"], case["vocab"]
    return {"bytes": R * V * (2 if case["type"] == "bf16" else 4) + 28 * R, "flops": 6 * R * V}


# ------------------------------------------------------------------------------- 64 bits

def _exact_fp8(x, pow2):
    """What the values would be without the rounding to E4M3."""
    scales = torch.stack([b.abs().amax(1) for b in x.split(BLOCK, 1)], 1) / TOP
    scales = torch.maximum(scales, torch.full_like(scales, TINY))
    if pow2:
        scales = 2.0 ** torch.ceil(torch.log2(scales))
    return torch.cat([b / scales[:, i:i + 1] for i, b in enumerate(x.split(BLOCK, 1))], 1), scales


def _exact_norm(case, s):
    r = s.residual.double() + s.y.double()
    v = r.to(s.residual.dtype).double()  # the norm reads the residual as it is stored
    x = v / torch.sqrt(torch.mean(v * v, -1, True) + EPS) * (s.weight.double() + case["offset"])
    q, scales = _exact_fp8(x, False)
    return {"q": q, "scales": scales, "residual": r, **({"x": x} if case["x"] else {})}


def _exact_rows(case, s):
    x, W, limit = s.x.double(), case["width"], case["limit"]
    if case["swiglu"]:
        up, gate = (x[:, :W], x[:, W:]) if case["up_first"] else (x[:, W:], x[:, :W])
        if limit:
            up, gate = torch.clip(up, -limit, limit), torch.clip(gate, max=limit)
        x = up * gate / (1 + torch.exp(-gate))
    return _exact_fp8(x, case["pow2"])


def _exact_linear(case, s):
    y = torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device="cuda") if s.add is None else s.add.double()
    rows = torch.arange(case["n"], device="cuda") // BLOCK
    for i in range(s.scales.shape[1]):  # block by block along K
        at = slice(i * BLOCK, (i + 1) * BLOCK)
        y += (s.x[:, at].double() * s.scales[:, i:i + 1].double()) @ (s.weight[:, at].double().t() *
                                                                      s.weight_scales[rows, i].double())
    return y


def _exact_sample(case, s):
    mine = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    logits, u, temp, tk, tp, mp = (mine(t) for t in (s.logits, s.uniforms, s.temperature, s.top_k, s.top_p, s.min_p))
    tokens, logp = [], []
    for r in range(case["rows"]):
        l = logits[r]
        order = np.argsort(-l, kind="stable")
        order = order[np.isfinite(l[order])]
        if temp[r] == 0:
            order = order[:1]
        elif tk is not None and tk[r] > 0:
            order = order[:int(tk[r])]
        p = np.exp((l[order] - l[order[0]]) / (temp[r] if temp[r] else 1.0))
        n = len(order)
        if tp is not None and tp[r] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(p)[:-1], tp[r] * p.sum(), side="left"))
        if mp is not None:
            n = min(n, int((p >= mp[r]).sum()))
        ids = np.sort(order[:n])
        q = np.zeros(case["vocab"])
        q[order[:n]] = p[:n]
        run = np.cumsum(q[ids])
        token = ids[np.searchsorted(run, u[r] * run[-1], side="right")]
        tokens.append(token)
        logp.append(math.log(q[token] / run[-1]))
    return {"tokens": np.array(tokens, np.int32), "logp": np.array(logp)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rows": _exact_rows, "linear": _exact_linear, "sample": _exact_sample}[case["kind"]](case, s)
