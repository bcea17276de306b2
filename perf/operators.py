"""The steps around the expert products whose speed is measured: tokens sorted by expert and back
with their gradients, the norms around a block, and the logits on their way to acceptance.

``run`` computes a case in plain torch operations, in 32 bits and rounded once at the end, or
(``own``) through the framework's entry points. ``exact`` restates each case in 64 bits.

Shapes are the repository's own configurations (hidden 2048 / 512 experts / top 10, 2560 / 512 /
10, 4096 / 128 / 8, 7168 / 256 / 8, 5120 / 384 / 6; a vocabulary of 129,280) and, in ``draw``, any
size of the ranges they span.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

VOCAB = 129280
EPS = 1e-6
TILE_ROWS = 128


# ------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decode token's row to its ten experts: nothing but latency
        {"name": "sort-decode-1", "kind": "sort", "grad": False, "tokens": 1, "k": 10, "experts": 512, "hidden": 2048,
         "type": "bf16", "absent": 0.0},
        # a prompt chunk of the widest model, a few tokens of it padding
        {"name": "sort-prompt-4096", "kind": "sort", "grad": False, "tokens": 4096, "k": 8, "experts": 256, "hidden": 7168,
         "type": "bf16", "absent": 0.02},
        # the gradient of the sort for a ragged batch
        {"name": "sort-grad-1501", "kind": "sort", "grad": True, "tokens": 1501, "k": 10, "experts": 512, "hidden": 2560,
         "type": "bf16", "absent": 0.05},
        # the rows of a speculative verify round back from their experts
        {"name": "back-verify-8", "kind": "back", "grad": False, "tokens": 8, "k": 10, "experts": 512, "hidden": 2560,
         "type": "bf16", "absent": 0.0, "add": True},
        # a prompt chunk back from its experts onto the shared expert's output
        {"name": "back-prompt-4096", "kind": "back", "grad": False, "tokens": 4096, "k": 8, "experts": 256, "hidden": 7168,
         "type": "bf16", "absent": 0.02, "add": True},
        # the gradients of rows and router weights in a training step held in fp32
        {"name": "back-grad-2048", "kind": "back", "grad": True, "tokens": 2048, "k": 6, "experts": 384, "hidden": 5120,
         "type": "fp32", "absent": 0.0, "add": False},
        # one decode token between its block and the next, gated by the shared expert's logit
        {"name": "norm-decode-1", "kind": "norm", "grad": False, "tokens": 1, "hidden": 2048, "residual": "fp32",
         "gate": "token", "sigmoid": True, "post": True, "offset": 0.0},
        # a long prompt through a block with a learned scale per channel
        {"name": "norm-prompt-16384", "kind": "norm", "grad": False, "tokens": 16384, "hidden": 4096, "residual": "fp32",
         "gate": "channel", "sigmoid": False, "post": True, "offset": 0.0},
        # a training step's gradients with a bf16 residual and a gate of every element
        {"name": "norm-grad-4001", "kind": "norm", "grad": True, "tokens": 4001, "hidden": 5120, "residual": "bf16",
         "gate": "full", "sigmoid": False, "post": True, "offset": 1.0},
        # the next token of one request that is sampled plainly
        {"name": "logits-decode-1", "kind": "logits", "rows": 1, "vocab": VOCAB, "type": "fp32", "history": 300,
         "shared": False, "biases": 8, "mask": False, "logp": False},
        # a verify round: four rows over one history that grows by a draft a row, to log-probabilities
        {"name": "logits-verify-4", "kind": "logits", "rows": 4, "vocab": VOCAB, "type": "fp32", "history": 4096,
         "shared": True, "biases": 0, "mask": True, "logp": True},
        # a batch of requests with histories of their own, grammar masks and biases
        {"name": "logits-batch-192", "kind": "logits", "rows": 192, "vocab": VOCAB, "type": "bf16", "history": 2000,
         "shared": False, "biases": 64, "mask": True, "logp": True},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _hidden(rng):
    h, form = _log(rng, 96, 8192), rng.random()
    return h if form < 0.2 else -(-h // 8) * 8 if form < 0.5 else -(-h // 128) * 128


def draw(rng):
    kind = rng.choice(["sort", "back", "norm", "logits"])
    grad = rng.random() < 0.5
    if kind in ("sort", "back"):
        H, E = _hidden(rng), rng.randint(8, 512)
        k = rng.randint(1, min(E, 12))
        T = _log(rng, 1, min(16384, 4096 * 6 * 7168 // (k * H)))
        case = {"kind": kind, "grad": grad, "tokens": T, "k": k, "experts": E, "hidden": H,
                "type": rng.choice(["bf16", "bf16", "fp32"]), "absent": rng.choice([0.0, 0.0, 0.1, 0.5])}
        if case["type"] == "fp32":
            case["tokens"] = max(1, T // 2)
        if kind == "back":
            case["add"] = not grad and rng.random() < 0.5
        return case
    if kind == "norm":
        H = _hidden(rng)
        return {"kind": kind, "grad": grad, "tokens": _log(rng, 1, min(20000, 14000 * 4096 // (H * (2 if grad else 1)))),
                "hidden": H, "residual": rng.choice(["fp32", "bf16"]), "gate": rng.choice(["none", "token", "channel", "full"]),
                "sigmoid": rng.random() < 0.5, "post": rng.random() < 0.75, "offset": rng.choice([0.0, 1.0])}
    V = rng.choice([VOCAB, rng.randint(500, 160000), rng.randint(20000, 160000)])
    shared = rng.random() < 0.4
    R = rng.randint(1, 16) if shared else _log(rng, 1, min(256, 192 * VOCAB // V))
    return {"kind": kind, "rows": R, "vocab": V, "type": rng.choice(["fp32", "bf16"]),
            "history": _log(rng, 16, 32768 if R <= 16 else 4096), "shared": shared, "biases": rng.choice([0, rng.randint(1, 300)]),
            "mask": rng.random() < 0.5, "logp": rng.random() < 0.6}


# ------------------------------------------------------------------------------- inputs

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _routes(g, T, k, E, absent):
    """k different experts a token, some of them far busier than others; tokens that are padding,
    and experts that are not resident, have the id -1."""
    busy = -1.5 * torch.log1p(torch.randperm(E, device="cuda", generator=g).float())
    idx = torch.topk(torch.randn(T, E, device="cuda", generator=g) + busy * 0.5, k, dim=1).indices.to(torch.int32)
    if absent:
        u = torch.rand(T, k, device="cuda", generator=g)
        pad = torch.arange(T, device="cuda") >= T - int(T * absent / 2)
        idx = torch.where((u < absent / 2) | pad[:, None], -1, idx)
    return idx.contiguous()


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = SimpleNamespace(case=dict(case))
    if kind in ("sort", "back"):
        T, k, E, H, dt = case["tokens"], case["k"], case["experts"], case["hidden"], _TYPES[case["type"]]
        s.indices = _routes(g, T, k, E, case["absent"])
        if kind == "sort" and not case["grad"]:
            s.x = _randn(g, T, H, dtype=dt)
            return s
        # what the sort has given the program before
        s.lists = _lists(s.indices, E)
        s.rows = _randn(g, T * k, H, dtype=dt)
        s.rows[int(s.lists["offsets"][-1]):] = 0
        if kind == "back":
            s.weights = torch.softmax(torch.randn(T, k, device="cuda", generator=g), dim=1)
            s.dy = _randn(g, T, H, dtype=dt) if case["grad"] else None
            s.add = _randn(g, T, H, dtype=dt) if case["add"] else None
        return s
    if kind == "norm":
        T, H, off = case["tokens"], case["hidden"], case["offset"]
        rt = _TYPES[case["residual"]]
        loud = torch.exp(torch.randn(H, device="cuda", generator=g) * 0.5)  # channels of uneven size, as a residual has
        s.residual = (torch.randn(T, H, device="cuda", generator=g) * loud * 2).to(rt)
        s.y = _randn(g, T, H, std=0.5, dtype=torch.bfloat16)
        s.post = (1 - off + torch.randn(H, device="cuda", generator=g) * 0.1).to(torch.bfloat16) if case["post"] else None
        s.pre = (1 - off + torch.randn(H, device="cuda", generator=g) * 0.1).to(torch.bfloat16)
        s.gate = {"none": lambda: None, "token": lambda: _randn(g, T, 1), "channel": lambda: _randn(g, H),
                  "full": lambda: _randn(g, T, H, dtype=torch.bfloat16)}[case["gate"]]()
        s.scale = 0.7
        if case["grad"]:
            s.dx, s.dres = _randn(g, T, H, dtype=torch.bfloat16), _randn(g, T, H, std=0.3, dtype=rt)
        return s
    R, V, L = case["rows"], case["vocab"], case["history"]
    s.logits = _randn(g, R, V, std=3.0, dtype=_TYPES[case["type"]])
    n = 1 if case["shared"] else R
    s.history = (torch.rand(n, L, device="cuda", generator=g) ** 4 * V).to(torch.int32).clamp_(max=V - 1)
    if case["shared"]:
        s.lengths = (L - R + 1 + torch.arange(R, device="cuda")).clamp_(min=0).to(torch.int32)
        s.prompts = torch.full((R,), L // 2, dtype=torch.int32, device="cuda")
    else:
        s.lengths = torch.randint(L // 4, L + 1, (R,), device="cuda", generator=g, dtype=torch.int32)
        s.prompts = (s.lengths * torch.rand(R, device="cuda", generator=g)).to(torch.int32)
    s.repetition = 1 + torch.rand(R, device="cuda", generator=g) * 0.5
    s.frequency = torch.rand(R, device="cuda", generator=g) * 0.5
    s.presence = torch.rand(R, device="cuda", generator=g) * 0.5
    s.temperature = 0.5 + torch.rand(R, device="cuda", generator=g)
    s.bias_ids = s.bias_values = s.mask = None
    if case["biases"]:
        s.bias_ids = torch.stack([torch.randperm(V, device="cuda", generator=g)[:case["biases"]] for _ in range(R)]).to(torch.int32)
        s.bias_values = _randn(g, R, case["biases"], std=3.0)
    if case["mask"]:
        bits = [torch.randint(-2**31, 2**31, (R, -(-V // 32)), device="cuda", generator=g, dtype=torch.int64) for _ in range(2)]
        s.mask = (bits[0] | bits[1]).to(torch.int32)  # three of four tokens fit the grammar
    return s


# ------------------------------------------------------------------------------- one pass

def _lists(indices, experts):
    """The lists of a sort by expert, -1 behind their ends."""
    P = indices.numel()
    flat = indices.reshape(-1).long()
    key, order = torch.sort(torch.where((flat >= 0) & (flat < experts), flat, experts), stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=key.device))
    at = torch.arange(P, device=key.device)
    live = at < offsets[-1]
    inverse = torch.empty_like(order)
    inverse[order] = torch.where(live, at, -1)
    tiles = (offsets[1:] - offsets[:-1] + TILE_ROWS - 1) // TILE_ROWS
    end = torch.cumsum(tiles, 0)
    t = torch.arange(-(-P // TILE_ROWS) + experts, device=key.device)
    e = torch.searchsorted(end, t, right=True).clamp(max=experts - 1)
    first = offsets[e] + (t - (end[e] - tiles[e])) * TILE_ROWS
    tile = torch.where((t < end[-1])[:, None], torch.stack([e, first], 1), -1)
    got = {"order": torch.where(live, order, -1), "inverse": inverse, "offsets": offsets, "tiles": tile, "tile_count": end[-1:]}
    return {name: v.to(torch.int32) for name, v in got.items()}


def _permutation(lists):
    from whallm_amd import Permutation
    return Permutation(lists["order"], lists["inverse"], lists["offsets"], lists["tiles"], lists["tile_count"])


def _pairs(s):
    """The rows of every token's pairs in 32 bits, zero where a pair is absent, and which are there."""
    inverse = s.lists["inverse"].view(s.case["tokens"], s.case["k"]).long()
    live = inverse >= 0
    return torch.where(live[..., None], s.rows[inverse.clamp(min=0)].float(), 0.0), live


def _run_sort(s):
    c = s.case
    if own:
        import whallm_amd as wa
        if c["grad"]:
            return wa.sort_tokens_backward(s.rows, _permutation(s.lists), c["k"])
        rows, p = wa.sort_tokens(s.x, s.indices, c["experts"], TILE_ROWS)
        return {"rows": rows, "order": p.order, "inverse": p.inverse, "offsets": p.offsets, "tiles": p.tiles,
                "tile_count": p.tile_count}
    if c["grad"]:
        return _pairs(s)[0].sum(1).to(s.rows.dtype)
    lists = _lists(s.indices, c["experts"])
    order = lists["order"].long()
    rows = torch.where((order >= 0)[:, None], s.x[order.clamp(min=0) // c["k"]], 0.0)
    return {"rows": rows, **lists}


def _run_back(s):
    c = s.case
    if own:
        import whallm_amd as wa
        if not c["grad"]:
            return wa.combine_rows(s.rows, s.weights, _permutation(s.lists), s.add)
        drows, dweights = wa.combine_rows_backward(s.dy, s.rows, s.weights, _permutation(s.lists))
        return {"rows": drows, "weights": dweights}
    rows, live = _pairs(s)
    if not c["grad"]:
        y = (rows * torch.where(live, s.weights, 0.0)[..., None]).sum(1)
        return (y if s.add is None else y + s.add.float()).to(s.rows.dtype)
    dy = s.dy.float()
    order = s.lists["order"].long()
    pair = order.clamp(min=0)
    drows = s.weights.view(-1)[pair][:, None] * dy[pair // c["k"]]
    return {"rows": torch.where((order >= 0)[:, None], drows, 0.0).to(s.rows.dtype), "weights": (rows * dy[:, None]).sum(-1)}


def _run_norm(s):
    c = s.case
    if own:
        import whallm_amd as wa
        how = dict(gate=s.gate, gate_sigmoid=c["sigmoid"], scale=s.scale, eps=EPS, weight_offset=c["offset"], post_norm=c["post"])
        if not c["grad"]:
            x, residual = wa.block_norm(s.residual, s.y, s.post, s.pre, **how)
            return {"x": x, "residual": residual}
        d = wa.block_norm_backward(s.dx, s.dres, s.residual, s.y, s.post, s.pre, **how)
        return {"residual": d.residual, "y": d.y, "post": d.post_weight, "pre": d.pre_weight, "gate": d.gate}
    off, y = c["offset"], s.y.float()
    wpre = s.pre.float() + off
    wpost = s.post.float() + off if c["post"] else 1.0
    g = 1.0 if s.gate is None else torch.sigmoid(s.gate.float()) if c["sigmoid"] else s.gate.float()
    p = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) if c["post"] else 1.0
    if not c["grad"]:
        r = (s.residual.float() + s.scale * g * (y * p * wpost)).to(s.residual.dtype)
        v = r.float()
        return {"x": (v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * wpre).to(torch.bfloat16), "residual": r}
    # s.residual is the residual behind the block here, what the forward pass gave
    v, dx = s.residual.float(), s.dx.float()
    q = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    a = dx * wpre
    dr = s.dres.float() + q * (a - v * q.square() * (a * v).mean(-1, keepdim=True))
    b = dr * (s.scale * g)
    cc = b * wpost
    dy = p * (cc - y * p.square() * (cc * y).mean(-1, keepdim=True)) if c["post"] else cc
    dgate = None
    if s.gate is not None:
        dgate = s.scale * dr * (y * p * wpost) * (g * (1 - g) if c["sigmoid"] else 1.0)
        dgate = {"token": lambda: dgate.sum(-1, keepdim=True), "channel": lambda: dgate.sum(0),
                 "full": lambda: dgate.to(s.gate.dtype)}[c["gate"]]()
    return {"residual": dr.to(s.residual.dtype), "y": dy.to(torch.bfloat16),
            "post": (b * y * p).sum(0) if c["post"] else None, "pre": (dx * v * q).sum(0), "gate": dgate}


def _run_logits(s):
    c = s.case
    if own:
        import whallm_amd as wa
        return wa.process_logits(s.logits, history=s.history, lengths=s.lengths, prompt_lengths=s.prompts,
                                 repetition=s.repetition, frequency=s.frequency, presence=s.presence, bias_ids=s.bias_ids,
                                 bias_values=s.bias_values, mask=s.mask, temperature=s.temperature, log_probs=c["logp"])
    R, V = s.logits.shape
    v = s.logits.float()
    at = torch.arange(c["history"], device=v.device)
    said = at < s.lengths[:, None]
    answer = said & (at >= s.prompts[:, None])
    ids = s.history.long().expand(R, -1)
    zero = torch.zeros(R, V, device=v.device)
    seen = zero.scatter_add(1, ids, said.float()) > 0
    count = zero.scatter_add(1, ids, answer.float())
    rep = s.repetition[:, None]
    v = torch.where(seen, torch.where(v > 0, v / rep, v * rep), v)
    v = v - s.frequency[:, None] * count - s.presence[:, None] * (count > 0)
    if s.bias_ids is not None:
        v = v.scatter_add(1, s.bias_ids.long(), s.bias_values)
    v = v / s.temperature[:, None]
    if s.mask is not None:
        i = torch.arange(V, device=v.device)
        v = torch.where((s.mask[:, i // 32] >> (i % 32)) & 1 != 0, v, -math.inf)
    if c["logp"]:
        top = v.amax(1, keepdim=True)
        v = v - top - torch.log(torch.exp(v - top).sum(1, keepdim=True))
    return v


def run(s):
    return {"sort": _run_sort, "back": _run_back, "norm": _run_norm, "logits": _run_logits}[s.case["kind"]](s)


# ------------------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind in ("sort", "back"):
        T, k, H = case["tokens"], case["k"], case["hidden"]
        P, size = T * k, 2 if case["type"] == "bf16" else 4
        read = P * (1 - case["absent"])  # pairs that are there
        if kind == "sort":
            if case["grad"]:
                return {"bytes": size * H * (read + T) + 4 * P, "flops": read * H}
            return {"bytes": size * H * (T + P) + 12 * P + 4 * case["experts"], "flops": P}
        if case["grad"]:
            return {"bytes": size * H * (read + T + P) + 12 * P, "flops": 3 * read * H}
        return {"bytes": size * H * (read + T * (2 if case["add"] else 1)) + 8 * P, "flops": 2 * read * H}
    if kind == "norm":
        T, H, r = case["tokens"], case["hidden"], 4 if case["residual"] == "fp32" else 2
        gate = {"none": 0, "token": 4 * T, "channel": 4 * H, "full": 2 * T * H}[case["gate"]]
        weights = 4 * H if case["post"] else 2 * H
        if case["grad"]:
            return {"bytes": T * H * (3 * r + 6) + 2 * gate + 3 * weights, "flops": 30 * T * H}
        return {"bytes": T * H * (2 * r + 4) + gate + weights, "flops": 10 * T * H}
    R, V, L = case["rows"], case["vocab"], case["history"]
    read = 2 if case["type"] == "bf16" else 4
    lists = 4 * L * (1 if case["shared"] else R) + 8 * R * case["biases"] + (R * V // 8 if case["mask"] else 0)
    return {"bytes": R * V * (read + 4) + lists, "flops": R * V * (10 if case["logp"] else 4)}


# ------------------------------------------------------------------------------- 64 bits

def _exact_rows(case, s):
    T, k, H = case["tokens"], case["k"], case["hidden"]
    idx = s.indices.cpu().numpy().reshape(-1)
    present = np.nonzero((idx >= 0) & (idx < case["experts"]))[0]
    pairs = present[np.argsort(idx[present], kind="stable")]  # the pair of each row
    n = len(pairs)
    token = torch.from_numpy(pairs // k).cuda()
    if case["kind"] == "sort" and not case["grad"]:
        rows = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
        rows[:n] = s.x.double()[token]
        order, inverse = np.full(T * k, -1), np.full(T * k, -1)
        order[:n], inverse[pairs] = pairs, np.arange(n)
        count = np.bincount(idx[present], minlength=case["experts"])
        offsets = np.concatenate([[0], np.cumsum(count)])
        tiles = np.array([(e, r) for e in range(case["experts"]) for r in range(offsets[e], offsets[e + 1], TILE_ROWS)]).reshape(-1, 2)
        whole = np.full((-(-T * k // TILE_ROWS) + case["experts"], 2), -1)
        whole[:len(tiles)] = tiles
        whole, order, inverse, offsets = (v.astype(np.int32) for v in (whole, order, inverse, offsets))
        return {"rows": rows, "order": order, "inverse": inverse, "offsets": offsets, "tiles": whole,
                "tile_count": np.array([len(tiles)], np.int32)}
    rows = s.rows[:n].double()
    if case["kind"] == "sort":
        return torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, token, rows)
    pair = torch.from_numpy(pairs).cuda()
    w = s.weights.double().reshape(-1)[pair]
    if not case["grad"]:
        y = torch.zeros(T, H, dtype=torch.float64, device="cuda") if s.add is None else s.add.double()
        return y.index_add_(0, token, rows * w[:, None])
    dy = s.dy.double()[token]
    drows = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
    drows[:n] = dy * w[:, None]
    dw = torch.zeros(T * k, dtype=torch.float64, device="cuda")
    dw[pair] = torch.linalg.vecdot(dy, rows)
    return {"rows": drows, "weights": dw.view(T, k)}


def _exact_norm(case, s):
    """The forward pass in 64 bits; its gradients by automatic differentiation of the same lines."""
    def leaf(t, offset=0.0):
        return None if t is None else (t.double() + offset).requires_grad_(case["grad"])
    y, gate, post, pre = leaf(s.y), leaf(s.gate), leaf(s.post, case["offset"]), leaf(s.pre, case["offset"])
    z = y if post is None else y / torch.sqrt(torch.mean(y * y, -1, True) + EPS) * post
    if gate is not None:
        z = z * (1 / (1 + torch.exp(-gate)) if case["sigmoid"] else gate)
    branch = s.scale * z
    # behind the block: a gradient pass is given that residual, the sum is taken from before it
    before = s.residual.double() - branch.detach() if case["grad"] else s.residual.double()
    before.requires_grad_(case["grad"])
    r = before + branch
    # the next block's norm reads the residual as it is stored
    v = r if case["grad"] else r.to(s.residual.dtype).double()
    x = v / torch.sqrt(torch.mean(v * v, -1, True) + EPS) * pre
    if not case["grad"]:
        return {"x": x, "residual": r}
    torch.autograd.backward([x, r], [s.dx.double(), s.dres.double()])
    return {"residual": before.grad, "y": y.grad, "post": None if post is None else post.grad, "pre": pre.grad,
            "gate": None if gate is None else gate.grad}


def _exact_logits(case, s):
    R, V = case["rows"], case["vocab"]
    v = s.logits.double().cpu().numpy()
    history = s.history.cpu().numpy()
    mine = lambda t: t.double().cpu().numpy()  # noqa: E731
    rep, freq, pres, temp = mine(s.repetition), mine(s.frequency), mine(s.presence), mine(s.temperature)
    lengths, prompts = s.lengths.cpu().numpy(), s.prompts.cpu().numpy()
    for r in range(R):
        h = history[0 if case["shared"] else r][:lengths[r]]
        u = np.unique(h)
        v[r, u] = np.where(v[r, u] > 0, v[r, u] / rep[r], v[r, u] * rep[r])
        c = np.bincount(h[prompts[r]:], minlength=V)
        v[r] -= freq[r] * c + pres[r] * (c > 0)
        if s.bias_ids is not None:
            v[r, s.bias_ids[r].cpu().numpy()] += mine(s.bias_values[r])
        v[r] /= temp[r]
        if s.mask is not None:
            bits = np.unpackbits(s.mask[r].cpu().numpy().view(np.uint8), bitorder="little")[:V]
            v[r, bits == 0] = -np.inf
        if case["logp"]:
            top = v[r].max()
            v[r] -= top + np.log(np.exp(v[r] - top).sum())
    return v


def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_logits if case["kind"] == "logits" else _exact_norm if case["kind"] == "norm" else _exact_rows)(case, s)
