"""The token sort, the block norms and the logit rules in one run, as a decoder layer and its head use them:
norm, route, tokens to their experts, the experts' products, back, gated norm, head, penalties and
mask, acceptance; its gradients; and captured.

Bar: every step against its formula in 64 bits, from the values that the step was given, within the
bounds of the step's own tests; what runs through autograd or a graph bit for bit as the plain calls.
"""
import numpy as np
import pytest
import torch

import whallm_amd as wa
from running_error import Fp32, check
from test_gpu_block_norm import f64, want_forward, want_grads, want_x
from test_gpu_process_logits import want_logits

pytestmark = pytest.mark.gpu
EPS, SCALE = 1e-6, 0.6


def rand(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def layer(device, T, H, I, E, V, seed):
    g = torch.Generator().manual_seed(seed)
    s = dict(residual=rand(g, T, H, std=2.0, dtype=torch.float32), y=rand(g, T, H, std=0.5), post=1 + rand(g, H, std=0.2),
             pre=1 + rand(g, H, std=0.2), channel=rand(g, H, std=0.5, dtype=torch.float32), router=rand(g, E, H, std=H ** -0.5),
             gate_w=rand(g, E, I, H, std=H ** -0.5), up_w=rand(g, E, I, H, std=H ** -0.5),
             down_w=rand(g, E, H, I, std=I ** -0.5), token=rand(g, T, 1, dtype=torch.float32),
             head=rand(g, V, H, std=2 * H ** -0.5),
             history=torch.randint(0, V, (1, 40 + T), generator=g, dtype=torch.int32),
             mask=torch.randint(-2 ** 31, 2 ** 31 - 1, (1, -(-V // 32)), generator=g, dtype=torch.int32),
             drafts=torch.randint(0, V, (T - 1,), generator=g, dtype=torch.int32))
    return {k: v.to(device) for k, v in s.items()}


def rules(s):
    T = s["y"].shape[0]
    per = lambda v: torch.full((T,), v, device=s["y"].device)  # noqa: E731
    return dict(history=s["history"], lengths=(40 + torch.arange(T, device=s["y"].device)).to(torch.int32),
                prompt_lengths=per(20).to(torch.int32), repetition=per(1.2), frequency=per(0.3), presence=per(0.1),
                mask=s["mask"], temperature=per(0.8))


def rows_sum(terms, add, name, got):
    """A weighted sum in fp32, in order, rounded once."""
    total = Fp32(0.0) if add is None else Fp32(add)
    magnitude = np.abs(terms).sum(1) + (0.0 if add is None else np.abs(add))
    check(name, got, Fp32(terms.sum(1) + total.v, (terms.shape[1] + 2) * 2.0 ** -24 * magnitude))


@pytest.mark.parametrize("T,H,I,E,K,V", [(1, 128, 64, 8, 2, 500), (5, 256, 64, 12, 3, 1003), (300, 512, 128, 16, 4, 4096)])
def test_layer_and_head(device, T, H, I, E, K, V):
    s = layer(device, T, H, I, E, V, T)
    first = dict(residual=s["residual"], y=s["y"], post_weight=s["post"], pre_weight=s["pre"], gate=s["channel"], weight_offset=0.0)
    x, r = wa.block_norm(**{k: v for k, v in first.items()}, scale=SCALE, eps=EPS)
    check("residual", r, want_forward(first, False, SCALE, EPS, True))
    check("x", x, want_x(r, first, EPS))

    idx, w = wa.route_softmax_topk(wa.linear_bf16(x, s["router"]), K)
    if T > 2:
        idx[1, 0] = -1                                   # a pair that goes nowhere
    rows, p = wa.sort_tokens(x, idx, E, tile_rows=32)
    at = p.offsets.tolist()
    prod = torch.zeros_like(rows)
    for e in range(E):
        if at[e + 1] > at[e]:
            prod[at[e]:at[e + 1]] = wa.mlp_bf16(rows[at[e]:at[e + 1]], s["gate_w"][e], s["up_w"][e], s["down_w"][e])
    out = wa.combine_rows(prod, w, p, add=x)
    pairs = np.zeros((T, K, H))
    flat = idx.cpu().numpy()
    for t in range(T):                                   # each token's experts by themselves, from the token's row
        for k in range(K):
            if flat[t, k] >= 0:
                row = f64(x[t])
                assert np.array_equal(f64(rows[p.inverse.reshape(T, K)[t, k]]), row)
                pairs[t, k] = f64(prod[p.inverse.reshape(T, K)[t, k]])
    rows_sum(pairs * f64(w)[..., None], f64(x), "combined", out)

    second = dict(residual=r, y=out, post_weight=s["post"], pre_weight=s["pre"], gate=s["token"], weight_offset=0.0)
    x2, r2 = wa.block_norm(**second, gate_sigmoid=True, scale=SCALE, eps=EPS)
    check("second residual", r2, want_forward(second, True, SCALE, EPS, True))
    check("second x", x2, want_x(r2, second, EPS))

    logits = wa.linear_bf16(x2, s["head"])
    got = wa.process_logits(logits, **rules(s))
    check("logits", got, want_logits(logits, **rules(s)))
    few = min(T, 16)                                     # a verify round has at most 15 drafts
    accepted, token = wa.mtp_verify_greedy(got[:few], s["drafts"][:few - 1]).tolist()
    best = got.argmax(-1)
    n = 0
    while n < few - 1 and best[n] == s["drafts"][n]:
        n += 1
    assert (accepted, token) == (n, int(best[n]))
    logp = wa.process_logits(logits, log_probs=True, **rules(s))
    check("log-probabilities", logp, want_logits(logits, log_probs=True, **rules(s)))


class Experts(torch.autograd.Function):
    """Tokens to their experts, one linear layer per expert, and back."""
    @staticmethod
    def forward(ctx, x, w, weight, idx):
        rows, p = wa.sort_tokens(x, idx, weight.shape[0])
        prod = products(rows, weight, p.offsets)
        ctx.save_for_backward(rows, prod, w, weight)
        ctx.p = p
        return wa.combine_rows(prod, w, p)

    @staticmethod
    def backward(ctx, dy):
        rows, prod, w, weight = ctx.saved_tensors
        dprod, dw = wa.combine_rows_backward(dy, prod, w, ctx.p)
        drows = products(dprod, weight.transpose(1, 2), ctx.p.offsets)
        at = ctx.p.offsets.tolist()
        dweight = torch.stack([dprod[a:b].float().t() @ rows[a:b].float() for a, b in zip(at, at[1:])])
        return wa.sort_tokens_backward(drows, ctx.p, w.shape[1]), dw, dweight.to(weight.dtype), None


def products(rows, weight, offsets):
    out, at = torch.zeros(rows.shape[0], weight.shape[1], dtype=rows.dtype, device=rows.device), offsets.tolist()
    for e, (a, b) in enumerate(zip(at, at[1:])):
        out[a:b] = (rows[a:b].float() @ weight[e].float().t()).to(rows.dtype)
    return out


class Norms(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, y, post, pre, gate):
        x, r = wa.block_norm(residual, y, post, pre, gate, scale=SCALE, eps=EPS)
        ctx.save_for_backward(r, y, post, pre, gate)
        return x, r

    @staticmethod
    def backward(ctx, dx, dr):
        r, y, post, pre, gate = ctx.saved_tensors
        d = wa.block_norm_backward(dx, dr, r, y, post, pre, gate, scale=SCALE, eps=EPS)
        return d.residual, d.y, d.post_weight.to(post.dtype), d.pre_weight.to(pre.dtype), d.gate.to(gate.dtype)


@pytest.mark.parametrize("T,H,E,K", [(1, 64, 4, 2), (37, 264, 7, 3)])
def test_gradients_of_a_run(device, T, H, E, K):
    """Two norms around the experts, trained by autograd: every leaf's gradient is that of the calls in turn, and
    theirs, step by step, the formulas'."""
    s = layer(device, T, H, 32, E, 100, 3)
    expert = s["gate_w"].new_empty(E, H, H).normal_(0, H ** -0.5, generator=torch.Generator(device).manual_seed(5))
    leaves = {k: s[k].clone().requires_grad_() for k in ("residual", "y", "post", "pre", "channel")}
    leaves["expert"] = expert.clone().requires_grad_()
    gen = torch.Generator().manual_seed(9)
    dx, dr = rand(gen, T, H).to(device), rand(gen, T, H, dtype=torch.float32).to(device)
    norm = lambda r, y: Norms.apply(r, y, leaves["post"], leaves["pre"], leaves["channel"])  # noqa: E731

    x1, r1 = norm(leaves["residual"], leaves["y"])
    with torch.no_grad():
        idx, w = wa.route_softmax_topk(wa.linear_bf16(x1, s["router"]), K)
    w = w.requires_grad_()
    y2 = Experts.apply(x1, w, leaves["expert"], idx)
    x2, r2 = norm(r1, y2)
    torch.autograd.backward([x2, r2], [dx, dr])

    with torch.no_grad():
        base = dict(post_weight=s["post"], pre_weight=s["pre"], gate=s["channel"])
        how = dict(scale=SCALE, eps=EPS)
        a1, b1 = wa.block_norm(s["residual"], s["y"], **base, **how)
        rows, p = wa.sort_tokens(a1, idx, E)
        prod = products(rows, expert, p.offsets)
        out = wa.combine_rows(prod, w, p)
        a2, b2 = wa.block_norm(b1, out, **base, **how)
        assert torch.equal(a2, x2) and torch.equal(b2, r2)
        d2 = wa.block_norm_backward(dx, dr, b2, out, **base, **how)
        want = want_grads(dict(residual=b2, y=out, weight_offset=0.0, **base), dx, dr, False, SCALE, EPS, True)
        for name in ("residual", "y", "post_weight", "pre_weight", "gate"):
            check("second d" + name, getattr(d2, name), want[name])
        dprod, dw = wa.combine_rows_backward(d2.y, prod, w, p)
        inverse, dy = p.inverse.cpu().numpy().reshape(T, K), f64(d2.y)
        dots = f64(prod)[inverse] * dy[:, None]
        check("dw", dw, Fp32(dots.sum(-1), (-(-H // 64) + 65) * 2.0 ** -24 * np.abs(dots).sum(-1)))
        check("dprod", dprod[p.inverse.long()].reshape(T, K, H), Fp32(f64(w)[..., None] * dy[:, None]))
        drows = products(dprod, expert.transpose(1, 2), p.offsets)
        da1 = wa.sort_tokens_backward(drows, p, K)
        rows_sum(f64(drows)[inverse], None, "dx", da1)
        d1 = wa.block_norm_backward(da1, d2.residual, b1, s["y"], **base, **how)
        want = want_grads(dict(residual=b1, y=s["y"], weight_offset=0.0, **base), da1, d2.residual, False, SCALE, EPS, True)
        for name in ("residual", "y", "post_weight", "pre_weight", "gate"):
            check("first d" + name, getattr(d1, name), want[name])
        assert torch.equal(leaves["residual"].grad, d1.residual) and torch.equal(leaves["y"].grad, d1.y)
        assert torch.equal(w.grad, dw)
        for leaf, name in (("post", "post_weight"), ("pre", "pre_weight"), ("channel", "gate")):
            both = [getattr(d, name).to(leaves[leaf].dtype) for d in (d2, d1)]
            assert torch.equal(leaves[leaf].grad, both[0] + both[1]), leaf
        assert leaves["expert"].grad.isfinite().all()


def test_two_captured_runs(device):
    """Two graphs of the run, replayed in turn with new inputs and eager calls between, bit for bit as eager; the
    gradients' calls among them."""
    K, E, shapes = 3, 12, [(4, 256, 1003), (9, 128, 500)]

    def run(s, idx_rows):
        x, r = wa.block_norm(s["residual"], s["y"], s["post"], s["pre"], s["channel"], scale=SCALE)
        idx, w = wa.route_softmax_topk(wa.linear_bf16(x, s["router"]), K)
        rows, p = wa.sort_tokens(x, idx, E)
        prod = wa.linear_bf16(rows, s["square"])
        y = wa.combine_rows(prod, w, p).to(torch.bfloat16)
        x2, r2 = wa.block_norm(r, y, s["post"], s["pre"], s["token"], gate_sigmoid=True)
        d = wa.block_norm_backward(x, r, r2, y, s["post"], s["pre"], s["token"], gate_sigmoid=True)
        drows, dw = wa.combine_rows_backward(d.y.float(), prod, w, p)
        dx = wa.sort_tokens_backward(drows, p, K)
        logits = wa.process_logits(wa.linear_bf16(x2, s["head"]), **idx_rows, log_probs=True)
        return [x2, r2, logits, wa.mtp_verify_greedy(logits, s["drafts"]), d.y, d.post_weight, d.gate, dw, dx, p.tiles]

    graphs = []
    for T, H, V in shapes:
        s = layer(device, T, H, 32, E, V, T)
        s["square"] = s["down_w"].new_empty(H, H).normal_(0, H ** -0.5, generator=torch.Generator(device).manual_seed(1))
        fixed = rules(s)
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            run(s, fixed)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(s, fixed)
        graphs.append((s, fixed, graph, outs))
    for step in range(4):
        for s, fixed, graph, outs in graphs:
            gen = torch.Generator().manual_seed(step)
            s["residual"].copy_(rand(gen, *s["residual"].shape, dtype=torch.float32))
            s["y"].copy_(rand(gen, *s["y"].shape))
            graph.replay()
        for s, fixed, graph, outs in graphs:
            want = run(s, fixed)
            for i, (a, b) in enumerate(zip(outs, want)):
                assert torch.equal(a, b), (step, i)
        torch.cuda.synchronize(device)


def test_inference_mode_and_grad_mode(device):
    """The same results under inference mode, where outputs are inference tensors, and for leaves under no_grad."""
    s = layer(device, 6, 128, 32, 5, 100, 2)

    def run():
        x, r = wa.block_norm(s["residual"].clone(), s["y"], s["post"], s["pre"], s["channel"])
        again = r.clone()
        wa.block_norm(again, s["y"], residual_out=again)
        idx = (torch.arange(18, device=device, dtype=torch.int32) % 6 - 1).view(6, 3)
        rows, p = wa.sort_tokens(x, idx, 5)
        y = wa.combine_rows(rows, torch.ones(6, 3, device=device), p, add=x)
        logits = wa.process_logits(wa.linear_bf16(y, s["head"]), **rules(s))
        wa.process_logits(logits, out=logits, log_probs=True)
        d = wa.block_norm_backward(y, r, again, s["y"], s["post"], s["pre"], s["channel"])
        return [x, r, again, p.order, p.inverse, p.offsets, p.tile_count, y, logits, d.post_weight, d.pre_weight, d.gate]

    want = run()
    with torch.inference_mode():
        got = run()
        assert all(t.is_inference() for t in got)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for t in (s["residual"], s["post"], s["channel"]):
        t.requires_grad_()
    with pytest.raises(ValueError, match="autograd"):
        wa.block_norm(s["residual"], s["y"], s["post"], s["pre"], s["channel"])
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(want, run()))
