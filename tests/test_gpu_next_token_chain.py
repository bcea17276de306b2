"""The calls from the residual to the next token in one run, as a decoder layer in FP8 and its head use them: norm, gate and
up, SwiGLU, down, norm, head, penalties and mask, the draw; its gradients; captured, and from two threads.

Bar: every step against its formula in 64 bits, from the values that the step was given, within the bounds of the step's own
tests; what runs through autograd, a graph or another stream bit for bit as the plain calls.
"""
import threading

import numpy as np
import pytest
import torch

import whallm_amd as wa
from running_error import Fp32, check
from test_gpu_block_norm import f64, want_grads
from test_gpu_fp8_rows import check_rows, want_norm, want_swiglu
from test_gpu_linear_fp8 import check as check_product, exact, spread
from test_gpu_process_logits import want_logits
from test_gpu_sample_logits import rule

pytestmark = pytest.mark.gpu
EPS = 1e-6


def stored(w):
    """A weight in E4M3 by blocks of 128 x 128, each scaled to its largest value."""
    N, K = w.shape
    pad = torch.nn.functional.pad(w, (0, -K % 128, 0, -N % 128))
    blocks = pad.view(pad.shape[0] // 128, 128, pad.shape[1] // 128, 128)
    s = blocks.abs().amax((1, 3)) / 448
    q = (blocks / s[:, None, :, None]).reshape(pad.shape)[:N, :K]
    return q.to(torch.float8_e4m3fn), s


def layer(device, T, H, I, V, seed):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *shape, std=1.0: torch.randn(*shape, generator=g) * std   # noqa: E731
    s = dict(residual=rand(T, H, std=2.0), y=rand(T, H, std=0.5).bfloat16(), norm=(1 + rand(H, std=0.2)).bfloat16(),
             last=(1 + rand(H, std=0.2)).bfloat16(), u=torch.rand(T, generator=g), top_k=torch.randint(0, 60, (T,), generator=g, dtype=torch.int32),
             top_p=torch.rand(T, generator=g), min_p=torch.rand(T, generator=g) * 0.05,
             mask=torch.randint(-2 ** 31, 2 ** 31 - 1, (1, -(-V // 32)), generator=g, dtype=torch.int32),
             temperature=0.3 + torch.rand(T, generator=g), history=torch.randint(0, V, (T, 30), generator=g, dtype=torch.int32),
             repetition=torch.full((T,), 1.2))
    for name, shape in (("gate_up", (2 * I, H)), ("down", (H, I)), ("head", (V, H))):
        s[name], s[name + "_scales"] = stored(rand(*shape, std=(3.0 if name == "head" else 1.0) * shape[1] ** -0.5))
    return {k: v.to(device) for k, v in s.items()}


def rules(s):
    return dict(history=s["history"], repetition=s["repetition"], mask=s["mask"])


def run(s):
    q, xs, r = wa.norm_fp8(s["residual"], s["y"], s["norm"], eps=EPS)
    gate_up = wa.linear_fp8(q, xs, s["gate_up"], s["gate_up_scales"])
    h, hs = wa.swiglu_fp8(gate_up)
    down = wa.linear_fp8(h, hs, s["down"], s["down_scales"])
    q2, xs2, r2, x2 = wa.norm_fp8(r, down, s["last"], eps=EPS, pow2_scales=True, with_x=True)
    raw = wa.linear_fp8(q2, xs2, s["head"], s["head_scales"], out_dtype=torch.float32)
    logits = wa.process_logits(raw, **rules(s))
    tokens, logp = wa.sample_logits(logits, s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return [q, xs, r, gate_up, h, hs, down, q2, xs2, r2, x2, raw, logits, tokens, logp]


def same(a, b):
    return all(torch.equal(x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x,
                           y.view(torch.uint8) if y.dtype == torch.float8_e4m3fn else y) for x, y in zip(a, b))


SHAPES = [(1, 256, 128, 2000), (6, 400, 208, 5003), (70, 512, 384, 2304)]


@pytest.mark.parametrize("T,H,I,V", SHAPES)
def test_each_step(device, T, H, I, V):
    s = layer(device, T, H, I, V, T)
    q, xs, r, gate_up, h, hs, down, q2, xs2, r2, x2, raw, logits, tokens, logp = run(s)

    def product(x, x_scales, name, y):
        want, size = exact(x, x_scales, s[name], s[name + "_scales"])
        check_product(y, want, size, x_scales.shape[1], y.dtype)

    check("residual", r, Fp32(f64(s["residual"])) + Fp32(f64(s["y"])))
    check_rows("norm", q, xs, want_norm(r, s["norm"], EPS, 0.0))
    product(q, xs, "gate_up", gate_up)
    check_rows("swiglu", h, hs, want_swiglu(gate_up, False, 0.0))
    product(h, hs, "down", down)
    check("second residual", r2, Fp32(f64(r)) + Fp32(f64(down)))
    check("x", x2, want_norm(r2, s["last"], EPS, 0.0))
    check_rows("second norm", q2, xs2, want_norm(r2, s["last"], EPS, 0.0), pow2=True)
    product(q2, xs2, "head", raw)
    check("logits", logits, want_logits(raw, **rules(s)))
    unit, clear = V * 2.0 ** -45, 0            # V sums of weights rounded to 2^-49 or finer, as the draw's own tests
    for t in range(T):
        value = lambda name: float(s[name][t])   # noqa: E731
        want, lp, near = rule(f64(logits[t]).astype(np.float32), value("u"), value("temperature"), int(s["top_k"][t]), value("top_p"),
                              value("min_p"))
        if near > unit:
            clear += 1
            assert int(tokens[t]) == want, t
            assert abs(float(logp[t]) - lp) <= 2.0 ** -23 * abs(lp) + 2 * unit
    assert clear >= 0.9 * T
    # the layer against itself without FP8: norms and products in 64 bits on the stored weights. Each of 3 roundings to E4M3 moves a
    # value by 2^-4 at most, a bf16 one by 2^-8, and the products' sums of many such keep well below the sum of both
    full = lambda n: s[n].double() * spread(spread(s[n + "_scales"], s[n].shape[1], 1), s[n].shape[0], 0).double()   # noqa: E731
    norm = lambda v, w: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * w.double()   # noqa: E731
    a = s["residual"].double() + s["y"].double()
    gu = norm(a, s["norm"]) @ full("gate_up").t().contiguous()
    act = torch.nn.functional.silu(gu[:, :I]) * gu[:, I:]
    b = a + act @ full("down").t().contiguous()
    off = (r2.double() - b).norm() / (b - a).norm()
    assert float(off) <= 3 * 2.0 ** -4


class Projection(torch.autograd.Function):
    """linear_fp8 of the normed residual, rounding passed through: dy in FP8 times the transposed weights, then the norm's."""
    @staticmethod
    def forward(ctx, residual, y, weight, w8, scales):
        q, xs, r = wa.norm_fp8(residual, y, weight, eps=EPS)
        ctx.save_for_backward(r, y, weight, w8, scales)
        return wa.linear_fp8(q, xs, w8, scales), r

    @staticmethod
    def backward(ctx, dout, dr):
        r, y, weight, w8, scales = ctx.saved_tensors
        dx = backward_product(dout, w8, scales)
        d = wa.block_norm_backward(dx, dr, r, y, pre_weight=weight, eps=EPS, post_norm=False)
        return d.residual, d.y, d.pre_weight.to(weight.dtype), None, None


def backward_product(dout, w8, scales):
    return wa.linear_fp8(*wa.quantize_fp8(dout), w8.view(torch.uint8).t().contiguous(), scales.t().contiguous())


@pytest.mark.parametrize("T,H,N", [(1, 128, 256), (37, 272, 400)])
def test_gradients(device, T, H, N):
    s = layer(device, T, H, N // 2, 64, 7)
    w8, scales = s["gate_up"], s["gate_up_scales"]
    leaves = [s[k].clone().requires_grad_() for k in ("residual", "y", "norm")]
    g = torch.Generator().manual_seed(2)
    dout, dr = torch.randn(T, N, generator=g).bfloat16().to(device), torch.randn(T, H, generator=g).to(device)
    out, r = Projection.apply(*leaves, w8, scales)
    torch.autograd.backward([out, r], [dout, dr])
    q, xs, r_plain = wa.norm_fp8(s["residual"], s["y"], s["norm"], eps=EPS)
    assert torch.equal(out, wa.linear_fp8(q, xs, w8, scales)) and torch.equal(r, r_plain)

    dq, ds = wa.quantize_fp8(dout)
    check_rows("dout", dq, ds, Fp32(f64(dout)))
    dx = backward_product(dout, w8, scales)
    full = w8.double() * spread(spread(scales, H, 1), N, 0).double()
    dq = dq.double() * spread(ds, N, 1).double()
    check_product(dx, dq @ full, dq.abs() @ full.abs(), ds.shape[1], torch.bfloat16)
    case = dict(residual=r.detach(), y=s["y"], post_weight=None, pre_weight=s["norm"], gate=None, weight_offset=0.0)
    want = want_grads(case, dx, dr, False, 1.0, EPS, False)
    with torch.no_grad():
        d = wa.block_norm_backward(dx, dr, r, s["y"], pre_weight=s["norm"], eps=EPS, post_norm=False)
    for name in ("residual", "y", "pre_weight"):
        check("d" + name, getattr(d, name), want[name])
    assert torch.equal(leaves[0].grad, d.residual) and torch.equal(leaves[1].grad, d.y)
    assert torch.equal(leaves[2].grad, d.pre_weight.bfloat16())

    # the formula against differences of <dx, v> + <dr, residual'> in 64 bits: central ones of a smooth function, off by the square
    # of the step
    rng = np.random.default_rng(3)
    a, w, c, e = f64(r), f64(s["norm"]), f64(dx), f64(dr)
    value = lambda a, w: (c * a / np.sqrt((a * a).mean(-1, keepdims=True) + EPS) * w).sum() + (e * a).sum()   # noqa: E731
    da, dw = rng.standard_normal(a.shape), rng.standard_normal(w.shape)
    h = 1e-4
    difference = (value(a + h * da, w + h * dw) - value(a - h * da, w - h * dw)) / (2 * h)
    terms = [want["residual"].v * da, want["pre_weight"].v * dw]
    assert abs(difference - sum(t.sum() for t in terms)) <= 1e-5 * sum(np.abs(t).sum() for t in terms)


def test_two_captured_runs(device):
    """Two graphs of the run, replayed in turn with new inputs and eager calls between, bit for bit as eager."""
    graphs = []
    for shape in SHAPES[:2]:
        s = layer(device, *shape, 11)
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            run(s)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(s)
        graphs.append((s, graph, outs))
    for step in range(4):
        for s, graph, outs in graphs:
            gen = torch.Generator().manual_seed(step)
            s["residual"].copy_(torch.randn(s["residual"].shape, generator=gen))
            s["u"].copy_(torch.rand(s["u"].shape, generator=gen))
            s["top_k"].copy_(torch.randint(0, 400, s["top_k"].shape, generator=gen))
            graph.replay()
        for s, graph, outs in graphs:
            assert same(outs, run(s)), step
        torch.cuda.synchronize(device)


def test_two_threads(device):
    """Each on its own stream, at the same time: the results of one alone."""
    states = [layer(device, *SHAPES[i], 5) for i in (1, 2)]
    want = [run(s) for s in states]
    torch.cuda.synchronize(device)
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(device)):
                for _ in range(10):
                    out = run(states[i])
                    torch.cuda.current_stream(device).synchronize()
                    if not same(out, want[i]):
                        bad.append(i)
        except Exception as e:   # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_inference_mode_and_grad_mode(device):
    s = layer(device, *SHAPES[1], 9)
    want = run(s)
    with torch.inference_mode():
        got = run(s)
        assert all(t.is_inference() for t in got) and same(want, got)
    s["residual"].requires_grad_()
    with pytest.raises(ValueError, match="autograd"):
        run(s)
    with torch.no_grad():
        assert same(want, run(s))
    s["residual"].requires_grad_(False)
    kept = s["residual"].clone()
    wa.norm_fp8(kept, s["y"], s["norm"], residual_out=kept)
    assert torch.equal(kept, want[2]) and kept._version > 0
