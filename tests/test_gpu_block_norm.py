"""GPU parity of the norms around a block (wm_block_norm) and their gradients
(wm_block_norm_backward) against the formulas in 64 bits.

Bar: the running error of the same steps in fp32 (running_error.py) and one rounding to the
output's type. x is held against the norm of the residual as the kernel stored it. A row's sums pass
at most 16 columns of a thread, 6 steps of a wave and 16 waves; a sum over T tokens passes the
tokens of a thread group, at most T / 256 + 1 (with fewer than 256 groups it is one token a group),
16 groups of a workgroup, 64 of at most 1024 workgroups and 16 slices.
"""
import numpy as np
import pytest
import torch

import whallm_amd as wa
from running_error import Fp32, check

pytestmark = pytest.mark.gpu

ROW = 16 + 6 + 16 + 1
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def f64(t):
    return t.detach().double().cpu().numpy()


def randn(rng, shape, dtype, device, std=1.0, mean=0.0):
    return torch.from_numpy((rng.standard_normal(shape) * std + mean).astype(np.float32)).to(dtype).to(device)


def make(rng, T, H, device, residual="fp32", gate=None, gate_type="fp32", post=True, pre=True, offset=0.0):
    rt = TYPES[residual]
    s = dict(residual=randn(rng, (T, H), rt, device, 2.0), y=randn(rng, (T, H), torch.bfloat16, device, 0.5),
             post_weight=randn(rng, (H,), torch.bfloat16, device, 0.2, 1 - offset) if post else None,
             pre_weight=randn(rng, (H,), torch.bfloat16, device, 0.2, 1 - offset) if pre else None,
             gate=None, weight_offset=offset)
    if gate:
        s["gate"] = randn(rng, {"token": (T, 1), "channel": (H,), "full": (T, H)}[gate], TYPES[gate_type], device)
    return s


def weight(w, offset):
    return Fp32(1.0) if w is None else Fp32(f64(w)) + Fp32(offset)


def gate_value(s, sigmoid):
    if s["gate"] is None:
        return Fp32(1.0)
    g = Fp32(f64(s["gate"]))
    return g.sigmoid() if sigmoid else g


def want_forward(s, sigmoid, scale, eps, post_norm):
    y = Fp32(f64(s["y"]))
    z = y
    if post_norm:
        z = y * ((y * y).mean(ROW) + eps).rsqrt() * weight(s["post_weight"], s["weight_offset"])
    return Fp32(f64(s["residual"])) + z * gate_value(s, sigmoid) * scale


def want_x(residual_out, s, eps):
    r = Fp32(f64(residual_out))
    return r * ((r * r).mean(ROW) + eps).rsqrt() * weight(s["pre_weight"], s["weight_offset"])


def want_grads(s, dx, dres, sigmoid, scale, eps, post_norm):
    """s['residual'] is the residual behind the block."""
    T = s["y"].shape[0]
    tokens = T // 256 + 1 + 16 + 64 + 16
    r, y, dx = Fp32(f64(s["residual"])), Fp32(f64(s["y"])), Fp32(f64(dx))
    wpre, wpost = weight(s["pre_weight"], s["weight_offset"]), weight(s["post_weight"], s["weight_offset"])
    q = ((r * r).mean(ROW) + eps).rsqrt()
    a = dx * wpre
    dr = (Fp32(0.0) if dres is None else Fp32(f64(dres))) + q * a - r * (q * q * q * (a * r).mean(ROW))
    p = ((y * y).mean(ROW) + eps).rsqrt() if post_norm else Fp32(1.0)
    g = gate_value(s, sigmoid)
    b = dr * scale * g
    n = y * p
    c = b * wpost
    dy = p * c - y * (p * p * p * (c * y).mean(ROW)) if post_norm else c
    out = {"residual": dr, "y": dy, "post_weight": None if s["post_weight"] is None else (b * n).sum(0, tokens),
           "pre_weight": None if s["pre_weight"] is None else (dx * r * q).sum(0, tokens), "gate": None}
    if s["gate"] is not None:
        dg = dr * scale * (n * wpost)
        if sigmoid:
            dg = dg * (g * (Fp32(1.0) - g))
        shape = tuple(s["gate"].shape)
        out["gate"] = dg.sum(0, tokens) if len(shape) == 1 else dg if shape == tuple(s["y"].shape) else dg.sum(-1, ROW, True)
    return out


def run_case(device, seed, T, H, residual="fp32", gate=None, gate_type="fp32", sigmoid=False, post_norm=True, post=True, pre=True,
             offset=0.0, scale=0.7, eps=1e-6, with_dres=True):
    rng = np.random.default_rng(seed)
    s = make(rng, T, H, device, residual, gate, gate_type, post and post_norm, pre, offset)
    how = dict(gate_sigmoid=sigmoid, scale=scale, eps=eps, post_norm=post_norm)
    before = {k: v.clone() for k, v in s.items() if torch.is_tensor(v)}
    x, r_out = wa.block_norm(**s, **how)
    assert x.dtype == torch.bfloat16 and r_out.dtype == s["residual"].dtype
    check("residual", r_out, want_forward(s, sigmoid, scale, eps, post_norm))
    check("x", x, want_x(r_out, s, eps))
    dx = randn(rng, (T, H), torch.bfloat16, device)
    dres = randn(rng, (T, H), s["residual"].dtype, device, 0.5) if with_dres else None
    assert all(torch.equal(s[k], v) for k, v in before.items())
    s["residual"] = r_out
    args = {k: v for k, v in s.items() if k != "residual"}
    d = wa.block_norm_backward(dx, dres, r_out, **args, **how)
    want = want_grads(s, dx, dres, sigmoid, scale, eps, post_norm)
    for name in ("residual", "y", "post_weight", "pre_weight", "gate"):
        got = getattr(d, name)
        assert (got is None) == (want[name] is None), name
        if got is not None:
            check("d" + name, got, want[name])
    return s, (x, r_out), d


@pytest.mark.parametrize("H", [1, 7, 8, 96, 511, 1000, 2048, 2051, 4104, 7168, 8200, 9001, 16384])
@pytest.mark.parametrize("T", [1, 5])
def test_sizes(device, T, H):
    run_case(device, H + T, T, H, gate="channel", residual="fp32")
    run_case(device, H + T + 1, T, H, gate="full", gate_type="bf16", residual="bf16", offset=1.0)


@pytest.mark.parametrize("gate,gate_type,sigmoid", [(None, "fp32", False), ("token", "fp32", True), ("token", "bf16", False),
                                                    ("channel", "bf16", True), ("channel", "fp32", False),
                                                    ("full", "bf16", True), ("full", "fp32", False)])
@pytest.mark.parametrize("residual", ["fp32", "bf16"])
def test_gates(device, gate, gate_type, sigmoid, residual):
    run_case(device, 3, 37, 264, residual, gate, gate_type, sigmoid)
    run_case(device, 4, 37, 75, residual, gate, gate_type, sigmoid, offset=1.0)


@pytest.mark.parametrize("kw", [dict(post_norm=False), dict(post=False), dict(pre=False), dict(with_dres=False),
                                dict(post_norm=False, pre=False, gate="token", sigmoid=True), dict(scale=0.0), dict(eps=0.5)])
def test_forms(device, kw):
    run_case(device, 6, 130, 520, **kw)
    run_case(device, 7, 3, 33, residual="bf16", **kw)


@pytest.mark.parametrize("T,H,residual", [(1500, 640, "fp32"), (2049, 130, "bf16"), (4500, 72, "fp32")])
def test_many_tokens(device, T, H, residual):
    """More tokens than workgroups: rows and sums over tokens of the later rounds."""
    run_case(device, T, T, H, residual, gate="channel")
    run_case(device, T + 1, T, H, residual, gate="token", sigmoid=True)


def test_rows_of_zeros_and_extremes(device):
    """A zero y and a zero residual norm to zero (eps), large rows stay finite."""
    T, H = 4, 128
    r = torch.zeros(T, H, device=device)
    y = torch.zeros(T, H, dtype=torch.bfloat16, device=device)
    x, out = wa.block_norm(r, y)
    assert not x.any() and not out.any()
    y[1], y[2] = 1e15, 1e-20
    r[3] = -1e18
    x, out = wa.block_norm(r, y, scale=2.0)
    check("residual", out, want_forward(dict(residual=r, y=y, post_weight=None, gate=None, weight_offset=0.0), False, 2.0, 1e-6, True))
    assert torch.isfinite(x.float()).all() and torch.equal(x[3], torch.full((H,), -1.0, dtype=torch.bfloat16, device=device))
    # a NaN stays in its row
    y[0, 5] = float("nan")
    x2, out2 = wa.block_norm(r, y, scale=2.0)
    assert torch.isnan(x2[0].float()).all() and torch.equal(x2[1:], x[1:]) and torch.equal(out2[1:], out[1:])


def test_in_place_strided_unaligned_and_no_tokens(device):
    rng = np.random.default_rng(8)
    T, H = 19, 264
    s = make(rng, T, H, device, gate="full", gate_type="bf16")
    x, out = wa.block_norm(**s)
    mine = dict(s, residual=s["residual"].clone())
    x2, same = wa.block_norm(**mine, residual_out=mine["residual"])
    assert same is mine["residual"] and torch.equal(same, out) and torch.equal(x2, x)
    wide = torch.zeros(T, 2 * H, dtype=torch.bfloat16, device=device)
    wide[:, ::2] = s["y"]
    batched = {k: v.view(1, T, H) for k, v in s.items() if k in ("residual", "gate")}
    x3, out3 = wa.block_norm(**dict(s, y=wide[:, ::2].unsqueeze(0), **batched))
    assert x3.shape == (1, T, H) and torch.equal(x3[0], x) and torch.equal(out3[0], out)
    off = torch.empty(T * H + 1, dtype=torch.bfloat16, device=device)[1:].view(T, H).copy_(s["y"])
    x4, out4 = wa.block_norm(**dict(s, y=off))     # value by value: the sums' order may differ
    check("residual", out4, want_forward(s, False, 1.0, 1e-6, True))
    check("x", x4, want_x(out4, s, 1e-6))
    none = {k: (v[:0] if torch.is_tensor(v) and v.dim() == 2 else v) for k, v in s.items()}
    x5, out5 = wa.block_norm(**none)
    assert x5.shape == (0, H)
    args = {k: v for k, v in none.items() if k != "residual"}
    d = wa.block_norm_backward(x5, None, out5, **args)
    assert d.y.shape == (0, H) and not d.post_weight.any() and not d.pre_weight.any() and d.gate.shape == (0, H)


def test_agrees_with_residual_rmsnorm(device):
    """Without the post norm, gate and weights it is the framework's residual add and norm."""
    rng = np.random.default_rng(10)
    r, y = randn(rng, (9, 2048), torch.float32, device), randn(rng, (9, 2048), torch.bfloat16, device)
    x, out = wa.block_norm(r, y, post_norm=False)
    from whallm_amd.ops import residual_rmsnorm
    r2 = r.clone()
    x2 = residual_rmsnorm(r2, y)
    assert torch.equal(out, r2)
    assert (x != x2).float().mean() <= 1e-3    # the sums' order differs: a value on a rounding border moves


def test_gradients_against_differences(device):
    """Along a direction, the difference quotient of <residual', u> + <x, dx> is the gradients' product with
    the direction. x is bf16 (each value off by half a step, 2^-8), so the quotient of H T values of
    about 1 times dx of about 1 is off by about sqrt(H T) 2^-8 / step: held to six of these."""
    rng = np.random.default_rng(12)
    T, H, step = 16, 512, 0.25
    s = make(rng, T, H, device, gate="token", gate_type="fp32")
    how = dict(gate_sigmoid=True, scale=0.9, eps=1e-6)
    dx, u = randn(rng, (T, H), torch.bfloat16, device), randn(rng, (T, H), torch.float32, device)
    x, out = wa.block_norm(**s, **how)
    args = {k: v for k, v in s.items() if k != "residual"}
    d = wa.block_norm_backward(dx, u, out, **args, **how)

    def value(**kw):
        x, out = wa.block_norm(**dict(s, **kw), **how)
        return float((x.double() * dx.double()).sum() + (out.double() * u.double()).sum())

    noise = 6 * (T * H) ** 0.5 * 2.0 ** -8 / step
    for name, grad in (("residual", d.residual), ("gate", d.gate)):
        v = randn(rng, tuple(s[name].shape), torch.float32, device)
        v *= 0.05 if name == "residual" else 0.2
        got = (value(**{name: s[name] + step * v}) - value(**{name: s[name] - step * v})) / (2 * step)
        want = float((grad.double() * v.double()).sum())
        assert abs(got - want) <= noise + 0.02 * abs(want), (name, got, want)


def test_other_stream_and_graph_replays(device):
    rng = np.random.default_rng(14)
    for T, H in ((1, 2048), (600, 320)):
        s = make(rng, T, H, device, gate="channel")
        dx, dres = randn(rng, (T, H), torch.bfloat16, device), randn(rng, (T, H), torch.float32, device)
        args = {k: v for k, v in s.items() if k != "residual"}

        def step():
            x, out = wa.block_norm(**s)
            d = wa.block_norm_backward(dx, dres, out, **args)
            return x, out, d.residual, d.y, d.post_weight, d.pre_weight, d.gate

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for k in range(3):
            if k:
                s["residual"].copy_(randn(rng, (T, H), torch.float32, device))
                s["y"].copy_(randn(rng, (T, H), torch.bfloat16, device))
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
            if k == 0:
                assert all(torch.equal(a, b) for a, b in zip(outs, first))


def test_offsets_past_2_31_elements(device):
    """Rows far into a tensor give what the same rows give by themselves, bit for bit."""
    T, H, last = 131100, 16384, 3
    gen = torch.Generator(device).manual_seed(2)
    y = torch.randn(T, H, generator=gen, device=device, dtype=torch.bfloat16)
    w = torch.ones(H, device=device, dtype=torch.bfloat16)
    x, r = wa.block_norm(y, y, w, w, y)
    xl, rl = wa.block_norm(y[-last:], y[-last:], w, w, y[-last:])
    assert torch.equal(x[-last:], xl) and torch.equal(r[-last:], rl)
    d = wa.block_norm_backward(x, y, r, y, w, w, y)
    dl = wa.block_norm_backward(xl, y[-last:], rl, y[-last:], w, w, y[-last:])
    for name in ("residual", "y", "gate"):
        assert torch.equal(getattr(d, name)[-last:], getattr(dl, name)), name


@pytest.mark.parametrize("T,H,residual", [(5, 96, "fp32"), (300, 1000, "bf16"), (700, 6152, "bf16"), (3, 9000, "fp32")])
def test_gradients_written_over_what_came_in(device, T, H, residual):
    """The C call's dresidual may be dresidual_out and its dy may be dx."""
    from whallm_amd import _lib
    rng = np.random.default_rng(H)
    s = make(rng, T, H, device, residual, gate="full", gate_type="bf16")
    dx, dres = randn(rng, (T, H), torch.bfloat16, device), randn(rng, (T, H), TYPES[residual], device)
    r_out = s.pop("residual")
    want = wa.block_norm_backward(dx, dres, r_out, **s)
    dpost, dpre, dgate = torch.empty(H, device=device), torch.empty(H, device=device), torch.empty_like(s["gate"])
    form = _lib.BlockNormFormC(s["post_weight"].data_ptr(), s["pre_weight"].data_ptr(), s["gate"].data_ptr(), 0.0, 1.0, 1e-6, 1, 3, 0,
                               0, int(residual == "fp32"))
    ws = torch.empty(_lib.load().wm_block_norm_backward_workspace_size(T, H), dtype=torch.uint8, device=device)
    _lib.call("wm_block_norm_backward", form, dx.data_ptr(), dres.data_ptr(), r_out.data_ptr(), s["y"].data_ptr(), T, H, dres.data_ptr(),
              dx.data_ptr(), dpost.data_ptr(), dpre.data_ptr(), dgate.data_ptr(), ws.data_ptr(), ws.numel(),
              torch.cuda.current_stream(device).cuda_stream)
    for got, name in ((dres, "residual"), (dx, "y"), (dpost, "post_weight"), (dpre, "pre_weight"), (dgate, "gate")):
        assert torch.equal(got, getattr(want, name)), name
