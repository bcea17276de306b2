"""GPU parity of the 8-bit rows (wm_norm_fp8, wm_fp8_rows) against their formulas in 64 bits.

Bar: the running error of the same steps in fp32 (running_error.py); a block's scale within its values' error, one
division and, with pow2, the next power of two of either end; a value within half a step of E4M3 from what it
stands for (2^-4 of it, 2^-10 scales below the smallest normal number) and the two roundings of v / s. Where scales
are powers of two and rows are as given, v / s is exact and the bytes have to be torch's. The silu is x times the
reciprocal of 1 + exp(-x), whose exponential is good to 4 units with its argument's rounding. A row's sum passes at
most 16 columns of a thread, 6 steps of a wave and 16 waves.
"""
import numpy as np
import pytest
import torch

import whallm_amd as wa
from running_error import U, Fp32, check

pytestmark = pytest.mark.gpu

ROW = 16 + 6 + 16 + 1
BLOCK = 128
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def f64(t):
    return t.detach().double().cpu().numpy()


def randn(rng, shape, dtype, device, std=1.0, mean=0.0):
    return torch.from_numpy((rng.standard_normal(shape) * std + mean).astype(np.float32)).to(dtype).to(device)


def blocks_max(v):
    """[T, W] -> [T, ceil(W / 128)]: each block's largest value."""
    T, W = v.shape
    pad = np.zeros((T, -W % BLOCK))
    return np.concatenate([v, pad], 1).reshape(T, -1, BLOCK).max(2)


def next_pow2(s):
    return 2.0 ** np.ceil(np.log2(s))


def check_rows(name, q, scales, want, pow2=False):
    """q, scales of rows ``want`` (an Fp32 value: 64 bits and a bound)."""
    v, e = want.v, want.e
    T, W = v.shape
    assert q.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32
    assert tuple(q.shape)[-1] == W and tuple(scales.shape)[-1] == -(-W // BLOCK)
    s = f64(scales).reshape(T, -1)
    low = np.maximum(blocks_max(np.maximum(np.abs(v) - e, 0)) / 448 * (1 - U), 2.0 ** -126)
    high = np.maximum(blocks_max(np.abs(v) + e) / 448 * (1 + U), 2.0 ** -126)
    if pow2:
        low, high = next_pow2(low * (1 - U)), next_pow2(high)
        assert (np.log2(s) % 1 == 0).all(), name
    assert (s >= low * (1 - U)).all() and (s <= high * (1 + U)).all(), (name, "scales")
    each = np.repeat(s, BLOCK, 1)[:, :W]
    got = f64(q.float()).reshape(T, W) * each
    bound = np.maximum(2.0 ** -4 * np.abs(v), 2.0 ** -10 * each) + (e + 4 * U * np.abs(v)) * (1 + 2.0 ** -4)
    off = np.abs(got - v)
    assert (off <= bound).all(), (name, int((off > bound).sum()), float((off / bound).max()))


# ----------------------------------------------------------------------------- norm

def want_norm(r, w, eps, offset):
    r = Fp32(f64(r).reshape(-1, r.shape[-1]))
    weight = Fp32(1.0) if w is None else Fp32(f64(w)) + Fp32(np.float32(offset))
    return r * (((r * r).mean(ROW) + eps).rsqrt() * weight)


def run_norm(device, T, H, residual="fp32", add=True, weight=True, offset=0.0, eps=1e-6, pow2=False, std=2.0, seed=None):
    rng = np.random.default_rng([T, H] if seed is None else seed)
    r = randn(rng, (T, H), TYPES[residual], device, std)
    y = randn(rng, (T, H), torch.bfloat16, device, std / 4) if add else None
    w = randn(rng, (H,), torch.bfloat16, device, 0.2, 1 - offset) if weight else None
    keep = [None if t is None else t.clone() for t in (r, y, w)]
    q, s, out, x = wa.norm_fp8(r, y, w, eps=eps, weight_offset=offset, pow2_scales=pow2, with_x=True)
    assert all(a is None or torch.equal(a, b) for a, b in zip(keep, (r, y, w)))
    if add:
        check("residual", out, Fp32(f64(r)) + Fp32(f64(y)))
    else:
        assert out is r
    want = want_norm(out, w, eps, offset)
    check("x", x, want)
    check_rows("norm", q, s, want, pow2)
    again = wa.norm_fp8(r, y, w, eps=eps, weight_offset=offset, pow2_scales=pow2)
    assert len(again) == 3 and torch.equal(again[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(again[1], s)


@pytest.mark.parametrize("residual", ["fp32", "bf16"])
@pytest.mark.parametrize("T,H", [(1, 7168), (1, 1), (3, 7), (5, 127), (4, 128), (2, 129), (7, 500), (300, 96), (33, 512), (9, 520),
                                 (70, 2560), (6, 4097), (3, 8192), (3, 8200), (2, 16384), (2, 16383), (1100, 1024)])
def test_norm(device, T, H, residual):
    run_norm(device, T, H, residual)


@pytest.mark.parametrize("kw", [dict(add=False), dict(weight=False), dict(offset=1.0), dict(pow2=True), dict(eps=0.0),
                                dict(add=False, weight=False, residual="bf16", pow2=True), dict(std=1e12), dict(std=1e-12, eps=0.0)])
def test_norm_forms(device, kw):
    run_norm(device, 6, 1000, **kw)


def test_norm_in_place_strides_and_batches(device):
    rng = np.random.default_rng(5)
    r, y = randn(rng, (2, 3, 640), torch.float32, device), randn(rng, (2, 3, 640), torch.bfloat16, device)
    w = randn(rng, (640,), torch.bfloat16, device)
    q, s, out = wa.norm_fp8(r, y, w)
    assert q.shape == (2, 3, 640) and s.shape == (2, 3, 5) and out.shape == r.shape
    same = r.clone()
    version = same._version
    got = wa.norm_fp8(same, y, w, residual_out=same)
    assert got[2] is same and same._version == version + 1 and torch.equal(same, out)
    wide = torch.zeros(2, 3, 1283, device=device)[..., 1:1281:2]
    wide.copy_(r)
    odd = torch.zeros(2 * 3 * 640 + 1, dtype=torch.bfloat16, device=device)[1:].view(2, 3, 640)   # 2 bytes past 16
    odd.copy_(y)
    for a, b in zip(wa.norm_fp8(wide, odd, w), (q, s, out)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    with pytest.raises(ValueError, match="share no memory"):
        wa.norm_fp8(r.bfloat16(), y, residual_out=y)


# ----------------------------------------------------------------------------- rows and gated activations

@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("T,W", [(1, 1), (1, 128), (5, 7), (3, 129), (2, 136), (300, 96), (17, 1000), (64, 2048), (2100, 4096),
                                 (1200, 8100)])
def test_rows(device, T, W, dtype, pow2):
    rng = np.random.default_rng([T, W])
    x = randn(rng, (T, W), TYPES[dtype], device, 3.0) * torch.from_numpy(2.0 ** rng.integers(-30, 30, (T, 1))).to(device).to(TYPES[dtype])
    q, s = wa.quantize_fp8(x, pow2_scales=pow2)
    check_rows("rows", q, s, Fp32(f64(x)), pow2)
    blocks = torch.nn.functional.pad(x.double(), (0, -W % BLOCK)).view(T, -1, BLOCK)
    # the maximum is exact; a tensor divides (torch takes a number's reciprocal)
    plain = (blocks.abs().amax(2).float() / torch.full((), 448.0, device=device)).clamp(min=2.0 ** -126)
    if pow2:
        plain = torch.exp2(torch.ceil(torch.log2(plain.double()))).float()
        bytes_ = (blocks / plain.double()[..., None]).view(T, -1)[:, :W].to(torch.float8_e4m3fn)
        assert torch.equal(q.view(torch.uint8), bytes_.view(torch.uint8))
    assert torch.equal(s, plain)


def want_swiglu(x, up_first, limit):
    v = f64(x)
    W = v.shape[1] // 2
    gate, up = (v[:, W:], v[:, :W]) if up_first else (v[:, :W], v[:, W:])
    if limit:
        gate, up = np.minimum(gate, limit), np.clip(up, -limit, limit)
    silu = gate / (1 + np.exp(-gate))
    return Fp32(silu, 10 * U * np.abs(silu) + 1e-38) * Fp32(up)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("up_first,limit,pow2", [(False, 0.0, False), (True, 0.0, False), (False, 2.0, False), (True, 2.0, True)])
@pytest.mark.parametrize("T,W", [(1, 2048), (1, 1), (6, 13), (3, 129), (64, 640), (1500, 2304), (1000, 8191)])
def test_swiglu(device, T, W, up_first, limit, pow2, dtype):
    rng = np.random.default_rng([T, W, 3])
    x = randn(rng, (T, 2 * W), TYPES[dtype], device, 3.0)
    q, s = wa.swiglu_fp8(x, up_first=up_first, limit=limit, pow2_scales=pow2)
    check_rows("swiglu", q, s, want_swiglu(x, up_first, limit), pow2)


def test_swiglu_far_gates(device):
    """Gates past the exponential's range: silu is the gate itself, or nothing."""
    gate = torch.tensor([-3e38, -1e4, -89.0, -60.0, 60.0, 89.0, 1e4, 3e38], device=device)
    q, s = wa.swiglu_fp8(torch.cat([gate.repeat(128, 1).t(), torch.ones(8, 128, device=device)], 1))
    got = q.float() * s
    want = torch.where(gate > 0, gate, gate * torch.exp(gate.double()).float())
    assert (got[4:] - want[4:, None]).abs().le(2.0 ** -4 * want[4:, None].abs()).all()
    assert got[:4].abs().max() < 1e-20


def test_zeros_tiny_and_nan(device):
    x = torch.zeros(4, 384, device=device)
    x[1, 130] = float("nan")
    x[2, 0], x[2, 1] = float("inf"), 5.0
    x[3, :128] = 2.0 ** -149
    q, s = wa.quantize_fp8(x)
    assert (s[0] == 2.0 ** -126).all() and (q[0].view(torch.uint8) == 0).all()
    assert s[1].isnan().tolist() == [False, True, False] and q[1, 128:256].float().isnan().all() and (q[1, :128].float() == 0).all()
    assert s[2, 0].isinf() and q[2, 0].float().isnan() and q[2, 1].float() == 0
    assert s[3, 0] == 2.0 ** -126 and (q[3].float() == 0).all()
    q, s, _ = wa.norm_fp8(torch.zeros(2, 300, device=device), torch.zeros(2, 300, dtype=torch.bfloat16, device=device))
    assert (q.float() == 0).all() and (s == 2.0 ** -126).all()


def test_empty(device):
    for shape in ((0, 64), (2, 0, 64)):
        x = torch.zeros(shape, device=device)
        for q, s in (wa.quantize_fp8(x), wa.swiglu_fp8(torch.cat([x, x], -1)), wa.norm_fp8(x, x.bfloat16())[:2]):
            assert q.shape == shape and s.shape == (*shape[:-1], 1)


def test_side_stream_and_graph(device):
    rng = np.random.default_rng(9)
    r, y = randn(rng, (40, 1024), torch.float32, device), randn(rng, (40, 1024), torch.bfloat16, device)

    def step():
        q, s, out = wa.norm_fp8(r, y)
        return (q, s, out, *wa.swiglu_fp8(out), *wa.quantize_fp8(y, pow2_scales=True))

    bits = lambda ts: [t.clone().view(torch.uint8) for t in ts]   # noqa: E731
    eager = bits(step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(bits(other), eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        r.mul_(-1)
        y.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(bits(captured), bits(step()))), k


def test_past_32_bits(device):
    """The last rows of more than 2^31 elements."""
    T, W = 131100, 16384
    x = torch.empty(T, W, dtype=torch.bfloat16, device=device)
    x[-3:].normal_()
    q, s = wa.quantize_fp8(x)
    a, b = wa.quantize_fp8(x[-3:].clone())
    assert torch.equal(q[-3:].view(torch.uint8), a.view(torch.uint8)) and torch.equal(s[-3:], b)
    del q, s
    q, s, r, = wa.norm_fp8(x, x)
    a, b, c = wa.norm_fp8(x[-3:].clone(), x[-3:].clone())
    assert torch.equal(q[-3:].view(torch.uint8), a.view(torch.uint8)) and torch.equal(s[-3:], b) and torch.equal(r[-3:], c)
