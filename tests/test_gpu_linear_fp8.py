"""GPU parity of the FP8 product with block scales (wm_linear_fp8) against its formula in 64 bits.

Bar, with S the sum of the magnitudes |xs ws x w| over K: a block's 128 products, the two scales' product, its
multiply-add and the sums over blocks and waves pass at most 128 + 4 + blocks + 8 roundings of fp32, so an
output is off by (140 + blocks) 2^-24 S and one rounding to its type; the FP8 matrix instructions, behind bf16
outputs, keep a block's sum to 2^-12 of its magnitudes besides. Whole numbers with power-of-two scales have exact sums on either
way, and then have to be equal.
"""
import ctypes

import numpy as np
import pytest
import torch

import whallm_amd as wa
from whallm_amd import _lib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def spread(scales, n, dim):
    return scales.repeat_interleave(128, dim).narrow(dim, 0, n)


def make(device, M, N, K, seed=0, whole=False):
    g = torch.Generator().manual_seed(seed)
    nb, kb = -(-N // 128), -(-K // 128)
    if whole:
        x, w = torch.randint(-4, 5, (M, K), generator=g).float(), torch.randint(-4, 5, (N, K), generator=g).float()
        xs = 2.0 ** torch.randint(-3, 4, (M, kb), generator=g).float()
        ws = 2.0 ** torch.randint(-3, 4, (nb, kb), generator=g).float()
    else:
        x, w = torch.randn(M, K, generator=g) * 60, torch.randn(N, K, generator=g) * 60
        xs, ws = torch.rand(M, kb, generator=g) * 0.02 + 1e-3, torch.rand(nb, kb, generator=g) * 1e-3 + 1e-4
    f8 = torch.float8_e4m3fn
    return x.to(f8).to(device), xs.to(device), w.to(f8).to(device), ws.to(device)


def exact(x, xs, w, ws, add=None):
    """(64-bit result, sum of magnitudes)."""
    N, K = w.shape
    a = x.float().double() * spread(xs, K, 1).double()
    b = w.float().double() * spread(spread(ws, K, 1), N, 0).double()
    y, s = a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    return (y, s) if add is None else (y + add.double(), s + add.double().abs())


def check(y, want, S, blocks, dtype):
    e = (140 + blocks) * U * S
    if dtype == torch.bfloat16:
        e = e + 2.0 ** -12 * S
    bound = e + torch.finfo(dtype).eps / 2 * (want.abs() + e) + 1e-37
    off = (y.double() - want).abs()
    assert y.dtype == dtype and y.shape == want.shape
    assert bool((off <= bound).all()), (int((off > bound).sum()), float((off / bound).max()))


def run(device, M, N, K, out, with_add=False, whole=False):
    x, xs, w, ws = make(device, M, N, K, M * 31 + N * 7 + K, whole)
    dt = TYPES[out]
    add = (torch.randint(-8, 9, (M, N), device=device).to(dt) if whole else torch.randn(M, N, device=device).to(dt)) if with_add else None
    y = wa.linear_fp8(x, xs, w, ws, out_dtype=dt, add=add)
    want, S = exact(x, xs, w, ws, add)
    if whole:
        assert torch.equal(y, want.to(torch.float32).to(dt)), int((y != want.to(torch.float32).to(dt)).sum())
    else:
        check(y, want, S, xs.shape[1], dt)


@pytest.mark.parametrize("out", ["bf16", "fp32"])
@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 16), (1, 16, 128), (1, 4096, 7168), (2, 17, 144), (3, 129, 32), (5, 1000, 1040), (15, 127, 2560), (16, 257, 112),
    (6, 20000, 512), (9, 16389, 400), (17, 128, 256), (31, 1003, 640), (32, 64, 48), (33, 130, 1168), (64, 515, 896),
    (65, 64, 128), (96, 4608, 512), (127, 1, 528), (128, 192, 1280), (129, 65, 80), (200, 1283, 2560), (600, 333, 144)])
def test_shapes(device, M, N, K, whole, out):
    run(device, M, N, K, out, with_add=(M + N) % 3 == 0, whole=whole)


@pytest.mark.parametrize("out", ["bf16", "fp32"])
@pytest.mark.parametrize("M,N,K", [(2100, 2200, 400), (1300, 3333, 528), (1025, 8200, 256), (4100, 4112, 272), (5000, 4099, 128),
                                   (8200, 2052, 640)])
def test_many_tokens(device, M, N, K, out):
    run(device, M, N, K, out, with_add=N % 2 == 1, whole=False)
    run(device, M, N, K, out, with_add=N % 2 == 0, whole=True)


@pytest.mark.parametrize("out", ["bf16", "fp32"])
@pytest.mark.parametrize("M,N,K", [(40, 25003, 4112), (64, 24576, 4096), (100, 25001, 4112), (128, 24640, 4224)])
def test_weights_past_the_caches(device, M, N, K, out):
    """One token tile and 100 MB of weights or more: odd and whole numbers of blocks and rows."""
    run(device, M, N, K, out, with_add=N % 2 == 1, whole=True)
    run(device, M, N, K, out, with_add=N % 2 == 0, whole=False)


@pytest.mark.parametrize("M", [1, 20, 50, 100, 700])
def test_forms_of_the_inputs(device, M):
    """uint8, batch dims, strides, views off 16 bytes, no tokens: the same bits."""
    N, K = 260, 400
    x, xs, w, ws = make(device, M, N, K, M)
    for dt in (torch.bfloat16, torch.float32):
        y = wa.linear_fp8(x, xs, w, ws, out_dtype=dt)
        assert torch.equal(wa.linear_fp8(x.view(torch.uint8), xs, w.view(torch.uint8), ws, out_dtype=dt), y)
        assert torch.equal(wa.linear_fp8(x[None], xs[None], w, ws, out_dtype=dt), y[None])
        wide = torch.zeros(M, 2 * K, dtype=torch.uint8, device=device)
        wide[:, ::2] = x.view(torch.uint8)
        assert torch.equal(wa.linear_fp8(wide[:, ::2], xs.t().contiguous().t(), w, ws, out_dtype=dt), y)
        shift = torch.zeros(M * K + 1, dtype=torch.uint8, device=device)[1:].view(M, K)
        shift.copy_(x.view(torch.uint8))
        wshift = torch.zeros(N * K + 3, dtype=torch.uint8, device=device)[3:].view(N, K)
        wshift.copy_(w.view(torch.uint8))
        assert torch.equal(wa.linear_fp8(shift, xs, wshift, ws, out_dtype=dt), y)
        add = torch.randn(M * N + 1, device=device).to(dt)
        assert torch.equal(wa.linear_fp8(x, xs, w, ws, out_dtype=dt, add=add[1:].view(M, N)),
                           wa.linear_fp8(x, xs, w, ws, out_dtype=dt, add=add[1:].view(M, N).clone()))
        assert wa.linear_fp8(x[:0], xs[:0], w, ws, out_dtype=dt).shape == (0, N)


@pytest.mark.parametrize("out", ["bf16", "fp32"])
@pytest.mark.parametrize("M,N,K", [(3, 37, 144), (40, 37, 272), (90, 130, 144), (2100, 2202, 144), (5000, 4099, 144)])
def test_writes_its_outputs_and_no_others(device, M, N, K, out):
    """Also with out in the place of add."""
    x, xs, w, ws = make(device, M, N, K, 5, True)
    dt = TYPES[out]
    for add in (False, True):
        buffer = torch.full((M * N + 256,), 77.0, dtype=dt, device=device)
        y = buffer[128:-128]
        y.fill_(3.0)
        at = ctypes.c_void_p(y.data_ptr())
        _lib.call("wm_linear_fp8", x.data_ptr(), xs.data_ptr(), M, K, w.data_ptr(), ws.data_ptr(), N, at if add else None,
                  int(out == "fp32"), at, torch.cuda.current_stream().cuda_stream)
        want = exact(x, xs, w, ws)[0] + (3.0 if add else 0.0)
        assert torch.equal(y.view(M, N), want.float().to(dt))
        assert bool((buffer[:128] == 77).all()) and bool((buffer[-128:] == 77).all())


@pytest.mark.parametrize("M", [2, 40, 100, 2100])
@pytest.mark.parametrize("out", ["bf16", "fp32"])
def test_nan_and_infinities_stay_in_their_rows(device, M, out):
    N, K = 2200, 272
    x, xs, w, ws = make(device, M, N, K, 3)
    want = wa.linear_fp8(x, xs, w, ws, out_dtype=TYPES[out])
    x.view(torch.uint8)[1, 7] = 0x7f
    w.view(torch.uint8)[5, 270] = 0xff
    xs[0, 1] = float("inf")
    y = wa.linear_fp8(x, xs, w, ws, out_dtype=TYPES[out])
    assert y[1].isnan().all() and y[:, 5].isnan().all() and not y[0].isfinite().any()
    rest = torch.ones_like(y, dtype=torch.bool)
    rest[:2], rest[:, 5] = False, False
    assert torch.equal(y[rest], want[rest])


def test_rows_do_not_depend_on_their_batch(device):
    """A token's result in a call of its own and among others: the same kernel, the same bits."""
    x, xs, w, ws = make(device, 64, 515, 1168, 1)
    for lo, hi in ((0, 16), (16, 32), (32, 64)):
        y = wa.linear_fp8(x[lo:hi], xs[lo:hi], w, ws)
        again = wa.linear_fp8(x[lo:hi].flip(0), xs[lo:hi].flip(0), w, ws)
        assert torch.equal(again.flip(0), y)


@pytest.mark.parametrize("M", [3, 24, 64, 150, 2100])
def test_repeats_streams_and_graphs(device, M):
    x, xs, w, ws = make(device, M, 2200, 1040, 2)
    eager = wa.linear_fp8(x, xs, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [wa.linear_fp8(x, xs, w, ws) for _ in range(3)]
    here = [wa.linear_fp8(x, xs, w, ws) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(y, eager) for y in other + here)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = wa.linear_fp8(x, xs, w, ws)
    for k in range(3):
        xs.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, wa.linear_fp8(x, xs, w, ws)), k


def test_gradient_through_transposed_weights(device):
    """dx = dy W: linear_fp8 of dy in 8 bits with the weights and their blocks transposed, against the formula."""
    M, N, K = 70, 640, 384
    _, _, w, ws = make(device, M, N, K, 8)
    dy = torch.randn(M, N, device=device)
    q, s = wa.quantize_fp8(dy)
    dx = wa.linear_fp8(q, s, w.view(torch.uint8).t().contiguous(), ws.t().contiguous(), out_dtype=torch.float32)
    dyq = q.float().double() * spread(s, N, 1).double()
    full = w.float().double() * spread(spread(ws, K, 1), N, 0).double()
    check(dx, dyq @ full, dyq.abs() @ full.abs(), 5, torch.float32)
    # the formula itself against differences of y = x W^T along dx, linear in x
    x, step = torch.randn(M, K, device=device).double(), torch.randn(M, K, device=device).double()
    difference = ((((x + step) @ full.t()) - (x @ full.t())) * dyq).sum()
    assert abs(float((dyq @ full * step).sum() - difference)) <= 1e-9 * float((dyq.abs() @ full.abs() * step.abs()).sum())


def test_past_32_bits(device):
    """Outputs of more than 2^31 elements, and weights of more than 2^32 bytes."""
    M, N, K = 70000, 32768, 128
    x, xs, w, ws = make(device, 1000, N, K, 4, True)
    x, xs = x.view(torch.uint8).repeat(70, 1), xs.repeat(70, 1)
    y = wa.linear_fp8(x, xs, w, ws)
    last = wa.linear_fp8(x[-1000:], xs[-1000:], w, ws)
    assert torch.equal(y[:1000], last) and torch.equal(y[-1000:], last)
    assert torch.equal(last, exact(x[-1000:].view(torch.float8_e4m3fn), xs[-1000:], w, ws)[0].float().bfloat16())
    del y, x, xs, w, ws, last
    N, K = 600001, 8192
    w = torch.randint(0, 0x70, (N, K), dtype=torch.uint8, device=device)
    ws = torch.full((-(-N // 128), K // 128), 2.0 ** -8, device=device)
    for M in (2, 70):
        x, xs, _, _ = make(device, M, 1, K, 6)
        y = wa.linear_fp8(x, xs, w, ws, out_dtype=torch.float32)
        tail = 128 * 3 + N % 128
        want, S = exact(x, xs, w[-tail:].view(torch.float8_e4m3fn), ws[-4:])
        check(y[:, -tail:], want, S, K // 128, torch.float32)
