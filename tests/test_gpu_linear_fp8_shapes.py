"""Every kernel of the FP8 product (wm_linear_fp8) with more steps along K than it holds stages or slots, so that its pipeline
turns over: against the formula in 64 bits.

The choice is restated here from the table in gemm_fp8.hip, so that a case says which kernel it runs; a test without a GPU holds that
the cases reach all of them. Bar: test_gpu_linear_fp8.py's.
"""
import re
from pathlib import Path

import pytest
import torch

import whallm_amd as wa
from test_gpu_linear_fp8 import TYPES, check, exact

SOURCE = (Path(__file__).resolve().parents[1] / "whallm_amd" / "csrc" / "gemm_fp8.hip").read_text()
SHAPES = [tuple(int(v) for v in s.split(",")) for s in
          re.findall(r"\{(\d+, \d+, \d+)\}", re.search(r"shape\[8\] = \{(.*?)\};", SOURCE, re.S).group(1))]
ONCE_BYTES = int(re.search(r"ONCE_BYTES = (\d+);", SOURCE).group(1))


def picked(M, N, K, out):
    """(kernel, blocks of K that it must pass for its loads to go into a slot for the second time)."""
    if M <= 16:
        few, X = N <= 8192, 8 if M <= 8 else 16
        return f"stream {16 if few else 32}x{X}", 8 * 4 if few else 4 * 3
    blocks = lambda n, t: -(-N // n) * -(-M // t)   # noqa: E731
    costs = [-(-blocks(n, t) // 256) * cost for n, t, cost in SHAPES[:7 if out == "fp32" else 8]]
    n, t, _ = SHAPES[costs.index(min(costs))]
    if (n, t) in ((16, 32), (32, 32), (64, 32)):
        return f"stream {n}x{t}", 4 * (3 if n == 16 else 2)
    once = M <= t and N * K >= ONCE_BYTES and (n, t) in ((64, 64), (128, 128))
    steps = {(64, 64): 2 * 4, (64, 128): 2 * 3, (128, 128): 4, (128, 256): 3, (256, 256): 2}[n, t]
    return f"tiled {n}x{t}{' once' if once else ''}", {(64, 64): 4 * 2, (128, 128): 2 * 2}[n, t] if once else steps


# the last ones of a stream's sizes have more than eight blocks of K a wave: its second set of scales
CASES = [
    (1, 300, 8336), (12, 300, 8336), (2, 4096, 7168), (6, 9000, 4240), (12, 9000, 4240), (8, 8200, 8192),
    (20, 500, 4240), (31, 515, 8208), (32, 8000, 4240), (24, 6000, 8192), (96, 4608, 5120), (128, 4096, 7168), (70, 4700, 4240),
    (256, 4096, 7168), (256, 4100, 1168), (300, 3333, 2064),
    (512, 4096, 1168), (512, 4100, 2064), (900, 2051, 4112),
    (1024, 4096, 2064), (1000, 4001, 1296),
    (2048, 4096, 7168), (2048, 4100, 1168), (2000, 4000, 2064),
    (4096, 4096, 2064), (4100, 4111, 1168),
    # weights of 100 MB and more under one token tile, and under the kernels that take them with ordinary loads
    (64, 24576, 4112), (100, 25001, 4112), (17, 24576, 7168), (24, 16384, 6160), (32, 24576, 7168), (32, 32773, 4112), (65, 16384, 7168),
    (96, 16384, 7168), (128, 16384, 7168)]


@pytest.mark.parametrize("out", ["bf16", "fp32"])
def test_cases_reach_every_kernel_past_its_stages(out):
    assert len(SHAPES) == 8 and ONCE_BYTES > 0
    want = {f"stream {n}x{x}" for n in (16, 32) for x in (8, 16)} | {"stream 16x32", "stream 32x32", "stream 64x32"}
    want |= {"tiled 64x64", "tiled 64x64 once", "tiled 64x128", "tiled 128x128", "tiled 128x128 once", "tiled 128x256"}
    want |= {"tiled 256x256"} if out == "bf16" else set()
    got, scales = set(), set()
    for M, N, K in CASES:
        name, most = picked(M, N, K, out)
        if -(-K // 128) > most:
            got.add(name)
        if name.startswith("stream") and K > 1024 * (8 if name in ("stream 16x8", "stream 16x16") else 4):
            scales.add(name)
    assert got == want, (want - got, got - want)
    assert scales == {name for name in want if name.startswith("stream")}


def make(device, M, N, K, whole):
    g = torch.Generator(device).manual_seed(M * 31 + N * 7 + K)
    nb, kb = -(-N // 128), -(-K // 128)
    rand = lambda *s: torch.rand(*s, device=device, generator=g)   # noqa: E731
    if whole:
        ints = lambda lo, hi, *s: torch.randint(lo, hi, s, device=device, generator=g).float()   # noqa: E731
        return (ints(-2, 3, M, K).to(torch.float8_e4m3fn), 2.0 ** ints(-3, 4, M, kb), ints(-2, 3, N, K).to(torch.float8_e4m3fn),
                2.0 ** ints(-3, 4, nb, kb))
    f8 = lambda *s: (torch.randn(*s, device=device, generator=g) * 60).to(torch.float8_e4m3fn)   # noqa: E731
    return f8(M, K), rand(M, kb) * 0.02 + 1e-3, f8(N, K), rand(nb, kb) * 1e-3 + 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["bf16", "fp32"])
@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("M,N,K", CASES)
def test_pipelines_turn_over(device, M, N, K, whole, out):
    """Whole numbers: every partial sum is a multiple of 2^-6, the least product of two scales, and fp32 holds those below
    2^24 units, so that the result is exact in any order."""
    x, xs, w, ws = make(device, M, N, K, whole)
    dt = TYPES[out]
    add = (torch.randint(-8, 9, (M, N), device=device).to(dt) if whole else torch.randn(M, N, device=device).to(dt)) if (M + N) % 3 == 0 else None
    y = wa.linear_fp8(x, xs, w, ws, out_dtype=dt, add=add)
    want, S = exact(x, xs, w, ws, add)
    if whole:
        assert float(S.max()) * 2.0 ** 6 < 2.0 ** 24
        assert torch.equal(y, want.to(torch.float32).to(dt)), int((y != want.to(torch.float32).to(dt)).sum())
    else:
        check(y, want, S, xs.shape[1], dt)
    again = wa.linear_fp8(x, xs, w, ws, out_dtype=dt, add=add)
    assert torch.equal(again, y)
