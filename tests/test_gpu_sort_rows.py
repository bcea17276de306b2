"""GPU parity of the sort of token rows by expert and the way back, with both gradients
(wm_sort_tokens, wm_sort_tokens_backward, wm_combine_rows, wm_combine_rows_backward) against a
plain restatement in 64 bits.

Bar: lists and moved rows exact. A sum of n products or terms in fp32 is off by at most
(n + 1) * 2^-24 of the sum of their magnitudes in any order; a result is then rounded once, by at
most half a step of its type (2^-8 bf16, 2^-24 fp32, relative).
"""
import numpy as np
import pytest
import torch

import whallm_amd as wa

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def make_indices(rng, T, K, E, absent):
    idx = np.stack([rng.choice(max(E, K), K, replace=False) for _ in range(T)]).astype(np.int64) if T else np.zeros((0, K), np.int64)
    if E < K:
        idx = rng.integers(0, E, size=(T, K))
    if absent == "some":
        bad = np.array([-1, E, E + 5, -2 ** 31, 2 ** 31 - 1])
        idx = np.where(rng.random((T, K)) < 0.3, bad[rng.integers(0, len(bad), size=(T, K))], idx)
    elif absent == "all":
        idx[:] = -1
    elif absent == "one expert":
        idx[:] = E - 1
    return idx.astype(np.int32)


def want_lists(idx, E, tile_rows):
    flat = idx.reshape(-1).astype(np.int64)
    present = np.nonzero((flat >= 0) & (flat < E))[0]
    pairs = present[np.argsort(flat[present], kind="stable")]
    P, n = flat.size, pairs.size
    order, inverse = np.full(P, -1), np.full(P, -1)
    order[:n], inverse[pairs] = pairs, np.arange(n)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[present], minlength=E))])
    tiles = [(e, r) for e in range(E) for r in range(offsets[e], offsets[e + 1], tile_rows)]
    whole = np.full((-(-P // tile_rows) + E, 2), -1)
    if tiles:
        whole[:len(tiles)] = tiles
    return order, inverse, offsets, whole, len(tiles)


def rows_tensor(rng, shape, dtype, device, std=1.0):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * std).to(dtype).to(device)


def f64(t):
    return t.detach().double().cpu().numpy()


def check(got, want, terms, magnitude, dtype=None):
    """got within the fp32 sum's error of want plus one rounding to its type."""
    err = (terms + 1) * 2.0 ** -24 * magnitude
    bound = err + STEP[dtype or got.dtype] * (np.abs(want) + err) + 1e-40
    g = f64(got)
    assert g.shape == want.shape
    bad = ~(np.abs(g - want) <= bound)
    assert not bad.any(), (int(bad.sum()), float(np.abs(g - want).max()))


CASES = [
    # T, K, E, H, tile_rows, absent
    (1, 10, 512, 2048, 128, None),       # one decode token
    (1, 1, 1, 1, 1, None),
    (8, 10, 512, 2560, 16, None),
    (3, 3, 5, 7, 2, "some"),
    (65, 8, 64, 200, 32, "some"),
    (300, 6, 1024, 96, 128, "some"),
    (40, 2, 8, 2049, 64, "all"),
    (517, 4, 3, 130, 128, None),         # fewer experts than k: a token's pairs share experts
    (1000, 10, 512, 264, 128, "some"),
    (2300, 8, 128, 136, 128, "one expert"),
    (700, 64, 256, 33, 100, "some"),
    (250, 9, 100, 4104, 128, "some"),    # a workgroup of 1024 a token
    (6, 4, 5, 16, 2 ** 31 - 1, None),    # one tile an expert, whose rows' sum passes 31 bits
    (5000, 4, 5, 16, 2 ** 31 - 1, "some"),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,K,E,H,tile_rows,absent", CASES)
def test_rows_and_gradients_match_the_formulas(device, T, K, E, H, tile_rows, absent, dtype):
    rng = np.random.default_rng(T * 31 + K + E + H)
    dt = DTYPES[dtype]
    idx = make_indices(rng, T, K, E, absent)
    order, inverse, offsets, tiles, count = want_lists(idx, E, tile_rows)
    n = offsets[-1]
    x = rows_tensor(rng, (T, H), dt, device)
    rows, p = wa.sort_tokens(x, torch.from_numpy(idx).to(device), E, tile_rows)
    assert rows.shape == (T * K, H) and rows.dtype == dt
    for got, want in ((p.order, order), (p.inverse, inverse), (p.offsets, offsets), (p.tiles, tiles), (p.tile_count, [count])):
        np.testing.assert_array_equal(got.cpu().numpy(), want)
    want = np.zeros((T * K, H))
    want[:n] = f64(x)[order[:n] // K]
    np.testing.assert_array_equal(f64(rows), want)

    # rows without a pair hold NaN: nothing may read them
    r = rows_tensor(rng, (T * K, H), dt, device)
    r[n:] = float("nan")
    w = torch.from_numpy(rng.standard_normal((T, K)).astype(np.float32)).to(device)
    w[torch.from_numpy(inverse.reshape(T, K) < 0)] = float("nan")
    add = rows_tensor(rng, (T, H), dt, device)
    live = inverse.reshape(T, K) >= 0
    safe = np.where(live[..., None], f64(r)[np.maximum(inverse, 0)].reshape(T, K, H), 0.0)
    sw = np.where(live, f64(w), 0.0)
    check(wa.sort_tokens_backward(r, p, K), safe.sum(1), K, np.abs(safe).sum(1))
    terms = safe * sw[..., None]
    check(wa.combine_rows(r, w, p), terms.sum(1), K, np.abs(terms).sum(1))
    check(wa.combine_rows(r, w, p, add), terms.sum(1) + f64(add), K + 1, np.abs(terms).sum(1) + np.abs(f64(add)))
    dy = rows_tensor(rng, (T, H), dt, device)
    drows, dw = wa.combine_rows_backward(dy, r, w, p)
    want = np.zeros((T * K, H))
    want[:n] = (sw[..., None] * f64(dy)[:, None]).reshape(T * K, H)[order[:n]]
    check(drows, want, 0, np.abs(want))
    dots = safe * f64(dy)[:, None]
    # at least 64 lanes share a dot product's H terms, then at most 64 partial sums are added
    check(dw, dots.sum(-1), -(-H // 64) + 64, np.abs(dots).sum(-1), torch.float32)


def test_lists_equal_permute_and_no_tokens(device):
    rng = np.random.default_rng(5)
    idx = torch.from_numpy(make_indices(rng, 400, 8, 60, "some")).to(device)
    rows, p = wa.sort_tokens(torch.zeros(400, 8, dtype=torch.bfloat16, device=device), idx, 60)
    q = wa.permute(idx, 60)
    n, tiles = int(q.offsets[-1]), int(q.tile_count)
    assert torch.equal(p.order[:n], q.order[:n]) and torch.equal(p.inverse, q.inverse) and torch.equal(p.offsets, q.offsets)
    assert torch.equal(p.tiles[:tiles], q.tiles[:tiles]) and torch.equal(p.tile_count, q.tile_count)
    # permute's own lists serve the way back as well
    r = rows_tensor(rng, (3200, 24), torch.float32, device)
    w = torch.rand(400, 8, device=device)
    assert torch.equal(wa.combine_rows(r, w, q), wa.combine_rows(r, w, p))

    rows, p = wa.sort_tokens(torch.zeros(0, 64, device=device), torch.zeros(0, 4, dtype=torch.int32, device=device), 6)
    assert rows.shape == (0, 64) and p.offsets.tolist() == [0] * 7 and p.tile_count.tolist() == [0]
    assert p.tiles.tolist() == [[-1, -1]] * 6
    w = torch.zeros(0, 4, device=device)
    assert wa.combine_rows(rows, w, p).shape == (0, 64) and wa.sort_tokens_backward(rows, p, 4).shape == (0, 64)
    drows, dw = wa.combine_rows_backward(torch.zeros(0, 64, device=device), rows, w, p)
    assert drows.shape == (0, 64) and dw.shape == (0, 4)


def test_strided_batched_and_unaligned_inputs(device):
    """Leading axes, transposed and sliced inputs, rows that start off a 16-byte boundary."""
    rng = np.random.default_rng(9)
    B, L, K, E, H = 3, 17, 4, 20, 72
    wide = rows_tensor(rng, (B, L, 2 * H), torch.bfloat16, device)
    x = wide[..., 1:2 * H:2]
    idx = torch.from_numpy(make_indices(rng, B * L, K, E, "some").reshape(B, L, K)).to(device)
    rows, p = wa.sort_tokens(x, idx.transpose(0, 1).contiguous().transpose(0, 1), E)
    want, q = wa.sort_tokens(x.reshape(-1, H).clone(), idx.reshape(-1, K), E)
    assert torch.equal(rows, want) and torch.equal(p.inverse, q.inverse)
    w = torch.rand(K, B, L, device=device).permute(1, 2, 0)
    y = wa.combine_rows(rows, w, p, add=x)
    assert y.shape == (B, L, H)
    off = torch.empty(rows.numel() + 1, dtype=rows.dtype, device=device)[1:].view_as(rows).copy_(rows)
    assert off.data_ptr() % 16
    assert torch.equal(wa.combine_rows(off, w, p, add=x), y)
    assert torch.equal(wa.sort_tokens_backward(off, p, K), wa.sort_tokens_backward(rows, p, K))
    for a, b in zip(wa.combine_rows_backward(y, off, w, p), wa.combine_rows_backward(y, rows, w, p)):
        assert torch.allclose(a.float(), b.float(), rtol=1e-5, atol=1e-5)   # the dot's order may differ
    got, _ = wa.sort_tokens(off[:30], idx.reshape(-1, K)[:30].contiguous(), E)
    want, _ = wa.sort_tokens(rows[:30].clone(), idx.reshape(-1, K)[:30].contiguous(), E)
    assert torch.equal(got, want)


def test_gradients_against_differences(device):
    """The passes are linear in x, rows and weights, so a difference quotient along a direction is
    the gradient's product with it up to rounding."""
    rng = np.random.default_rng(11)
    T, K, E, H = 21, 5, 9, 48
    idx = torch.from_numpy(make_indices(rng, T, K, E, "some")).to(device)
    x, vx, dy = (rows_tensor(rng, (T, H), torch.float32, device) for _ in range(3))
    rows, p = wa.sort_tokens(x, idx, E)
    d = rows_tensor(rng, tuple(rows.shape), torch.float32, device)
    moved = wa.sort_tokens(x + vx, idx, E)[0].double() - wa.sort_tokens(x - vx, idx, E)[0].double()
    a, b = float((moved * d.double()).sum() / 2), float((wa.sort_tokens_backward(d, p, K).double() * vx.double()).sum())
    assert abs(a - b) <= 1e-4 * abs(b) + 1e-3
    w, vw = torch.rand(T, K, device=device), torch.randn(T, K, device=device)
    drows, dw = wa.combine_rows_backward(dy, rows, w, p)
    a = float(((wa.combine_rows(rows, w + vw, p).double() - wa.combine_rows(rows, w - vw, p).double()) * dy.double()).sum() / 2)
    b = float((dw.double() * vw.double()).sum())
    assert abs(a - b) <= 1e-4 * abs(b) + 1e-2
    a = float(((wa.combine_rows(rows + d, w, p).double() - wa.combine_rows(rows - d, w, p).double()) * dy.double()).sum() / 2)
    b = float((drows.double() * d.double()).sum())
    assert abs(a - b) <= 1e-4 * abs(b) + 1e-2


def test_other_stream_and_graph_replays(device):
    """A captured round trip is replayed with new inputs; every replay equals the eager calls."""
    rng = np.random.default_rng(13)
    for T, K, E, H in ((4, 8, 64, 256), (900, 8, 64, 256)):
        x = rows_tensor(rng, (T, H), torch.bfloat16, device)
        idx = torch.from_numpy(make_indices(rng, T, K, E, None)).to(device)
        w = torch.rand(T, K, device=device)

        def step():
            rows, p = wa.sort_tokens(x, idx, E)
            y = wa.combine_rows(rows, w, p, add=x)
            return (rows, p.inverse, p.order, p.tiles, y, *wa.combine_rows_backward(y, rows, w, p), wa.sort_tokens_backward(rows, p, K))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for seed in range(3):
            r2 = np.random.default_rng(seed)
            x.copy_(rows_tensor(r2, (T, H), torch.bfloat16, device))
            idx.copy_(torch.from_numpy(make_indices(r2, T, K, E, "some")).to(device))
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
        del eager


@pytest.mark.parametrize("T,K,H,dtype", [(9001, 4, 3001, "bf16"),     # rows past 192 MiB, odd rows
                                         (9000, 4, 3008, "fp32"),     # gradients past 384 MiB, whole lines
                                         (16400, 8, 16384, "bf16")])  # offsets past 2^31 elements
def test_large_tensors(device, T, K, H, dtype):
    """Moved rows exact; the sums of the first and last tokens and of some between against 64 bits."""
    E, dt = 64, DTYPES[dtype]
    gen = torch.Generator(device).manual_seed(T)
    x = torch.randn(T, H, generator=gen, device=device, dtype=torch.float32).to(dt)
    idx = torch.randint(0, E + 1, (T, K), generator=gen, device=device).to(torch.int32)  # E: no expert
    rows, p = wa.sort_tokens(x, idx, E)
    order, inverse, offsets, _, _ = want_lists(idx.cpu().numpy(), E, 128)
    np.testing.assert_array_equal(p.order.cpu().numpy(), order)
    np.testing.assert_array_equal(p.inverse.cpu().numpy(), inverse)
    n = int(offsets[-1])
    for a in range(0, n, 8192):
        b = min(a + 8192, n)
        assert torch.equal(rows[a:b], x[p.order[a:b].long() // K])
    assert not rows[n:].any()
    some = [0, 1, T // 3, T // 2, T - 2, T - 1]
    live = inverse.reshape(T, K)[some] >= 0
    at = torch.from_numpy(np.maximum(inverse.reshape(T, K)[some], 0)).to(device)
    w = torch.randn(T, K, generator=gen, device=device)
    own = f64(rows[at]) * live[..., None]
    check(wa.sort_tokens_backward(rows, p, K)[some], own.sum(1), K, np.abs(own).sum(1))
    terms = own * f64(w[some])[..., None]
    check(wa.combine_rows(rows, w, p)[some], terms.sum(1), K, np.abs(terms).sum(1))
    drows, dw = wa.combine_rows_backward(x, rows, w, p)
    assert not drows[n:].any()
    want = f64(w[some])[..., None] * f64(x[some])[:, None]
    for t, k in np.ndindex(len(some), K):
        if live[t, k]:
            check(drows[at[t, k]], want[t, k], 0, np.abs(want[t, k]))
    dots = own * f64(x[some])[:, None]
    check(dw[some], dots.sum(-1), -(-H // 64) + 64, np.abs(dots).sum(-1), torch.float32)


@pytest.mark.parametrize("H,dtype", [(24, "bf16"), (257, "fp32"), (4099, "bf16")])
def test_back_over_what_it_adds_to(device, H, dtype):
    """The C call's y may be add."""
    from whallm_amd import _lib
    rng = np.random.default_rng(H)
    T, K, E = 70, 5, 9
    idx = torch.from_numpy(make_indices(rng, T, K, E, "some")).to(device)
    rows, p = wa.sort_tokens(rows_tensor(rng, (T, H), DTYPES[dtype], device), idx, E)
    w, add = torch.rand(T, K, device=device), rows_tensor(rng, (T, H), DTYPES[dtype], device)
    want = wa.combine_rows(rows, w, p, add)
    _lib.call("wm_combine_rows", rows.data_ptr(), int(dtype == "fp32"), w.data_ptr(), p.inverse.data_ptr(), T, K, H, add.data_ptr(),
              add.data_ptr(), torch.cuda.current_stream(device).cuda_stream)
    assert torch.equal(add, want)
