"""The sort of token rows for millions of pairs: what a workgroup counts does not grow with them, and the lists and
rows are exact."""
import numpy as np
import pytest
import torch

import whallm_amd as wa
from whallm_amd import _lib


@pytest.mark.parametrize("k", [1, 3, 8, 10, 64])
@pytest.mark.parametrize("pairs", [2 ** 15, 2 ** 19, 2 ** 20, 2 ** 25, 2 ** 31 - 64])
def test_spans_stay_small(k, pairs):
    """The workspace has a count for each expert and span: a workgroup counts the pairs of its own span again, so a span
    has at most 8192 pairs and a chunk (256), whatever the call's size."""
    tokens, experts = pairs // k, 100
    need = _lib.load().wm_sort_tokens_workspace_size(tokens, k, experts)
    spans = need // (4 * experts)
    assert need == spans * 4 * experts and tokens * k <= spans * (8192 + 256)


def torch_lists(idx, E, tile_rows):
    """The lists on the GPU, by a stable sort."""
    flat = idx.reshape(-1).long()
    P = flat.numel()
    key, pair = torch.sort(torch.where((flat >= 0) & (flat < E), flat, E), stable=True)
    offsets = torch.searchsorted(key, torch.arange(E + 1, device=key.device))
    at = torch.arange(P, device=key.device)
    n = int(offsets[-1])
    inverse = torch.empty_like(pair)
    inverse[pair] = torch.where(at < n, at, -1)
    lists = {"order": torch.where(at < n, pair, -1), "inverse": inverse, "offsets": offsets}
    tiles = [(e, r) for e, (a, b) in enumerate(zip(offsets[:-1].tolist(), offsets[1:].tolist())) for r in range(a, b, tile_rows)]
    return {k: v.to(torch.int32) for k, v in lists.items()}, torch.tensor(tiles, dtype=torch.int32, device=idx.device).view(-1, 2), n


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,H,dtype,form", [
    (52428, 10, 512, 3, "bf16", "some"),        # the last size whose spans every workgroup adds up (524280 pairs)
    (52430, 10, 512, 3, "bf16", "some"),        # the next one
    (700000, 3, 1, 2, "fp32", "all"),           # one expert
    (524289, 1, 1024, 5, "bf16", "some"),
    (20000, 64, 65, 8, "bf16", "one"),          # a chunk of 4 tokens, every pair the last expert's
    (600000, 8, 130, 2, "bf16", "half"),        # 4.8 million pairs, the busiest first
    (4194301, 8, 33, 1, "bf16", "some"),        # 33.5 million
])
def test_lists_and_rows_of_many_pairs(device, T, k, E, H, dtype, form):
    gen = torch.Generator(device).manual_seed(T)
    idx = torch.randint(-1 if form == "some" else 0, E + (form == "some"), (T, k), generator=gen, device=device, dtype=torch.int32)
    if form == "one":
        idx.fill_(E - 1)
    if form == "half":
        idx[: T // 2] = 0
    x = torch.randn(T, H, generator=gen, device=device).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    rows, p = wa.sort_tokens(x, idx, E, 4096)
    want, tiles, n = torch_lists(idx, E, 4096)
    for name, w in want.items():
        assert torch.equal(getattr(p, name), w), name
    assert p.tile_count.item() == len(tiles) and torch.equal(p.tiles[: len(tiles)], tiles) and (p.tiles[len(tiles):] == -1).all()
    assert torch.equal(rows[:n], x[want["order"][:n].long() // k]) and not rows[n:].any()


@pytest.mark.gpu
def test_replayed_graphs_of_many_pairs(device):
    """Three launches and a workspace: every replay as the eager call."""
    T, k, E, H = 70001, 9, 300, 8
    gen = torch.Generator(device).manual_seed(1)
    draw = lambda: torch.randint(-1, E, (T, k), generator=gen, device=device, dtype=torch.int32)  # noqa: E731
    idx, x = draw(), torch.randn(T, H, generator=gen, device=device).bfloat16()
    wa.sort_tokens(x, idx, E)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, p = wa.sort_tokens(x, idx, E)
    for _ in range(3):
        idx.copy_(draw())
        graph.replay()
        want, q = wa.sort_tokens(x, idx, E)
        torch.cuda.synchronize()
        assert torch.equal(rows, want)
        for name in ("order", "inverse", "offsets", "tiles", "tile_count"):
            assert torch.equal(getattr(p, name), getattr(q, name)), name
    lists, _, n = torch_lists(idx, E, 128)
    assert torch.equal(p.order, lists["order"]) and np.array_equal(p.offsets.cpu().numpy(), lists["offsets"].cpu().numpy())
