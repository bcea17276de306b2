"""Permuted rows of 192 to 256 MB, which the sort and the gradients of back store partly past the cache: moved rows and
w dy are exact whichever way a row went, at both sides of the split and in the rows without a pair.

Bar: moved rows bit for bit; w dy is one product in fp32, rounded once to the rows' type, which torch's own gives bit for
bit.
"""
import pytest
import torch

import whallm_amd as wa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,K,H,dtype", [(5300, 8, 1200, torch.float32),      # 194 MB
                                         (2600, 20, 1001, torch.float32),     # 199 MB, odd rows, more than a batch of pairs
                                         (2100, 6, 9984, torch.bfloat16),     # 240 MB
                                         (17000, 12, 523, torch.bfloat16),    # 203 MB, odd rows
                                         (52000, 8, 250, torch.bfloat16),     # 198 MB of short rows, which all stay
                                         (26300, 8, 160, torch.float32)])     # 128 MB, which all stay
def test_moved_rows_are_exact(device, T, K, H, dtype):
    E = 40
    gen = torch.Generator(device).manual_seed(T)
    idx = torch.randint(0, E + 1, (T, K), generator=gen, device=device, dtype=torch.int32)   # E: no expert
    x = torch.randn(T, H, generator=gen, device=device).to(dtype)
    w = torch.randn(T, K, generator=gen, device=device)
    n = int((idx < E).sum())
    for _ in range(2):                                       # the second call over memory that the first one wrote
        rows, p = wa.sort_tokens(x, idx, E)
        drows, _ = wa.combine_rows_backward(x, rows, w, p)
        assert int(p.offsets[-1]) == n and not rows[n:].any() and not drows[n:].any()
        for a in range(0, n, 8192):
            pair = p.order[a:min(a + 8192, n)].long()
            assert torch.equal(rows[a:a + len(pair)], x[pair // K])
            assert torch.equal(drows[a:a + len(pair)], (x[pair // K].float() * w.view(-1)[pair, None]).to(dtype))
        del rows, drows
