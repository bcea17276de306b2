"""Rows, widths and k that 32 bits do not hold are refused before they are cut to them (tensors without memory stand for
the large ones; what passes every check stops at the one for device tensors)."""
import pytest
import torch

from whallm_amd import ops


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def permutation(pairs):
    i32 = lambda n: meta(n, dtype=torch.int32)  # noqa: E731
    return ops.Permutation(i32(pairs), i32(pairs), i32(5), i32(8), i32(1))


def calls(T, k, H):
    """The three calls that take rows [T * k, H]."""
    rows, p, w = meta(T * k, H), permutation(T * k), meta(T, k, dtype=torch.float32)
    return (lambda: ops.sort_tokens_backward(rows, p, k), lambda: ops.combine_rows(rows, w, p),
            lambda: ops.combine_rows_backward(meta(T, H), rows, w, p))


@pytest.mark.parametrize("T,k,H,msg", [(2 ** 32, 1, 1, "below 2"), (2 ** 32 + 6, 1, 4, "below 2"), (2 ** 31, 1, 8, "below 2"),
                                       (2 ** 28, 8, 2, "below 2"), (3, 2, 2 ** 32 + 8, "hidden"), (3, 2, 2 ** 20 + 1, "hidden"),
                                       (0, 2, 2 ** 32, "hidden"), (2, 65, 8, "k must"), (0, 2 ** 32 + 1, 8, "k must"),
                                       (1, 2 ** 32 + 2, 8, "k must")])
def test_rows_past_32_bits(T, k, H, msg):
    for call in calls(T, k, H):
        with pytest.raises(ValueError, match=msg):
            call()


@pytest.mark.parametrize("T,k,H", [(2 ** 31 - 1, 1, 1), (2 ** 25, 63, 2), (3, 2, 2 ** 20), (0, 64, 8)])
def test_the_largest_pass(T, k, H):
    for call in calls(T, k, H):
        with pytest.raises(ValueError, match="device"):
            call()


@pytest.mark.parametrize("T,k,H,E", [(2 ** 32, 1, 1, 4), (2 ** 31, 1, 1, 4), (2, 2 ** 32 + 1, 8, 4), (2, 2, 2 ** 32 + 8, 4),
                                     (2, 2, 8, 2 ** 32 + 4)])
def test_sort_past_32_bits(T, k, H, E):
    with pytest.raises(ValueError, match="below 2|at most"):
        ops.sort_tokens(meta(T, H), meta(T, k, dtype=torch.int32), E)


def test_norms_and_logits_past_32_bits():
    with pytest.raises(ValueError, match="below 2"):
        ops.block_norm(meta(2 ** 32 + 1, 2, dtype=torch.float32), meta(2 ** 32 + 1, 2))
    with pytest.raises(ValueError, match="H from 1"):
        ops.block_norm(meta(2, 2 ** 32 + 8, dtype=torch.float32), meta(2, 2 ** 32 + 8))
    with pytest.raises(ValueError, match="at most"):
        ops.process_logits(meta(2, 2 ** 32 + 8))
    with pytest.raises(ValueError, match="rows"):
        ops.process_logits(meta(2 ** 32 + 2, 8))
    with pytest.raises(ValueError, match="history must hold"):
        ops.process_logits(meta(2, 8), history=meta(2, 2 ** 32 + 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="bias_ids must hold"):
        ops.process_logits(meta(2, 8), bias_ids=meta(2, 2 ** 32 + 2, dtype=torch.int32), bias_values=meta(2, 2 ** 32 + 2, dtype=torch.float32))
