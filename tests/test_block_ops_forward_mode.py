"""Inputs with a forward-mode tangent are refused like those that require gradients: no call gives a tangent back.
torch.no_grad() does not switch forward mode off, torch.inference_mode() does."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from whallm_amd import ops

T, K, H, V = 6, 2, 8, 40


def inputs():
    bf16 = torch.bfloat16
    r, y, w = torch.ones(T, H), torch.ones(T, H, dtype=bf16), torch.ones(H, dtype=bf16)
    rows, weights = torch.ones(T * K, H), torch.ones(T, K)
    p = ops.Permutation(*(torch.zeros(n, dtype=torch.int32) for n in (T * K, T * K, 5, 8, 1)))
    idx, value = torch.zeros(T, K, dtype=torch.int32), torch.ones(T)
    history, ids = torch.zeros(T, 3, dtype=torch.int32), torch.zeros(T, 3, dtype=torch.int32)
    return [(ops.sort_tokens, dict(x=r, indices=idx, experts=4), ["x"]),
            (ops.sort_tokens_backward, dict(drows=rows, permutation=p, k=K), ["drows"]),
            (ops.combine_rows, dict(rows=rows, weights=weights, permutation=p, add=r), ["rows", "weights", "add"]),
            (ops.combine_rows_backward, dict(dy=r, rows=rows, weights=weights, permutation=p), ["dy", "rows", "weights"]),
            (ops.block_norm, dict(residual=r, y=y, post_weight=w, pre_weight=w, gate=r.clone(), residual_out=r.clone()),
             ["residual", "y", "post_weight", "pre_weight", "gate", "residual_out"]),
            (ops.block_norm_backward, dict(dx=y, dresidual=r, residual_out=r, y=y, post_weight=w, pre_weight=w, gate=r),
             ["dx", "dresidual", "residual_out", "y", "post_weight", "pre_weight", "gate"]),
            (ops.process_logits, dict(logits=torch.ones(T, V), history=history, repetition=value, frequency=value, presence=value,
                                      bias_ids=ids, bias_values=torch.ones(T, 3), temperature=value, out=torch.ones(T, V)),
             ["logits", "repetition", "frequency", "presence", "bias_values", "temperature", "out"])]


CASES = [(i, name) for i, (_, _, names) in enumerate(inputs()) for name in names]


@pytest.mark.parametrize("i,name", CASES)
@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_are_refused(i, name, grad_mode):
    call, kw, _ = inputs()[i]
    with fwad.dual_level(), torch.set_grad_enabled(grad_mode):
        kw[name] = fwad.make_dual(kw[name], torch.ones_like(kw[name]))
        with pytest.raises(ValueError, match="forward-mode"):
            call(**kw)
        with fwad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="device"):
            call(**kw)
        kw[name] = fwad.unpack_dual(kw[name]).primal
        with pytest.raises(ValueError, match="device"):
            call(**kw)


@pytest.mark.parametrize("i", range(7))
def test_inference_mode_passes(i):
    with torch.inference_mode():
        call, kw, _ = inputs()[i]
        with pytest.raises(ValueError, match="device"):
            call(**kw)
