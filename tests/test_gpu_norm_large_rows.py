"""Rows of a block norm whose squares fp32 holds and whose sum of squares it does not: the mean is what counts.

Bar: as in test_gpu_block_norm.py, the running error of the same steps in fp32 against the formulas in
64 bits.
"""
import numpy as np
import pytest
import torch

import test_gpu_block_norm as norms
import whallm_amd as wa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [1, 40, 300, 1001, 6000, 16384])
@pytest.mark.parametrize("residual", ["fp32", "bf16"])
def test_norms_of_rows_up_to_1e18(device, H, residual):
    rng = np.random.default_rng(H)
    T = 4
    s = norms.make(rng, T, H, device, residual)
    up = lambda t, *f: (t.double() * torch.tensor(f, dtype=torch.float64, device=device)[:, None]).to(t.dtype)  # noqa: E731
    s["residual"] = up(s["residual"], 1.0, 1e18, 1.0, 1e18)
    s["y"] = up(s["y"], 1.0, 1.0, 4e18, 1.0)
    how = dict(scale=0.75, eps=2.0 ** -20)
    x, out = wa.block_norm(**s, **how)
    norms.check("residual", out, norms.want_forward(s, False, 0.75, 2.0 ** -20, True))
    norms.check("x", x, norms.want_x(out, s, 2.0 ** -20))
    assert x[1].any() and (out[2] != s["residual"][2]).any()


@pytest.mark.parametrize("H", [300, 6000, 16384])
def test_their_gradients_are_not_lost(device, H):
    """The gradients' scale as a row of ordinary size has it: a power of two in the residual comes out again."""
    rng = np.random.default_rng(H)
    s = norms.make(rng, 1, H, device)
    dx = norms.randn(rng, (1, H), torch.bfloat16, device)
    args = {k: v for k, v in s.items() if k not in ("residual", "y")}
    up = 2.0 ** 59                                          # 5.8e17
    d = wa.block_norm_backward(dx, None, s["residual"], s["y"], **args, eps=0.0)
    large = wa.block_norm_backward(dx, None, s["residual"] * up, s["y"], **args, eps=0.0)
    assert torch.equal(large.pre_weight, d.pre_weight) and large.pre_weight.any()
