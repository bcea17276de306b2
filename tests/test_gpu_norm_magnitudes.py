"""The gradients of a block norm for rows of any magnitude whose squares fp32 holds, with eps 0: the projections
on the row are as large as the terms they are taken from.

Bar: as in test_gpu_block_norm.py, the running error of the same steps in fp32 against the formulas in
64 bits.
"""
import numpy as np
import pytest
import torch

import test_gpu_block_norm as norms
import whallm_amd as wa

pytestmark = pytest.mark.gpu

# (residual, y) of each row, as powers of ten
ROWS = [(0, 0), (-17, 0), (17, 0), (0, -17), (0, 17), (-17, 17), (17, -17), (17, 17), (-13, -13), (13, 13), (15, 13), (-15, -4)]


@pytest.mark.parametrize("H", [40, 75, 300, 1000, 5001, 9000])
@pytest.mark.parametrize("residual,gate", [("fp32", None), ("bf16", "token"), ("fp32", "full"), ("bf16", "channel")])
def test_gradients_of_rows_of_any_magnitude(device, H, residual, gate):
    rng = np.random.default_rng(H)
    T = len(ROWS)
    s = norms.make(rng, T, H, device, residual, gate)
    scale = 10.0 ** torch.tensor(ROWS, dtype=torch.float64, device=device)
    s["residual"] = (s["residual"].double() * scale[:, :1]).to(s["residual"].dtype)
    s["y"] = (s["y"].double() * scale[:, 1:]).to(torch.bfloat16)
    dx = norms.randn(rng, (T, H), torch.bfloat16, device)
    args = {k: t for k, t in s.items() if k != "residual"}
    # each row by itself: the sums over tokens of one call would show the loudest row alone
    for t in range(T):
        one = {k: (v[t:t + 1] if torch.is_tensor(v) and v.dim() == 2 else v) for k, v in args.items()}
        r = s["residual"][t:t + 1]
        d = wa.block_norm_backward(dx[t:t + 1], None, r, **one, gate_sigmoid=gate is not None, scale=0.9, eps=0.0)
        want = norms.want_grads(dict(one, residual=r), dx[t:t + 1], None, gate is not None, 0.9, 0.0, True)
        for name in ("residual", "y", "post_weight", "pre_weight", "gate"):
            if want[name] is not None:
                norms.check(f"d{name} of row {ROWS[t]}", getattr(d, name), want[name])
