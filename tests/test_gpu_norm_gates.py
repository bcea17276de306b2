"""Gates of a block norm over the whole range of their type: through the sigmoid an infinite gate is 0 or 1, as is
any that is far enough out, in the forward pass and in the gradients.

Bar: as in test_gpu_block_norm.py, the running error of the same steps in fp32 against the formulas in
64 bits. What a sigmoid below 2^-126 adds is under the bar's absolute 1e-37.
"""
import numpy as np
import pytest
import torch

import test_gpu_block_norm as norms
import whallm_amd as wa

pytestmark = pytest.mark.gpu

ENDS = [float("-inf"), float("inf"), None, None, -1e8, -48496640.0, -1000.0, -100.0, -80.0, -20.0, 20.0, 80.0, 100.0, 1000.0, 1e8, 0.0]


def ends(dtype):
    """The lowest and the highest value of the type among them."""
    f = torch.finfo(dtype)
    v = list(ENDS)
    v[2], v[3] = f.min, f.max
    return torch.tensor(v, dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("gate", ["token", "channel", "full"])
@pytest.mark.parametrize("gate_type", ["fp32", "bf16"])
@pytest.mark.parametrize("T,H,residual,post_norm", [(35, 75, "fp32", True), (20, 264, "bf16", False), (33, 1000, "fp32", False),
                                                    (5, 5128, "bf16", True), (3, 9000, "fp32", True)])
def test_sigmoid_gates_over_their_range(device, gate, gate_type, T, H, residual, post_norm):
    rng = np.random.default_rng(T)
    s = norms.make(rng, T, H, device, residual, gate, gate_type, post_norm)
    v = ends(norms.TYPES[gate_type]).to(device)
    g = s["gate"]
    n = g.numel()
    s["gate"] = v[torch.from_numpy(rng.permutation(n) % len(v)).to(device)].view_as(g)
    how = dict(gate_sigmoid=True, scale=0.7, eps=1e-6, post_norm=post_norm)
    with np.errstate(over="ignore"):
        x, out = wa.block_norm(**s, **how)
        norms.check("residual", out, norms.want_forward(s, True, 0.7, 1e-6, post_norm))
        norms.check("x", x, norms.want_x(out, s, 1e-6))
        dx, dres = (norms.randn(rng, (T, H), t, device) for t in (torch.bfloat16, out.dtype))
        s["residual"] = out
        d = wa.block_norm_backward(dx, dres, out, **{k: t for k, t in s.items() if k != "residual"}, **how)
        want = norms.want_grads(s, dx, dres, True, 0.7, 1e-6, post_norm)
    for name in ("residual", "y", "post_weight", "pre_weight", "gate"):
        if want[name] is not None:
            norms.check("d" + name, getattr(d, name), want[name])


@pytest.mark.parametrize("H", [96, 512, 6000, 16384])
def test_a_closed_gate_adds_nothing(device, H):
    """A gate of -inf leaves the residual's bits, zeros among them; one of +inf is no gate."""
    rng = np.random.default_rng(H)
    s = norms.make(rng, 4, H, device)
    s["residual"][1] = 0.0
    closed, opened = (torch.full((4, 1), v, device=device) for v in (float("-inf"), float("inf")))
    _, out = wa.block_norm(**dict(s, gate=closed), gate_sigmoid=True)
    assert torch.equal(out, s["residual"])
    x, out = wa.block_norm(**dict(s, gate=opened), gate_sigmoid=True)
    x1, out1 = wa.block_norm(**s)
    assert torch.equal(out, out1) and torch.equal(x, x1)


def test_a_nan_gate_stays_in_its_row(device):
    rng = np.random.default_rng(1)
    s = norms.make(rng, 5, 300, device, gate="token")
    s["gate"][2] = float("nan")
    x, out = wa.block_norm(**s, gate_sigmoid=True)
    bad = torch.isnan(out).any(1)
    assert bad.tolist() == [False, False, True, False, False] and torch.isnan(out[2]).all() and torch.isnan(x[2].float()).all()
