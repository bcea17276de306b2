"""The draw of a token at the ends of fp32: temperatures so large that logits whose difference is past fp32 keep their weights, and
so small that the least differences decide.

Bar: as in test_gpu_sample_logits.py, the rules in 64 bits.
"""
import math

import numpy as np
import pytest
import torch

import whallm_amd as wa
from test_gpu_sample_logits import check

pytestmark = pytest.mark.gpu
MAX, LEAST = 3.4028234663852886e38, 2.0 ** -149

RULES = [{}, dict(k=40), dict(k=1500), dict(p=0.9), dict(k=3000, p=0.7), dict(m=0.2), dict(k=200, p=0.95, m=0.01)]


def spread(rng, R, V, size):
    """Rows over [-size, size], both ends among them."""
    l = rng.uniform(-1, 1, (R, V)) * size
    l[:, 3], l[:, V - 5] = size, -size
    return torch.from_numpy(l.astype(np.float32))


def draw(device, logits, rng, temp, rule):
    R = logits.shape[0]
    full = {k: np.full(R, v) for k, v in rule.items()}
    check(device, logits, rng.random(R).astype(np.float32), np.full(R, temp), **full)


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("V", [700, 2049, 9000, 50000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_temperatures(device, V, rule, dtype):
    rng = np.random.default_rng(V)
    for size, temp in ((1e38, 1e38), (3.3e38, 3e38), (3.3e38, 3e37), (3.3e38, MAX), (1e30, 1e30), (3e38, 1e36)):
        draw(device, spread(rng, 6, V, size).to(dtype), rng, temp, rule)


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("V", [700, 2049, 9000, 50000])
def test_small_temperatures(device, V, rule):
    rng = np.random.default_rng(V + 1)
    for size, temp in ((1e-30, 1e-30), (1e-37, 1e-38), (3e-38, 1e-40), (2.0 ** -130, 2.0 ** -140), (1.0, 2.0 ** -61), (1e-15, 2.0 ** -59),
                       (3e38, 1e-40), (2.0 ** 61, 1e-40), (2.0 ** 59, LEAST)):
        draw(device, spread(rng, 6, V, size), rng, temp, rule)


@pytest.mark.parametrize("V", [700, 9000])
def test_two_values_far_apart_share_by_the_temperature(device, V):
    """One logit at fp32's largest value and the others at its lowest, T half their distance: e^-2 for each of the others."""
    temp = torch.full((64,), MAX, device=device)
    logits = torch.full((64, V), -MAX, device=device)
    logits[:, 7] = MAX
    u = (torch.arange(64, device=device) + 0.5) / 64
    for k in (None, 100):
        kept = (k or V) - 1
        ks = None if k is None else torch.full((64,), k, dtype=torch.int32, device=device)
        tokens, logp = wa.sample_logits(logits, u, temp, ks)
        whole = 1 + kept * math.exp(-2.0)
        tail = (tokens != 7).cpu().numpy()
        assert tail.sum() >= 0.8 * 64 * (1 - 1 / whole)
        want = np.where(tail, -2.0, 0.0) - math.log(whole)
        assert np.abs(logp.cpu().numpy() - want).max() <= 2.0 ** -22 * np.abs(want).max()
        assert k is None or int(tokens.max()) < 100
