"""norm_fp8 refuses an eps and a weight offset that fp32 does not hold, without a GPU: an eps rounded to 0 makes rows of zeros NaN, and
one rounded to infinity makes all rows 0."""
import math

import pytest
import torch

from whallm_amd import ops


def call(**kw):
    r = torch.zeros(2, 64)
    return ops.norm_fp8(r, weight=torch.zeros(64, dtype=torch.bfloat16), **kw)


@pytest.mark.parametrize("eps", [1e-50, 5e-324, 2.0 ** -150, 1e39, 1.7e308])
def test_eps_past_fp32(eps):
    with pytest.raises(ValueError, match="eps must be 0 or a number that fp32 holds"):
        call(eps=eps)


@pytest.mark.parametrize("offset", [1e39, -1e300])
def test_offset_past_fp32(offset):
    with pytest.raises(ValueError, match="weight_offset must be a number that fp32 holds"):
        call(weight_offset=offset)


@pytest.mark.parametrize("kw", [dict(eps=0.0), dict(eps=1e-45), dict(eps=1e-40), dict(eps=3e38), dict(eps=math.inf), dict(weight_offset=math.inf),
                                dict(weight_offset=1e-60), dict(weight_offset=-3e38)])
def test_others_pass(kw):
    with pytest.raises(ValueError, match="device"):
        call(**kw)
