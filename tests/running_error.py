"""Running error analysis: a value in 64 bits with a bound on how far the same steps in fp32 may be
from it. Every fp32 operation is off by at most U relative to its result and passes its operands'
errors on; a fused multiply-add rounds once less than assumed here. Tolerances come from the
formula and the inputs alone."""
import numpy as np

U = 2.0 ** -24                                        # half a step of fp32
HALF_STEP = {"torch.bfloat16": 2.0 ** -8, "torch.float32": 2.0 ** -24}


class Fp32:
    def __init__(self, v, e=0.0):
        self.v = np.asarray(v, np.float64)
        self.e = np.broadcast_to(np.asarray(e, np.float64), self.v.shape)

    def __add__(self, o):
        o = lift(o)
        v = self.v + o.v
        return Fp32(v, self.e + o.e + U * (np.abs(v) + self.e + o.e))

    def __sub__(self, o):
        return self + lift(o) * -1.0

    def __mul__(self, o):
        o = lift(o)
        v = self.v * o.v
        e = self.e * np.abs(o.v) + o.e * np.abs(self.v) + self.e * o.e
        return Fp32(v, e + U * (np.abs(v) + e))

    __radd__, __rmul__ = __add__, __mul__

    def sum(self, axis, depth, keepdims=False):
        """A sum in which no term passes through more than ``depth`` additions, in any order."""
        big = (np.abs(self.v) + self.e).sum(axis, keepdims=keepdims)
        return Fp32(self.v.sum(axis, keepdims=keepdims), self.e.sum(axis, keepdims=keepdims) + 1.01 * depth * U * big)

    def mean(self, depth):
        """The sum by the length, or times its rounded reciprocal: two roundings."""
        s, n = self.sum(-1, depth, True), self.v.shape[-1]
        return Fp32(s.v / n, s.e / n + 2 * U * (np.abs(s.v) + s.e) / n)

    def rsqrt(self):
        """Good to 2 units of fp32."""
        v = 1.0 / np.sqrt(self.v)
        low = 1.0 / np.sqrt(np.maximum(self.v - self.e, 1e-300))
        return Fp32(v, (low - v) + 4 * U * low)

    def __truediv__(self, o):
        o = lift(o)
        v = self.v / o.v
        e = (self.e + np.abs(v) * o.e) / np.maximum(np.abs(o.v) - o.e, 1e-300)
        return Fp32(v, e + U * (np.abs(v) + e))

    def sigmoid(self):
        """1 / (1 + exp(-v)), the exponential good to 2 units, the quotient to 1."""
        v = 1.0 / (1.0 + np.exp(-self.v))
        return Fp32(v, v * (1 - v) * self.e * 1.01 + 8 * U * v)


def lift(v):
    """A Python number as a call's fp32 argument holds it."""
    return v if isinstance(v, Fp32) else Fp32(np.float32(v))


def check(name, got, want, type_name=None):
    """``got`` (a tensor) within the bound of ``want`` and one rounding to its type."""
    g = got.detach().double().cpu().numpy()
    assert g.shape == want.v.shape, (name, g.shape, want.v.shape)
    bound = want.e + HALF_STEP[type_name or str(got.dtype)] * (np.abs(want.v) + want.e) + 1e-37
    bound = np.where(np.isfinite(want.v), bound, 0.0)      # infinities are equal or wrong
    both_nan = np.isnan(g) & np.isnan(want.v)
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(g - want.v) <= bound) | (g == want.v) | both_nan)
    assert not bad.any(), (name, int(bad.sum()), float(np.abs(g - want.v)[bad].max()), float(bound[bad].max()))
