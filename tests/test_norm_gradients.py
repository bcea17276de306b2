"""The gradients of a block norm are the derivatives of its forward pass: the formulas that the GPU tests hold the
kernels against, by automatic differentiation of the forward formula in 64 bits; the kernels' gradients
against the same, and against differences of the kernels' own forward pass."""
import numpy as np
import pytest
import torch

import test_gpu_block_norm as norms
import whallm_amd as wa
from running_error import Fp32

FORMS = [dict(gate=None), dict(gate="token", sigmoid=True), dict(gate="token"), dict(gate="channel", sigmoid=True),
         dict(gate="channel", offset=1.0), dict(gate="full", sigmoid=True, offset=1.0), dict(gate="full"),
         dict(gate="token", sigmoid=True, post_norm=False), dict(gate="channel", post=False), dict(gate="full", pre=False)]
NAMES = ("residual", "y", "post_weight", "pre_weight", "gate")


def make(seed, T, H, device, form, residual="fp32"):
    rng = np.random.default_rng(seed)
    post_norm = form.get("post_norm", True)
    s = norms.make(rng, T, H, device, residual, form["gate"], "fp32", form.get("post", True) and post_norm, form.get("pre", True),
                   form.get("offset", 0.0))
    dx = norms.randn(rng, (T, H), torch.bfloat16, device)
    dres = norms.randn(rng, (T, H), s["residual"].dtype, device)
    return s, dx, dres, post_norm


def by_autograd(s, dx, dres, sigmoid, scale, eps, post_norm):
    """Of <x, dx> + <residual', dres> at s['residual'] = residual', through the forward formula alone."""
    leaf = {k: s[k].detach().double().cpu().requires_grad_() for k in NAMES if s[k] is not None}
    o = s["weight_offset"]
    z = leaf["y"]
    if post_norm:
        z = z / (z * z).mean(-1, keepdim=True).add(eps).sqrt()
    if s["post_weight"] is not None:
        z = z * (leaf["post_weight"] + o)
    g = 1.0 if s["gate"] is None else torch.sigmoid(leaf["gate"]) if sigmoid else leaf["gate"]
    add = scale * g * z
    r = leaf["residual"] - add.detach() + add
    x = r / (r * r).mean(-1, keepdim=True).add(eps).sqrt()
    if s["pre_weight"] is not None:
        x = x * (leaf["pre_weight"] + o)
    ((x * dx.double().cpu()).sum() + (r * dres.double().cpu()).sum()).backward()
    return {k: leaf[k].grad.numpy() if k in leaf else None for k in NAMES}


@pytest.mark.parametrize("form", FORMS)
def test_formulas_are_the_derivatives(form):
    s, dx, dres, post_norm = make(3, 7, 50, "cpu", form)
    args = (s, dx, dres, form.get("sigmoid", False), 0.7, 1e-6, post_norm)
    want, got = by_autograd(*args), norms.want_grads(*args)
    for name in NAMES:
        assert (want[name] is None) == (got[name] is None), name
        if want[name] is not None:
            # the scale and eps of a call are fp32: 2^-24 relative, and 2^-24 of eps, which is 1e-5 of the means
            np.testing.assert_allclose(got[name].v, want[name], rtol=1e-6, atol=1e-6 * np.abs(want[name]).max())


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("T,H,residual", [(9, 72, "fp32"), (300, 500, "bf16"), (5, 6000, "fp32"), (3, 9001, "bf16")])
def test_kernels_give_the_derivatives(device, form, T, H, residual):
    s, dx, dres, post_norm = make(T, T, H, device, form, residual)
    scale, eps = 0.75, 2.0 ** -20                          # exact in fp32
    args = (s, dx, dres, form.get("sigmoid", False), scale, eps, post_norm)
    r = s["residual"]
    d = wa.block_norm_backward(dx, dres, r, **{k: v for k, v in s.items() if k != "residual"},
                               gate_sigmoid=form.get("sigmoid", False), scale=scale, eps=eps, post_norm=post_norm)
    want, bound = by_autograd(*args), norms.want_grads(*args)
    for name in NAMES:
        if want[name] is not None:
            norms.check("d" + name, getattr(d, name), Fp32(want[name], bound[name].e))


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_kernels_against_differences_along_the_gradient(device, form):
    """From an input half a step back along its gradient to half a step ahead, the forward kernel's <residual', u> +
    <x, dx> grows by the gradient's product with the way taken. x is bf16: each of its H T values, of about 1,
    is off by at most 2^-8 of itself in each of two passes, times a dx of about 1; as independent errors
    that is sqrt(2 H T) 2^-8, held to six of these. The steps' third order is a hundredth or less. The way is along the
    gradient so that what is expected is far above both."""
    T, H = 600, 512
    s, dx, u, post_norm = make(21, T, H, device, form)
    how = dict(gate_sigmoid=form.get("sigmoid", False), scale=0.9, eps=1e-6, post_norm=post_norm)
    x, out = wa.block_norm(**s, **how)
    d = wa.block_norm_backward(dx, u, out, **{k: v for k, v in s.items() if k != "residual"}, **how)

    def value(name, t):
        x, out = wa.block_norm(**dict(s, **{name: t}), **how)
        return float((x.double() * dx.double()).sum() + (out.double() * u.double()).sum())

    noise = 6 * (2 * H * T) ** 0.5 * 2.0 ** -8
    for name in NAMES:
        if s[name] is None:
            continue
        grad = getattr(d, name).double()
        step = 0.05 * float(s[name].double().square().mean().sqrt()) if name in ("residual", "y") else 0.1
        half = grad * (step / grad.square().mean().sqrt())
        ahead, back = (s[name].double() + half).to(s[name].dtype), (s[name].double() - half).to(s[name].dtype)
        want = float((grad * (ahead.double() - back.double())).sum())
        got = value(name, ahead) - value(name, back)
        assert abs(want) > 10 * noise, (name, want, noise)
        assert abs(got - want) <= noise + 0.02 * abs(want), (name, got, want)
