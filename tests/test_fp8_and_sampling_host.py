"""Refusals of the calls between the residual and the next token, without a GPU: the C entry points' argument checks and
the compiled host side's, which come before the one for device tensors."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from whallm_amd import _lib, ops

A = 0x10000   # an aligned address that is never read
BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def refused(entry, base, cases):
    for kw, msg in cases:
        with pytest.raises(_lib.WhallmError, match=msg):
            _lib.call(entry, *{**base, **kw}.values())


NORM = dict(residual=A, fp32=1, y=A, weight=A, offset=0.0, eps=1e-6, tokens=4, hidden=64, pow2=0, residual_out=A, q=A, scales=A, x=A,
            stream=None)
ROWS = dict(x=A, fp32=0, rows=4, width=64, swiglu=0, up_first=0, limit=0.0, pow2=0, q=A, scales=A, stream=None)
LINEAR = dict(x=A, x_scales=A, tokens=4, k=64, weight=A, weight_scales=A, n=8, add=None, out_fp32=0, out=A, stream=None)
SAMPLE = dict(logits=A, fp32=1, rows=4, vocab=5000, uniforms=A, temperature=A, top_k=A, top_p=A, min_p=A, tokens=A, logp=A, workspace=A,
              workspace_bytes=1 << 30, stream=None)


def test_norm_c_refusals():
    refused("wm_norm_fp8", NORM, [
        ({"tokens": -1}, "negative"), ({"hidden": 0}, "hidden must be"), ({"hidden": 16385}, "hidden must be"), ({"fp32": 2}, "fp32 must be"),
        ({"pow2": 2}, "pow2 must be"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
        ({"residual": None}, "null"), ({"q": None}, "null"), ({"scales": None}, "null"),
        ({"residual": A + 2}, "aligned"), ({"residual_out": A + 2}, "aligned"), ({"residual": A + 1, "fp32": 0}, "aligned"),
        ({"y": A + 1}, "aligned"), ({"weight": A + 1}, "aligned"), ({"x": A + 1}, "aligned"), ({"scales": A + 2}, "aligned")])
    _lib.call("wm_norm_fp8", *{**NORM, "tokens": 0, "residual": None}.values())


def test_rows_c_refusals():
    refused("wm_fp8_rows", ROWS, [
        ({"rows": -1}, "negative"), ({"width": 0}, "width must be"), ({"width": (1 << 20) + 1}, "width must be"), ({"fp32": -1}, "fp32 must be"),
        ({"swiglu": 2}, "swiglu must be"), ({"up_first": 3}, "up_first must be"), ({"pow2": -1}, "pow2 must be"),
        ({"limit": -0.5}, "limit"), ({"limit": float("nan")}, "limit"), ({"x": None}, "null"), ({"q": None}, "null"),
        ({"scales": None}, "null"), ({"x": A + 1}, "aligned"), ({"x": A + 2, "fp32": 1}, "aligned"), ({"scales": A + 1}, "aligned"),
        ({"rows": 2 ** 31 - 1, "width": 1 << 20}, "too many rows"), ({"rows": (1 << 28) + 1, "width": 1}, "too many rows")])
    _lib.call("wm_fp8_rows", *{**ROWS, "rows": 0, "x": None}.values())


def test_linear_c_refusals():
    refused("wm_linear_fp8", LINEAR, [
        ({"tokens": -1}, "tokens must be"), ({"tokens": 2 ** 31 - 1}, "tokens must be"), ({"k": 0}, "k must be"), ({"k": 24}, "k must be"),
        ({"k": (1 << 20) + 16}, "k must be"), ({"n": 0}, "n must be"), ({"n": 2 ** 31 - 1}, "n must be"), ({"out_fp32": 2}, "out_fp32"),
        ({"x": None}, "null"), ({"x_scales": None}, "null"), ({"weight": None}, "null"), ({"weight_scales": None}, "null"),
        ({"out": None}, "null"), ({"x": A + 8}, "16-byte"), ({"weight": A + 4}, "16-byte"), ({"x_scales": A + 2}, "aligned"),
        ({"weight_scales": A + 1}, "aligned"), ({"out": A + 1}, "aligned"), ({"out": A + 2, "out_fp32": 1}, "aligned"), ({"add": A + 1}, "aligned"),
        ({"tokens": 2147418112, "n": 2147418112}, "too many rows")])
    _lib.call("wm_linear_fp8", *{**LINEAR, "tokens": 0, "x": None}.values())


def test_sample_c_refusals():
    refused("wm_sample_logits", SAMPLE, [
        ({"rows": -1}, "negative"), ({"vocab": 0}, "vocab must be"), ({"vocab": (1 << 22) + 1}, "vocab must be"), ({"fp32": 2}, "fp32 must be"),
        ({"rows": 2 ** 31 - 1}, "too many rows"), ({"logits": None}, "null"), ({"uniforms": None}, "null"), ({"tokens": None}, "null"),
        ({"logp": None}, "null"), ({"logits": A + 2}, "aligned"), ({"logits": A + 1, "fp32": 0}, "aligned"), ({"uniforms": A + 2}, "aligned"),
        ({"temperature": A + 1}, "aligned"), ({"top_k": A + 2}, "aligned"), ({"top_p": A + 1}, "aligned"), ({"min_p": A + 3}, "aligned"),
        ({"tokens": A + 2}, "aligned"), ({"logp": A + 1}, "aligned"), ({"workspace": None}, "workspace"), ({"workspace": A + 8}, "workspace"),
        ({"workspace_bytes": _lib.load().wm_sample_logits_workspace_size(4, 5000) - 1}, "workspace")])
    _lib.call("wm_sample_logits", *{**SAMPLE, "rows": 0, "logits": None}.values())


def test_sample_workspace():
    size = _lib.load().wm_sample_logits_workspace_size
    assert size(-1, 5000) == size(4, 0) == size(4, (1 << 22) + 1) == size(4, 100) == size(0, 5000) == 0
    assert 0 < size(1, 129280) < size(2, 129280) <= size(1 << 20, 129280) < 2 ** 27   # sets of rows share it
    assert 0 < size(1, 1 << 22) < 2 ** 20


def named():
    """Each call with what passes every check but the last, and its float inputs."""
    r, y, w = torch.zeros(6, 256), torch.zeros(6, 256, dtype=BF16), torch.zeros(256, dtype=BF16)
    x8, w8 = torch.zeros(6, 256).to(F8), torch.zeros(40, 256).to(F8)
    per = lambda: torch.zeros(6)   # noqa: E731
    return [(ops.norm_fp8, dict(residual=r, y=y, weight=w, residual_out=r.clone()), ["residual", "y", "weight", "residual_out"]),
            (ops.quantize_fp8, dict(x=r), ["x"]), (ops.swiglu_fp8, dict(gate_up=y), ["gate_up"]),
            (ops.linear_fp8, dict(x=x8, x_scales=torch.zeros(6, 2), weight=w8, weight_scales=torch.zeros(1, 2), add=torch.zeros(6, 40, dtype=BF16)),
             ["x_scales", "weight_scales", "add"]),
            (ops.sample_logits, dict(logits=r, uniforms=per(), temperature=per(), top_k=torch.zeros(6, dtype=torch.int32), top_p=per(),
                                     min_p=per()), ["logits", "uniforms", "temperature", "top_p", "min_p"])]


CASES = [(i, name) for i, (_, _, names) in enumerate(named()) for name in names]


@pytest.mark.parametrize("i", range(len(named())))
def test_device_tensors_only(i):
    call, kw, _ = named()[i]
    with pytest.raises(ValueError, match="device"):
        call(**kw)
    with torch.inference_mode(), pytest.raises(ValueError, match="device"):
        call(**kw)


@pytest.mark.parametrize("i,name", CASES)
def test_gradients_and_tangents_are_refused(i, name):
    call, kw, _ = named()[i]
    plain = kw[name]
    kw[name] = plain.clone().requires_grad_()
    with pytest.raises(ValueError, match="autograd"):
        call(**kw)
    with torch.no_grad(), pytest.raises(ValueError, match="device"):
        call(**kw)
    for grad_mode in (True, False):
        with fwad.dual_level(), torch.set_grad_enabled(grad_mode):
            kw[name] = fwad.make_dual(plain, torch.ones_like(plain))
            with pytest.raises(ValueError, match="forward-mode"):
                call(**kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(residual=torch.zeros(6, 256, dtype=torch.half)), "float32 or bfloat16"), (dict(residual=torch.zeros(())), "must be"),
    (dict(residual=torch.zeros(6, 0)), "H from 1"), (dict(residual=torch.zeros(2, 16385)), "H from 1"), (dict(eps=-1e-9), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(y=torch.zeros(6, 256)), "y must be"), (dict(y=torch.zeros(6, 255, dtype=BF16)), "match residual"),
    (dict(y=torch.zeros(256, dtype=BF16)), "match residual"), (dict(weight=torch.zeros(256)), "weight must be"),
    (dict(weight=torch.zeros(255, dtype=BF16)), r"weight must be \[H\]"), (dict(weight=torch.zeros(1, 256, dtype=BF16)), r"weight must be \[H\]"),
    (dict(y=None), "needs y"), (dict(residual_out=torch.zeros(6, 256, dtype=BF16)), "residual_out must be"),
    (dict(residual_out=torch.zeros(5, 256)), "residual_out must be"), (dict(residual_out=torch.zeros(256, 6).t()), "residual_out must be"),
    (dict(residual=torch.empty(2 ** 31, 1, device="meta")), "below 2")])
def test_norm_refusals(kw, msg):
    base = named()[0][1]
    with pytest.raises(ValueError, match=msg):
        ops.norm_fp8(**{**base, **kw})


def test_residual_out_over_an_input():
    r, y = torch.zeros(3, 8, dtype=BF16), torch.zeros(3, 8, dtype=BF16)
    row = torch.zeros(1, 8, dtype=BF16)
    buf = torch.zeros(40, dtype=BF16)
    for args, out in (((r, y), y), ((row.clone(), row.clone(), row[0]), row), ((buf[:24].view(3, 8), y), buf[8:32].view(3, 8))):
        with pytest.raises(ValueError, match="share no memory"):
            ops.norm_fp8(*args, residual_out=out)
    with pytest.raises(ValueError, match="device"):
        ops.norm_fp8(r, y, residual_out=r)


@pytest.mark.parametrize("call,x,kw,msg", [
    (ops.quantize_fp8, torch.zeros(2, 8, dtype=torch.half), {}, "bfloat16 or float32"), (ops.quantize_fp8, torch.zeros(()), {}, "must be"),
    (ops.quantize_fp8, torch.zeros(3, 0), {}, "must be"), (ops.quantize_fp8, torch.empty(1, (1 << 20) + 1, device="meta"), {}, "at most"),
    (ops.quantize_fp8, torch.empty(2 ** 31, 1, device="meta"), {}, "below 2"),
    (ops.swiglu_fp8, torch.zeros(2, 7), {}, "2 I"), (ops.swiglu_fp8, torch.zeros(2, 8, dtype=torch.int32), {}, "bfloat16 or float32"),
    (ops.swiglu_fp8, torch.empty(1, (1 << 21) + 2, device="meta"), {}, "at most"),
    (ops.swiglu_fp8, torch.zeros(2, 8), {"limit": 1e-60}, "limit"), (ops.swiglu_fp8, torch.zeros(2, 8), {"limit": -1.0}, "limit"), (ops.swiglu_fp8, torch.zeros(2, 8), {"limit": float("nan")}, "limit")])
def test_rows_refusals(call, x, kw, msg):
    with pytest.raises(ValueError, match=msg):
        call(x, **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(out_dtype=torch.half), "out_dtype"), (dict(out_dtype="bf16"), "torch.dtype"), (dict(x=torch.zeros(6, 256)), "float8_e4m3fn or uint8"),
    (dict(weight=torch.zeros(40, 256, dtype=BF16)), "float8_e4m3fn or uint8"), (dict(x=torch.zeros(6, 240, dtype=torch.uint8)), r"weight \[N, K\]"),
    (dict(weight=torch.zeros(256, dtype=torch.uint8)), r"weight \[N, K\]"), (dict(x_scales=torch.zeros(6, 2, dtype=BF16)), "x_scales must be"),
    (dict(x_scales=torch.zeros(6, 1)), "x_scales must be"), (dict(x_scales=torch.zeros(2)), "x_scales must be"),
    (dict(x_scales=torch.zeros(5, 2)), "x_scales must be"), (dict(weight_scales=torch.zeros(2, 2)), "weight_scales must be"),
    (dict(weight_scales=torch.zeros(1, 3)), "weight_scales must be"), (dict(add=torch.zeros(6, 40)), "add must be"),
    (dict(add=torch.zeros(40, dtype=BF16)), "add must be"),
    (dict(x=torch.zeros(6, 40, dtype=torch.uint8), weight=torch.zeros(4, 40, dtype=torch.uint8)), "multiple of 16"),
    (dict(x=torch.zeros(6, 0, dtype=torch.uint8), weight=torch.zeros(4, 0, dtype=torch.uint8)), "multiple of 16"),
    (dict(weight=torch.zeros(0, 256, dtype=torch.uint8)), "N must be"),
    (dict(x=torch.empty(2 ** 31 - 1, 16, dtype=torch.uint8, device="meta"), weight=torch.zeros(4, 16, dtype=torch.uint8)), "tokens must be")])
def test_linear_refusals(kw, msg):
    base = named()[3][1]
    with pytest.raises(ValueError, match=msg):
        ops.linear_fp8(**{**base, **kw})


@pytest.mark.parametrize("kw,msg", [
    (dict(logits=torch.zeros(256)), "rows, vocab"), (dict(logits=torch.zeros(6, 0)), "rows, vocab"),
    (dict(logits=torch.zeros(6, 8, dtype=torch.half)), "bfloat16 or float32"), (dict(logits=torch.empty(6, (1 << 22) + 1, device="meta")), "at most"),
    (dict(uniforms=torch.zeros(5)), r"uniforms must be \[rows\]"), (dict(uniforms=torch.zeros(6, 1)), r"uniforms must be \[rows\]"),
    (dict(uniforms=torch.zeros(6, dtype=torch.double)), "uniforms must be"), (dict(temperature=torch.zeros(1)), "temperature must be"),
    (dict(top_k=torch.zeros(6, dtype=torch.int64)), "top_k must be"), (dict(top_k=torch.zeros(6)), "top_k must be"),
    (dict(top_p=torch.zeros(6, dtype=BF16)), "top_p must be"), (dict(min_p=torch.zeros(7)), "min_p must be")])
def test_sample_refusals(kw, msg):
    base = named()[4][1]
    with pytest.raises(ValueError, match=msg):
        ops.sample_logits(**{**base, **kw})
