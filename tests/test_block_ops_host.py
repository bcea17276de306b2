"""Refusals of the calls around the expert products, without a GPU: the C entry points' argument checks
and the compiled host side's, which come before the one for device tensors."""
import pytest
import torch

from whallm_amd import _lib, ops

A = 0x10000   # an aligned address that is never read


def sort_args(**kw):
    a = dict(x=A, fp32=0, tokens=4, hidden=64, indices=A, k=2, experts=8, tile_rows=16, rows=A, order=A, inverse=A, offsets=A,
             tiles=A, tile_count=A, workspace=A, workspace_bytes=1 << 30, stream=None)
    a.update(kw)
    return a.values()


@pytest.mark.parametrize("kw,msg", [
    ({"tokens": -1}, "negative"), ({"k": 0}, "k must be"), ({"k": 65}, "k must be"), ({"hidden": 0}, "hidden must be"),
    ({"hidden": 1 << 21}, "hidden must be"), ({"fp32": 2}, "fp32 must be"), ({"experts": 0}, "experts must be"),
    ({"experts": 1025}, "experts must be"), ({"tile_rows": 0}, "tile_rows"), ({"tokens": 1 << 30, "k": 2}, "below 2"),
    ({"tokens": 2 ** 31 - 1, "k": 1}, "too many rows"),
    ({"x": None}, "null pointer"), ({"indices": None}, "null pointer"), ({"rows": None}, "null pointer"),
    ({"offsets": None}, "null pointer"), ({"workspace": None, "tokens": 1 << 20}, "null pointer"),
    ({"workspace_bytes": 8, "tokens": 1 << 20}, "workspace too small"),
    ({"x": A + 1}, "aligned"), ({"rows": A + 2, "fp32": 1}, "aligned"), ({"tiles": A + 4}, "aligned"),
])
def test_sort_tokens_c_refusals(kw, msg):
    with pytest.raises(_lib.WhallmError, match=msg):
        _lib.call("wm_sort_tokens", *sort_args(**kw))


def test_rows_c_refusals():
    def backward(drows=A, fp32=0, inverse=A, tokens=4, k=2, hidden=64, dx=A):
        _lib.call("wm_sort_tokens_backward", drows, fp32, inverse, tokens, k, hidden, dx, None)

    def combine(rows=A, fp32=0, weights=A, inverse=A, tokens=4, k=2, hidden=64, add=None, y=A):
        _lib.call("wm_combine_rows", rows, fp32, weights, inverse, tokens, k, hidden, add, y, None)

    def grads(dy=A, rows=A, fp32=0, weights=A, inverse=A, present=A, tokens=4, k=2, hidden=64, drows=A, dweights=A):
        _lib.call("wm_combine_rows_backward", dy, rows, fp32, weights, inverse, present, tokens, k, hidden, drows, dweights, None)

    for call in (backward, combine, grads):
        for kw, msg in (({"tokens": -2}, "negative"), ({"k": 0}, "k must be"), ({"k": 65}, "k must be"),
                        ({"hidden": 0}, "hidden must be"), ({"fp32": -1}, "fp32 must be"), ({"inverse": None}, "null pointer")):
            with pytest.raises(_lib.WhallmError, match=msg):
                call(**kw)
        call(tokens=0)   # nothing to do
    for call, kw in ((backward, {"dx": A + 1}), (combine, {"add": A + 1}), (combine, {"fp32": 1, "y": A + 2}), (grads, {"dy": A + 1})):
        with pytest.raises(_lib.WhallmError, match="aligned"):
            call(**kw)
    for call in (backward, combine, grads):
        with pytest.raises(_lib.WhallmError, match="too many rows"):
            call(tokens=1 << 24, k=1, hidden=4096)
    for kw in ({"present": None}, {"drows": None}, {"dweights": None}):
        with pytest.raises(_lib.WhallmError, match="null pointer"):
            grads(**kw)


def test_all_take_device_tensors_only():
    """What passes every other check."""
    x, idx, w = torch.zeros(6, 8), torch.zeros(6, 2, dtype=torch.int32), torch.zeros(6, 2)
    rows = torch.zeros(12, 8)
    p = ops.Permutation(*(torch.zeros(n, dtype=torch.int32) for n in (12, 12, 5, 8, 1)))
    y = torch.zeros(6, 8, dtype=torch.bfloat16)
    for call in (lambda: ops.sort_tokens(x, idx, 4), lambda: ops.sort_tokens_backward(rows, p, 2),
                 lambda: ops.combine_rows(rows, w, p, x), lambda: ops.combine_rows_backward(x, rows, w, p),
                 lambda: ops.block_norm(x, y, gate=torch.zeros(6, 1)), lambda: ops.block_norm_backward(y, None, x, y),
                 lambda: ops.process_logits(x, log_probs=True)):
        with pytest.raises(ValueError, match="device"):
            call()


def test_rows_python_refusals():
    x, idx, w = torch.zeros(6, 8), torch.zeros(6, 2, dtype=torch.int32), torch.zeros(6, 2)
    rows = torch.zeros(12, 8)
    p = ops.Permutation(*(torch.zeros(n, dtype=torch.int32) for n in (12, 12, 5, 8, 1)))
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        ops.sort_tokens(x.half(), idx, 4)
    with pytest.raises(ValueError, match="indices must be"):
        ops.sort_tokens(x, idx.long(), 4)
    with pytest.raises(ValueError, match="indices must be"):
        ops.sort_tokens(x, idx[:5], 4)
    with pytest.raises(ValueError, match="positive"):
        ops.sort_tokens(x[:, :0], idx, 4)
    with pytest.raises(ValueError, match="autograd"):
        ops.sort_tokens(x.clone().requires_grad_(), idx, 4)
    with pytest.raises(ValueError, match="not that of these rows"):
        ops.sort_tokens_backward(rows[:10], p, 2)
    with pytest.raises(ValueError, match="k rows of every token"):
        ops.sort_tokens_backward(rows, p, 5)
    with pytest.raises(ValueError, match="weights"):
        ops.combine_rows(rows, w[:5], p)
    with pytest.raises(ValueError, match="weights must be torch.float32"):
        ops.combine_rows(rows, w.double(), p)
    with pytest.raises(ValueError, match="add must be"):
        ops.combine_rows(rows, w, p, x.bfloat16())
    with pytest.raises(ValueError, match="add must be"):
        ops.combine_rows(rows, w, p, x[:5])
    with pytest.raises(ValueError, match="autograd"):
        ops.combine_rows(rows, w.clone().requires_grad_(), p)
    with pytest.raises(ValueError, match="dy must be"):
        ops.combine_rows_backward(x.bfloat16(), rows, w, p)
    with pytest.raises(ValueError, match="dy must be"):
        ops.combine_rows_backward(x[:, :4], rows, w, p)
    with torch.no_grad(), pytest.raises(ValueError, match="device"):   # past the check
        ops.combine_rows(rows.requires_grad_(), w, p)


# ----------------------------------------------------------------------------- block norm

def norm_form(**kw):
    f = dict(post_weight=A, pre_weight=A, gate=None, weight_offset=0.0, scale=1.0, eps=1e-6, post_norm=1, gate_kind=0, gate_fp32=0,
             gate_sigmoid=0, residual_fp32=1)
    f.update(kw)
    return _lib.BlockNormFormC(*f.values())


def norm_call(form=None, residual=A, y=A, tokens=2, hidden=64, residual_out=A, x=A, **kw):
    _lib.call("wm_block_norm", form or norm_form(**kw), residual, y, tokens, hidden, residual_out, x, None)


def norm_grad_call(dx=A, dres=A, residual_out=A, y=A, tokens=2, hidden=64, dr=A, dy=A, dpost=A, dpre=A, dgate=None, ws=A,
                   ws_bytes=1 << 30, **kw):
    _lib.call("wm_block_norm_backward", norm_form(**kw), dx, dres, residual_out, y, tokens, hidden, dr, dy, dpost, dpre, dgate, ws,
              ws_bytes, None)


@pytest.mark.parametrize("kw,msg", [
    ({"tokens": -1}, "negative"), ({"hidden": 0}, "hidden must be"), ({"hidden": 16385}, "hidden must be"),
    ({"gate_kind": 4, "gate": A}, "gate_kind"), ({"gate_kind": 1}, "go together"), ({"gate": A}, "go together"),
    ({"post_norm": 0}, "needs the post norm"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"y": None}, "null pointer"),
    ({"y": A + 1}, "aligned"), ({"gate_kind": 2, "gate_fp32": 1, "gate": A + 2, "dgate": A}, "aligned"),
])
def test_block_norm_c_refusals(kw, msg):
    with pytest.raises(_lib.WhallmError, match=msg):
        norm_call(**{k: v for k, v in kw.items() if k != "dgate"})
    with pytest.raises(_lib.WhallmError, match="go with their gradients" if kw.get("gate") and "dgate" not in kw and kw.get("gate_kind") in (1, 2, 3) else msg):
        norm_grad_call(**kw)


def test_block_norm_c_refusals_of_one_side():
    for kw, msg in (({"residual": None}, "null pointer"), ({"residual_out": None}, "null pointer"), ({"x": None}, "null pointer"),
                    ({"residual": A + 2}, "aligned")):
        with pytest.raises(_lib.WhallmError, match=msg):
            norm_call(**kw)
    with pytest.raises(_lib.WhallmError, match="null form"):
        _lib.call("wm_block_norm", None, A, A, 1, 64, A, A, None)
    for kw, msg in (({"dx": None}, "null pointer"), ({"dr": None}, "null pointer"), ({"dy": None}, "null pointer"),
                    ({"ws": None}, "null pointer"), ({"ws_bytes": 64}, "workspace too small"), ({"ws": A + 4}, "misaligned"),
                    ({"dpost": None}, "gradients"), ({"dpre": None}, "gradients"), ({"dgate": A}, "gradients"),
                    ({"gate": A, "gate_kind": 1}, "gradients"), ({"dpre": A + 2}, "aligned"), ({"dres": A + 2}, "aligned")):
        with pytest.raises(_lib.WhallmError, match=msg):
            norm_grad_call(**kw)
    norm_call(tokens=0)
    lib = _lib.load()
    assert lib.wm_block_norm_backward_workspace_size(-1, 64) == 0 and lib.wm_block_norm_backward_workspace_size(4, 0) == 0


def test_block_norm_python_refusals():
    r, y, w = torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(8, dtype=torch.bfloat16)
    for args, kw, msg in (
            ((r.half(), y), {}, "residual must be"), ((r, y.float()), {}, "y must be"), ((r, y[:2]), {}, "match residual"),
            ((r, y, w.float()), {}, "post_weight must be"), ((r, y, w[:4]), {}, "weights must be"),
            ((r, y, w), {"post_norm": False}, "needs post_norm"), ((r, y), {"eps": -1.0}, "eps"),
            ((r, y), {"gate": torch.zeros(3)}, "gate must be"), ((r, y), {"gate": torch.zeros(3, 1).double()}, "gate must be"),
            ((r, y), {"residual_out": torch.zeros(8, 3).t()}, "residual_out"), ((r.clone().requires_grad_(), y), {}, "autograd")):
        with pytest.raises(ValueError, match=msg):
            ops.block_norm(*args, **kw)
    for dx, dres, msg in ((y.float(), None, "dx must be"), (y[:2], None, "dx must match"), (y, y, "dresidual must be"),
                          (y, r[:2], "dresidual must be")):
        with pytest.raises(ValueError, match=msg):
            ops.block_norm_backward(dx, dres, r, y)


# ----------------------------------------------------------------------------- logits

def logits_call(logits=A, fp32=1, rows=2, vocab=100, log_probs=1, out=A, ws=A, ws_bytes=1 << 20, **kw):
    r = dict(history=None, history_stride=0, history_len=0, biases=0, lengths=None, prompt_lengths=None, repetition=None,
             frequency=None, presence=None, bias_ids=None, bias_values=None, bias_stride=0, mask=None, mask_stride=0, temperature=None)
    r.update(kw)
    _lib.call("wm_process_logits", logits, fp32, rows, vocab, _lib.LogitRulesC(*r.values()), log_probs, out, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,msg", [
    ({"rows": -1}, "rows must"), ({"vocab": 0}, "vocab must"), ({"vocab": (1 << 22) + 1}, "vocab must"), ({"fp32": 3}, "fp32 must"),
    ({"rows": 1 << 30, "vocab": 1 << 22}, "too many rows"), ({"rows": 1 << 24}, "too many rows"),
    ({"history": A, "history_len": 1 << 20}, "history_len"),
    ({"history": A, "history_len": -1}, "history_len"), ({"biases": 2048}, "biases must"), ({"biases": -1}, "biases must"),
    ({"history_stride": -1}, "strides"), ({"lengths": A}, "without a history"), ({"prompt_lengths": A}, "without a history"),
    ({"bias_ids": A}, "go together"), ({"bias_values": A}, "go together"), ({"logits": None}, "null pointer"),
    ({"out": None}, "null pointer"), ({"logits": A + 2}, "aligned"), ({"out": A + 2}, "aligned"), ({"mask": A + 1}, "aligned"),
    ({"ws": None}, "workspace"), ({"ws_bytes": 0}, "workspace"), ({"ws": A + 4}, "workspace"),
])
def test_process_logits_c_refusals(kw, msg):
    with pytest.raises(_lib.WhallmError, match=msg):
        logits_call(**kw)


def test_process_logits_python_refusals():
    logits = torch.zeros(3, 40)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(_lib.WhallmError, match="null rules"):
        _lib.call("wm_process_logits", A, 1, 1, 10, None, 0, A, None, 0, None)
    logits_call(rows=0)
    for args, kw, msg in (
            ((logits.half(),), {}, "bfloat16 or float32"), ((logits[0],), {}, "logits must be"),
            ((logits,), {"history": i32(2, 5)}, "history must be"), ((logits,), {"history": torch.zeros(3, 5)}, "history must be"),
            ((logits,), {"lengths": i32(3)}, "need a history"), ((logits,), {"history": i32(3, 5), "lengths": i32(2)}, "lengths must be"),
            ((logits,), {"history": i32(3, 5), "lengths": torch.zeros(3).long()}, "lengths must be"),
            ((logits,), {"repetition": torch.zeros(2)}, "repetition must be"), ((logits,), {"temperature": torch.zeros(3).double()}, "temperature must be"),
            ((logits,), {"bias_ids": i32(3, 2)}, "go together"), ((logits,), {"bias_ids": i32(3, 2), "bias_values": torch.zeros(3, 3)}, "one shape"),
            ((logits,), {"mask": i32(3, 1)}, "a bit for every token"), ((logits,), {"mask": torch.zeros(3, 2).bool()}, "mask must be"),
            ((logits,), {"out": torch.zeros(3, 40).bfloat16()}, "out must be"), ((logits,), {"out": torch.zeros(40, 3).t()}, "out must be"),
            ((logits,), {"out": torch.zeros(124)[4:].view(3, 40).requires_grad_()}, "autograd"),
            ((logits,), {"temperature": torch.ones(3).requires_grad_()}, "autograd"),
            ((logits.clone().requires_grad_(),), {}, "autograd")):
        with pytest.raises(ValueError, match=msg):
            ops.process_logits(*args, **kw)


def test_outputs_that_overlap_an_input_partly():
    buf = torch.zeros(64)
    rows = lambda at: buf[at:at + 24].view(3, 8)  # noqa: E731
    y = torch.zeros(3, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="share no memory"):
        ops.block_norm(rows(0), y, residual_out=rows(4))
    with pytest.raises(ValueError, match="share no memory"):
        ops.block_norm(rows(0), buf[30:42].view(torch.bfloat16).view(3, 8), residual_out=rows(24))
    with pytest.raises(ValueError, match="share no memory"):
        ops.process_logits(rows(0), out=rows(8))
    with pytest.raises(ValueError, match="device"):          # the input itself is fine
        ops.process_logits(rows(0), out=rows(0))
