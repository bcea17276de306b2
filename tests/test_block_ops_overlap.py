"""An output that the caller gives may be the one input that the call allows, and lies over no other: refused before
anything runs (no GPU needed; what passes stops at the check for device tensors)."""
import pytest
import torch

from whallm_amd import ops


def i32(t):
    return t.view(torch.int32)


@pytest.mark.parametrize("name", ["lengths", "prompt_lengths", "repetition", "frequency", "presence", "temperature"])
@pytest.mark.parametrize("at", [0, 5, 117])
def test_logits_out_over_values_of_its_rows(name, at):
    buf = torch.ones(130)
    logits, value = torch.zeros(3, 40), buf[at:at + 3]
    history = torch.zeros(3, 5, dtype=torch.int32)
    with pytest.raises(ValueError, match="share no memory"):
        ops.process_logits(logits, history=history, out=buf[:120].view(3, 40), **{name: i32(value) if "lengths" in name else value})
    with pytest.raises(ValueError, match="device"):          # right behind it is fine
        ops.process_logits(logits, history=history, out=buf[:120].view(3, 40),
                           **{name: i32(buf[120:123]) if "lengths" in name else buf[120:123]})


@pytest.mark.parametrize("shape", ["whole", "part"])
def test_logits_out_over_a_list(shape):
    buf = torch.zeros(3, 40)
    logits = torch.zeros(3, 40)
    some = buf if shape == "whole" else buf[1:2]
    ids = torch.zeros(some.shape, dtype=torch.int32)
    for kw in ({"history": i32(some)}, {"bias_ids": i32(some), "bias_values": torch.zeros(some.shape)},
               {"bias_ids": ids, "bias_values": some}, {"mask": i32(buf.view(-1)[2:8].view(3, 2))}):
        with pytest.raises(ValueError, match="share no memory"):
            ops.process_logits(logits, out=buf, **kw)


def test_logits_out_over_bf16_logits():
    buf = torch.zeros(3, 40)
    with pytest.raises(ValueError, match="share no memory"):
        ops.process_logits(buf.view(torch.bfloat16)[:, :40].contiguous().set_(buf.view(torch.bfloat16).untyped_storage(), 0, (3, 40)), out=buf)


def test_residual_out_is_the_residual_or_apart():
    r, y = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(3, 8, dtype=torch.bfloat16)
    row, full = torch.zeros(1, 8, dtype=torch.bfloat16), torch.zeros(3, 8, dtype=torch.bfloat16)
    for args, kw in (((r, y), {"residual_out": y}), ((r, y), {"gate": full, "residual_out": full}),
                     ((row, row.clone()), {"post_weight": row[0], "residual_out": row.clone().set_(row.untyped_storage(), 0, (1, 8))}),
                     ((row.clone(), row.clone()), {"pre_weight": row[0], "residual_out": row})):
        with pytest.raises(ValueError, match="share no memory"):
            ops.block_norm(*args, **kw)
    with pytest.raises(ValueError, match="device"):
        ops.block_norm(r, y, gate=full, residual_out=r)
    # as many elements from the same place on, but of rows that a view turned round: the residual is then copied first
    with pytest.raises(ValueError, match="device"):
        ops.block_norm(r.view(8, 3).t(), y, residual_out=r)


def test_memory_that_two_storages_hold():
    """Tensors of one memory that do not share a storage object."""
    import numpy as np
    memory = np.zeros(200, np.float32)
    a, b = torch.from_numpy(memory[:120]).view(3, 40), torch.from_numpy(memory[8:128]).view(3, 40)
    with pytest.raises(ValueError, match="share no memory"):
        ops.process_logits(a, out=b)
    with pytest.raises(ValueError, match="device"):
        ops.process_logits(a, out=torch.from_numpy(memory[:120]).view(3, 40))


def test_nothing_overlaps_an_empty_output():
    empty = torch.zeros(0, 40)
    with pytest.raises(ValueError, match="device"):
        ops.process_logits(torch.zeros(0, 40), out=empty)
