"""The launches of a draw: the pass over the bins is sent only where a row may take bins, so not for a temperature or min-p alone.

Counted as the kernel nodes of a captured call.
"""
import ctypes

import pytest
import torch

import whallm_amd as wa

pytestmark = pytest.mark.gpu


def hip():
    """The HIP runtime that this process has loaded."""
    with open("/proc/self/maps") as maps:
        return ctypes.CDLL(next(line.split()[-1] for line in maps if "libamdhip64" in line))


def nodes(call):
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        out = call()
    count = ctypes.c_size_t()
    assert hip().hipGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(count)) == 0
    graph.instantiate()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, call()))
    return count.value


@pytest.mark.parametrize("V,rows", [(2048, 3), (5000, 3), (129280, 1)])
def test_launches_of_a_draw(device, V, rows):
    logits, u = torch.randn(rows, V, device=device), torch.rand(rows, device=device)
    per = lambda v, t=torch.float32: torch.full((rows,), v, dtype=t, device=device)   # noqa: E731
    one = V <= 2048
    forms = [({}, 3), (dict(temperature=per(0.7)), 3), (dict(temperature=per(0.0)), 3), (dict(min_p=per(0.1)), 3),
             (dict(temperature=per(0.7), min_p=per(0.1)), 3), (dict(top_p=per(0.9)), 4), (dict(top_k=per(40, torch.int32)), 4),
             (dict(temperature=per(0.7), top_k=per(0, torch.int32), top_p=per(1.0)), 4)]
    for rules, want in forms:
        assert nodes(lambda: wa.sample_logits(logits, u, **rules)) == (1 if one else want), rules
