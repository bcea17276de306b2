"""GPU parity of the logit steps before acceptance (wm_process_logits) against the formula in 64 bits.

Bar: the running error of the same steps in fp32 (running_error.py). The log-softmax: a term exp(l - top)
is exp2 of the difference times log2 e, three roundings of the argument, over the five levels at
which maxima meet (thread, wave, workgroup, chunks, wave): their differences add up to l - top, and each
level adds an exp2 (2 units) and a product (1). A row's sum passes at most 32 values of a thread, 6 steps
of a wave, 6 of a workgroup, the chunks of a lane and 6 steps again. The logarithm is good to 2 units and
has the sum's relative error, and two subtractions follow.
"""
import numpy as np
import pytest
import torch

import whallm_amd as wa
from running_error import Fp32, U, check

pytestmark = pytest.mark.gpu

SUM = 32 + 6 + 6 + 14 + 6


def f64(t):
    return t.detach().double().cpu().numpy()


def want_logits(logits, log_probs=False, history=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None,
                presence=None, bias_ids=None, bias_values=None, mask=None, temperature=None):
    R, V = logits.shape
    n = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    history, lengths, prompts, ids, values, mask = map(n, (history, lengths, prompt_lengths, bias_ids, bias_values, mask))
    row = lambda a, r: a[0 if a.shape[0] == 1 else r]  # noqa: E731
    per = lambda t, r, default: default if t is None else float(t[r])  # noqa: E731
    out_v, out_e = np.empty((R, V)), np.empty((R, V))
    raw = f64(logits)
    for r in range(R):
        l = Fp32(raw[r])
        if history is not None:
            h = row(history, r)
            end = len(h) if lengths is None else min(max(int(lengths[r]), 0), len(h))
            p = 0 if prompts is None else min(max(int(prompts[r]), 0), end)
            ok = lambda a: a[(a >= 0) & (a < V)]  # noqa: E731
            seen = np.bincount(ok(h[:end]), minlength=V) > 0
            count = np.bincount(ok(h[p:end]), minlength=V).astype(np.float64)
            rep = per(repetition, r, 1.0)
            div, mul = l * (Fp32(1.0) / Fp32(rep)), l * rep    # by the reciprocal
            pos = l.v > 0
            l = Fp32(np.where(seen, np.where(pos, div.v, mul.v), l.v), np.where(seen, np.where(pos, div.e, mul.e), l.e))
            l = l - Fp32(per(frequency, r, 0.0)) * Fp32(count) - Fp32(per(presence, r, 0.0) * (count > 0))
        if ids is not None:
            b = np.zeros(V)
            for i, v in zip(row(ids, r), row(values, r)):
                if 0 <= i < V:
                    b[i] = v
            l = l + Fp32(b)
        t = per(temperature, r, 1.0)
        if t > 0:
            l = l * (Fp32(1.0) / Fp32(t))    # by the reciprocal
        if mask is not None:
            bits = np.unpackbits(row(mask, r).view(np.uint8), bitorder="little")[:V] != 0
            l = Fp32(np.where(bits, l.v, -np.inf), np.where(bits, l.e, 0.0))
        if log_probs:
            l = log_softmax(l)
        out_v[r], out_e[r] = l.v, l.e
    return Fp32(out_v, out_e)


def log_softmax(l):
    top = np.fmax.reduce(l.v)
    if np.isneginf(top) and not np.isnan(l.v).any():
        return l
    with np.errstate(invalid="ignore", over="ignore"):
        arg = l.v - top
        e_arg = np.where(np.isneginf(l.v), 0.0, 2 * l.e.max() + 3.01 * U * np.abs(np.where(np.isneginf(l.v), 0.0, arg)))
        term = np.exp(arg)
        total = term.sum()
        rel = (term * (e_arg * 1.01 + 5 * 4 * U)).sum() / total + SUM * U
        log = np.log(total)
        v = np.where(np.isneginf(l.v), -np.inf, l.v - top - log)
        e = l.e + l.e.max() + rel * 1.01 + 4 * U * abs(log) + 2 * U * (np.abs(np.where(np.isneginf(l.v), 0, arg)) + abs(log))
    return Fp32(v, e)


def make(rng, R, V, L, device, dtype=torch.float32, shared=False, biases=0, mask=None, dup=False, penalties=True, temps=True):
    to = lambda a, t=None: torch.from_numpy(np.ascontiguousarray(a)).to(device) if t is None else torch.from_numpy(np.ascontiguousarray(a)).to(t).to(device)  # noqa: E731
    kw = {}
    logits = to(rng.standard_normal((R, V)).astype(np.float32) * 4, dtype)
    if L:
        n = 1 if shared else R
        h = (rng.random((n, L)) ** 3 * V).astype(np.int32)
        h = np.where(rng.random((n, L)) < 0.05, np.array([-1, V, V + 7, -2 ** 31, 2 ** 31 - 1], np.int32)[rng.integers(0, 5, (n, L))], h).astype(np.int32)
        kw.update(history=to(h), lengths=to(rng.integers(-2, L + 3, R).astype(np.int32)),
                  prompt_lengths=to(rng.integers(-2, L + 3, R).astype(np.int32)))
    if penalties:
        kw.update(repetition=to(0.5 + rng.random(R).astype(np.float32) * 2), frequency=to(rng.standard_normal(R).astype(np.float32)),
                  presence=to(rng.standard_normal(R).astype(np.float32)))
    if temps:
        t = 0.3 + rng.random(R).astype(np.float32) * 2
        t[::3] = 0.0
        kw["temperature"] = to(t)
    if biases:
        n = 1 if shared else R
        ids = rng.integers(-1, V + 1, (n, biases)).astype(np.int32) if dup else np.stack([rng.permutation(max(V, biases))[:biases] for _ in range(n)]).astype(np.int32)
        kw.update(bias_ids=to(ids), bias_values=to(rng.standard_normal((n, biases)).astype(np.float32) * 5))
    if mask:
        n, W = (1 if shared else R), -(-V // 32)
        words = rng.integers(0, 2 ** 32, (n, W), dtype=np.uint32) | rng.integers(0, 2 ** 32, (n, W), dtype=np.uint32)
        if mask == "none":
            words[0] = 0
        if mask == "one":
            words[:] = 0
            words[:, (V - 1) // 32] = np.uint32(1 << ((V - 1) % 32))
        kw["mask"] = to(words.view(np.int32))
    return logits, kw


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,L,shared,biases,mask", [
    (1, 1, 3, False, 1, None),
    (3, 5, 9, False, 2, "some"),
    (2, 33, 1, False, 0, "one"),
    (4, 4095, 50, True, 3, "some"),
    (5, 4096, 700, False, 40, None),
    (3, 4097, 0, False, 7, "some"),
    (7, 4104, 333, True, 0, "none"),
    (2, 20001, 6000, False, 2047, "some"),
    (40, 1000, 257, False, 16, "none"),
    (300, 64, 17, False, 5, "one"),
    (4, 129280, 4096, True, 300, "some"),
    (3, 20003, 9001, False, 700, "some"),     # more ids than a round of them
    (2, 50, 20000, True, 3, None),
    (1, 8192, 8193, False, 0, "some"),
    (40, 130001, 8200, False, 1, None),       # and more tokens than are kept
])
def test_matches_the_formula(device, R, V, L, shared, biases, mask, dtype):
    rng = np.random.default_rng(R + V + L)
    logits, kw = make(rng, R, V, L, device, dtype, shared, biases, mask, dup=V > 40)
    for log_probs in (False, True):
        got = wa.process_logits(logits, log_probs=log_probs, **kw)
        assert got.dtype == torch.float32
        check("logp" if log_probs else "logits", got, want_logits(logits, log_probs, **kw))


@pytest.mark.parametrize("drop", ["history", "lengths", "prompt_lengths", "repetition", "frequency", "presence", "bias_ids", "mask",
                                  "temperature", "everything"])
def test_each_step_may_be_left_out(device, drop):
    rng = np.random.default_rng(3)
    logits, kw = make(rng, 6, 300, 80, device, biases=9, mask="some")
    gone = {"history": ("history", "lengths", "prompt_lengths"), "bias_ids": ("bias_ids", "bias_values"), "everything": tuple(kw)}
    for name in gone.get(drop, (drop,)):
        kw.pop(name)
    for log_probs in (False, True):
        check(drop, wa.process_logits(logits, log_probs=log_probs, **kw), want_logits(logits, log_probs, **kw))
    if drop == "everything":
        assert torch.equal(wa.process_logits(logits), logits)


def test_infinities_and_nan(device):
    """Masked values never matter; -inf stays; rows without an allowed token are -inf throughout; NaN and
    +inf that are allowed spoil their own row only."""
    V = 9000
    logits = torch.randn(6, V, device=device)
    mask = torch.full((6, -(-V // 32)), -1, dtype=torch.int32, device=device)
    mask[:, 3] = 0                                  # tokens 96..127 are not allowed
    logits[0, 100], logits[0, 101], logits[0, 102] = float("nan"), float("inf"), torch.finfo(torch.float32).min
    logits[1, 5000:] = float("-inf")                # whole chunks
    mask[2] = 0
    logits[3, 8000] = float("nan")
    logits[4, 7] = float("inf")
    logits[5] = float("-inf")
    got = wa.process_logits(logits, mask=mask, log_probs=True)
    allowed = torch.ones(V, dtype=torch.bool, device=device)
    allowed[96:128] = False
    for r in (0, 1):
        want = torch.log_softmax(logits[r].double().masked_fill(~allowed, float("-inf")), 0)
        fin = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got[r]), fin) and not torch.isnan(got[r]).any()
        assert (got[r][fin] - want[fin]).abs().max() <= 1e-5
    assert torch.equal(got[2], torch.full((V,), float("-inf"), device=device)) and torch.equal(got[5], got[2])
    for r in (3, 4):
        assert torch.isinf(got[r][~allowed]).all()
    assert torch.isnan(got[3][allowed]).all() and torch.isnan(got[4, 7])
    # the type's lowest value is an ordinary, very unlikely logit
    low = torch.full((1, 64), torch.finfo(torch.float32).min, device=device)
    check("lowest", wa.process_logits(low, log_probs=True), want_logits(low, True))


def test_in_place_strided_and_no_rows(device):
    rng = np.random.default_rng(6)
    logits, kw = make(rng, 5, 8200, 100, device, biases=4, mask="some")
    for log_probs in (False, True):
        want = wa.process_logits(logits, log_probs=log_probs, **kw)
        mine = logits.clone()
        got = wa.process_logits(mine, log_probs=log_probs, out=mine, **kw)
        assert got is mine and torch.equal(got, want)
        # [vocab, rows] logits, transposed; rows off a 16-byte boundary read value by value
        assert torch.equal(wa.process_logits(logits.t().contiguous().t(), log_probs=log_probs, **kw), want)
        off = torch.empty(logits.numel() + 1, device=device)[1:].view_as(logits).copy_(logits)
        check("unaligned", wa.process_logits(off, log_probs=log_probs, **kw), want_logits(logits, log_probs, **kw))
    assert wa.process_logits(logits[:0], log_probs=True).shape == (0, 8200)


def test_long_history_counts_every_token(device):
    """A history as long as the rule allows, of one token: the count is exact."""
    L = 2 ** 20 - 1
    logits = torch.zeros(2, 70, device=device)
    history = torch.full((1, L), 5, dtype=torch.int32, device=device)
    lengths = torch.tensor([L, 1000], dtype=torch.int32, device=device)
    got = wa.process_logits(logits, history=history, lengths=lengths, frequency=torch.ones(2, device=device))
    assert got[0, 5].item() == -L and got[1, 5].item() == -1000 and got.count_nonzero().item() == 2


def test_other_stream_and_graph_replays(device):
    rng = np.random.default_rng(7)
    for R, V in ((1, 20000), (70, 5000)):
        logits, kw = make(rng, R, V, 300, device, biases=20, mask="some")
        step = lambda: (wa.process_logits(logits, log_probs=True, **kw), wa.process_logits(logits, **kw))  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for k in range(3):
            if k:
                logits.copy_(torch.randn(R, V, device=device))
                kw["lengths"].add_(7)
                kw["history"].random_(0, V)
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
            if k == 0:
                assert all(torch.equal(a, b) for a, b in zip(outs, first))


def test_feeds_acceptance(device):
    """A verify round: rows over one history that grows by a draft a row, to greedy and to sampled
    acceptance, as the formula in 64 bits decides it."""
    from oracle import moe as M
    rng = np.random.default_rng(8)
    n, V, L = 3, 5000, 60
    logits = torch.from_numpy(rng.standard_normal((n + 1, V)).astype(np.float32) * 3).to(device)
    drafts = torch.tensor([17, 900, 4321], dtype=torch.int32, device=device)
    history = torch.cat([torch.randint(0, V, (L,), device=device, dtype=torch.int32), drafts])[None]
    lengths = (L + torch.arange(n + 1, device=device)).to(torch.int32)
    kw = dict(history=history, lengths=lengths, prompt_lengths=torch.full((n + 1,), 20, dtype=torch.int32, device=device),
              repetition=torch.full((n + 1,), 1.3, device=device), frequency=torch.full((n + 1,), 0.4, device=device),
              temperature=torch.full((n + 1,), 0.8, device=device))
    logits[0, 17] = 30.0
    logits[1, 900] = 40.0
    want = want_logits(logits, **kw).v
    greedy = wa.mtp_verify_greedy(wa.process_logits(logits, **kw), drafts).tolist()
    assert tuple(greedy) == tuple(M.verify_greedy(drafts.cpu().numpy(), want.astype(np.float32)))
    target = wa.process_logits(logits, log_probs=True, **kw)
    draft = wa.process_logits(torch.randn(n, V, device=device), log_probs=True)
    out = wa.mtp_verify_rejection(target, draft, drafts, torch.rand(n + 1, device=device)).tolist()
    assert 2 <= out[0] <= n and 0 <= out[1] < V    # the first two drafts are all but certain


def test_offsets_past_2_31_elements(device):
    """The last of so many rows that offsets pass 31 bits, at the largest vocabulary."""
    R, V = 520, 4194304
    gen = torch.Generator(device).manual_seed(4)
    logits = torch.randn(R, V, generator=gen, device=device)
    kw = dict(history=torch.randint(0, V, (1, 5000), generator=gen, device=device, dtype=torch.int32),
              mask=torch.randint(-2 ** 31, 2 ** 31 - 1, (1, V // 32), generator=gen, device=device).to(torch.int32))
    rows = dict(repetition=torch.full((R,), 1.5, device=device), temperature=torch.full((R,), 0.7, device=device))
    for log_probs in (False, True):
        out = wa.process_logits(logits, log_probs=log_probs, **kw, **rows)
        want = want_logits(logits[-1:], log_probs=log_probs, **kw, **{k: v[-1:] for k, v in rows.items()})
        check("last row", out[-1:], want)


def test_autograd_sees_an_output_change(device):
    x = torch.randn(2, 50, device=device, requires_grad=True)
    logits = x * 1.0
    loss = (logits * logits).sum()                           # keeps logits for its backward pass
    with torch.no_grad():
        wa.process_logits(logits, out=logits, temperature=torch.full((2,), 0.5, device=device))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
