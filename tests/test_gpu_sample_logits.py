"""GPU parity of the draw of a token (wm_sample_logits) against the rules in 64 bits, row by row on the host.

Bar: the token is that of the rules. Weights are multiples of 2^-s of the largest (s at least 40, 62 less the
bits of the vocabulary), so a case counts only where no sum that decides is within V 2^-s of its border (TIE): rows
nearer than that may fall either way and are asserted to be one of the two. Log-probabilities are fp32
roundings of a log good to V 2^-s.
"""
import math

import numpy as np
import pytest
import torch

import whallm_amd as wa

pytestmark = pytest.mark.gpu


def rule(l, u, temp=1.0, k=0, p=1.0, m=0.0):
    """One row: (tokens it may be, the one it is, its log-probability, how near a border is)."""
    V = len(l)
    l = l.astype(np.float64) + 0.0
    if np.isnan(l).any() or l.max() == -np.inf:
        return -1, math.nan, 1.0
    if not temp > 0:
        temp, k = 1.0, 1
    order = np.argsort(-l, kind="stable")
    if 0 < k < V:
        order = order[:k]
    with np.errstate(invalid="ignore"):
        d = np.where(l[order] == l[order[0]], 0.0, l[order] - l[order[0]])
        e = np.where(l[order] == -np.inf, 0.0, np.exp(d / temp) if math.isfinite(temp) else np.exp(np.where(np.isfinite(d), 0.0, d)))
    near = 1.0
    n = len(order)
    if p < 1:
        want = max(p, 0.0) * e.sum()
        before = np.cumsum(e) - e
        n = max(1, int((before < want).sum()))
        # ties of weight 0 behind the border do not matter
        near = min(near, float(np.abs(before[1:][e[1:] > 0] - want).min(initial=1.0)))
    if m > 0:
        m = min(m, 1.0)
        q = e[:n]
        near = min(near, float(np.abs(q[q < 1] - m).min(initial=1.0)))
        n = int((q >= m).sum())
    w = np.zeros(V)
    w[order[:n]] = e[:n]
    run = np.cumsum(w)
    want = (min(u, 1 - 2.0 ** -24) if u > 0 else 0.0) * run[-1]
    token = int(np.searchsorted(run, want, side="right"))
    live = run[w > 0]
    near = min(near, float(np.abs(live[:-1] - want).min(initial=1.0)))
    return token, math.log(w[token] / run[-1]), near


def check(device, logits, u, temp=None, k=None, p=None, m=None, least_clear=0.9):
    R, V = logits.shape
    dev = lambda v, t: None if v is None else torch.as_tensor(np.asarray(v), dtype=t).to(device)   # noqa: E731
    tokens, logp = wa.sample_logits(logits.to(device), dev(u, torch.float32), dev(temp, torch.float32), dev(k, torch.int32),
                                    dev(p, torch.float32), dev(m, torch.float32))
    assert tokens.dtype == torch.int32 and logp.dtype == torch.float32 and tokens.shape == logp.shape == (R,)
    tokens, logp = tokens.cpu().numpy(), logp.cpu().numpy()
    host = logits.float().cpu().numpy()
    f32 = lambda v, r, d: d if v is None else float(np.float32(v[r]))   # noqa: E731
    bits = max(V - 1, 0).bit_length()
    unit = V * 2.0 ** -min(62 - bits, 51) + 1e-15 * V
    clear = 0
    for r in range(R):
        args = (f32(temp, r, 1.0), 0 if k is None else int(k[r]), f32(p, r, 1.0), f32(m, r, 0.0))
        token, lp, near = rule(host[r], f32(u, r, 0.0), *args)
        if near <= 2 * unit:
            continue
        clear += 1
        assert tokens[r] == token, (r, tokens[r], token, near, args, u[r])
        if token < 0:
            assert math.isnan(logp[r])
        else:
            assert abs(logp[r] - lp) <= 2.0 ** -23 * abs(lp) + 4 * unit + 1e-12, (r, logp[r], lp)
    assert clear >= least_clear * R, clear
    return tokens


def head(rng, R, V, std=1.5):
    """A few tokens far above a long tail."""
    rank = np.stack([rng.permutation(V) for _ in range(R)])
    return torch.from_numpy((rng.standard_normal((R, V)) * std - 1.6 * np.log1p(rank)).astype(np.float32))


RULES = {"none": {}, "k": dict(k=True), "p": dict(p=True), "m": dict(m=True), "kp": dict(k=True, p=True), "pm": dict(p=True, m=True),
         "kpm": dict(k=True, p=True, m=True)}


def values(rng, R, V, rules):
    return dict(k=rng.integers(0, max(2, min(V, 300)), R) if rules.get("k") else None,
                p=rng.random(R).astype(np.float32) if rules.get("p") else None,
                m=(rng.random(R) * 0.2).astype(np.float32) if rules.get("m") else None)


@pytest.mark.parametrize("rules", list(RULES))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(1, 129280), (5, 129280), (3, 1), (4, 2), (7, 63), (40, 500), (6, 8192), (5, 8193), (9, 20001),
                                 (70, 32000), (2, 300007)])
def test_rules(device, R, V, dtype, rules):
    rng = np.random.default_rng([R, V, len(rules)])
    temp = rng.uniform(0.3, 1.6, R)
    if R > 2:
        temp[1] = 0.0
    logits = head(rng, R, V).to(dtype)
    if R > 3:
        logits[2][torch.from_numpy(rng.random(V) < 0.4)] = -math.inf
    check(device, logits, rng.random(R).astype(np.float32), temp, **values(rng, R, V, RULES[rules]))


@pytest.mark.parametrize("rules", ["k", "p", "kpm"])
def test_flat_rows(device, rules):
    """Nuclei of most of the vocabulary; steep and shallow temperatures."""
    rng = np.random.default_rng(3)
    for std, temps in ((0.01, (1.0, 3.0)), (3.0, (0.05, 20.0)), (30.0, (1.0, 100.0))):
        logits = torch.from_numpy((rng.standard_normal((6, 40000)) * std + 50).astype(np.float32))
        v = values(rng, 6, 40000, RULES[rules])
        if v["k"] is not None:
            v["k"] = rng.integers(1, 39999, 6)
        check(device, logits, rng.random(6).astype(np.float32), rng.uniform(*temps, 6), **v)


def test_ties_go_to_the_lowest_ids(device):
    """Rows of few values: cuts fall inside thousands of equal logits, where the ids decide. Weights are whole
    multiples of a power of two, so that the borders are exact."""
    V = 50000
    rng = np.random.default_rng(4)
    logits = torch.from_numpy(rng.integers(0, 3, (8, V)).astype(np.float32))
    logits[6] = 2.0
    logits[7] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
    k = [1, 100, 20000, 33000, 49999, 2500, 777, 25001]
    # row 1's number lies on a border: of 100 equal weights, 1 each, 50 are half, and the first running sum above 50 is the
    # 51st's. So 7 of the 8 rows are clear, and that one is exact all the same, since 1 is a whole multiple of 2^-s
    tokens = check(device, logits, [0.999, 0.5, 0.9999, 0.7, 0.25, 0.125, 0.99999, 0.99999], k=k, least_clear=7 / 8)
    assert tokens[1] == np.flatnonzero(logits[1].numpy() == 2)[50]
    assert tokens[6] == 776 and tokens[7] == 25000
    same = torch.full((4, V), -7.5)
    # of V equal tokens the first ceil(p V) stay
    tokens, logp = wa.sample_logits(same.to(device), torch.full((4,), 1 - 2.0 ** -24, device=device),
                                    top_p=torch.tensor([0.5, 0.25, 0.75, 0.0], device=device))
    assert tokens.tolist() == [24999, 12499, 37499, 0]
    assert np.allclose(logp.cpu().numpy(), -np.log([25000, 12500, 37500, 1]), atol=1e-6)


def test_greedy_and_degenerate_rules(device):
    rng = np.random.default_rng(6)
    logits = head(rng, 12, 3001)
    logits[3, 17] = logits[3, 2000] = logits[3].max() + 1
    best = logits.argmax(1)
    best[3] = 17
    n = 12
    u = rng.random(n).astype(np.float32)
    for kw in (dict(temp=np.zeros(n)), dict(temp=-np.ones(n)), dict(temp=np.full(n, np.nan)), dict(k=np.ones(n)), dict(p=np.zeros(n)),
               dict(p=np.full(n, -1.0)), dict(temp=np.full(n, 1e-30), k=np.ones(n))):
        assert check(device, logits, u, **kw).tolist() == best.tolist(), kw
    off = check(device, logits, u)
    for kw in (dict(k=np.zeros(n)), dict(k=np.full(n, -5)), dict(k=np.full(n, 3001)), dict(k=np.full(n, 2 ** 31 - 1)), dict(p=np.ones(n)),
               dict(p=np.full(n, 7.0)), dict(p=np.full(n, np.nan)), dict(m=np.zeros(n)), dict(m=np.full(n, -1.0)), dict(m=np.full(n, np.nan))):
        assert check(device, logits, u, **kw).tolist() == off.tolist(), kw
    assert check(device, logits[:3], u[:3], m=np.ones(3)).tolist() == best[:3].tolist()
    check(device, logits, u, temp=np.full(n, np.inf))
    check(device, logits, u, temp=np.full(n, 1e30))


def test_uniforms_at_the_ends(device):
    V = 9001
    logits = torch.full((6, V), -math.inf)
    logits[:, 5], logits[:, 8000] = 1.0, 1.0
    tokens = check(device, logits, [0.0, 1 - 2.0 ** -24, 1.0, 7.0, -3.0, float("nan")], least_clear=0.0)
    assert tokens.tolist() == [5, 8000, 8000, 8000, 5, 5]
    tokens, _ = wa.sample_logits(logits[:2].to(device), torch.tensor([0.5, 0.5 - 2.0 ** -25], device=device))
    assert tokens.tolist() == [8000, 5]     # the first running sum above u times the whole


def test_masked_rows_infinities_and_nan(device):
    V = 20000
    rng = np.random.default_rng(8)
    logits = head(rng, 7, V)
    logits[0] = -math.inf
    logits[1] = -math.inf
    logits[1, 12345] = -3e38
    logits[2, 7] = math.nan
    logits[3, 11] = logits[3, 19999] = math.inf
    logits[4] = torch.finfo(torch.float32).min
    logits[4, 100] = torch.finfo(torch.float32).max
    logits[5] = torch.finfo(torch.float32).min
    u = np.full(7, 0.75, np.float32)
    for kw in ({}, dict(k=np.full(7, 50), p=np.full(7, 0.9), m=np.full(7, 0.01)), dict(p=np.full(7, 0.9))):
        tokens = check(device, logits, u, least_clear=0.5, **kw)
        assert tokens[:4].tolist() == [-1, 12345, -1, 19999] and tokens[4] == 100
    assert (check(device, -torch.full((2, 40), math.inf), [0.1, 0.2], k=[3, 0], p=[0.5, 0.5]) == -1).all()


def test_frequencies(device):
    """20000 draws from one distribution: each token within five deviations of its share."""
    rng = np.random.default_rng(10)
    l = torch.from_numpy(rng.standard_normal(60).astype(np.float32) * 1.5)
    R = 20000
    tokens, _ = wa.sample_logits(l.repeat(R, 1).to(device), torch.rand(R, device=device, generator=torch.Generator(device).manual_seed(1)),
                                 top_k=torch.full((R,), 30, dtype=torch.int32, device=device))
    p = np.exp(l.double().numpy())
    p[np.argsort(-p)[30:]] = 0
    p /= p.sum()
    share = np.bincount(tokens.cpu().numpy(), minlength=60) / R
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / R)).all()


def test_largest_vocabulary_and_odd_rows(device):
    rng = np.random.default_rng(12)
    V = 1 << 22
    check(device, head(rng, 2, V), rng.random(2).astype(np.float32), k=[0, 70], p=[0.95, 1.0])
    wide = head(rng, 5, 4099)
    views = torch.zeros(5, 8198, device=device)[:, 1::2]
    views.copy_(wide)
    u = torch.rand(5, device=device)
    a, b = wa.sample_logits(views, u), wa.sample_logits(wide.to(device), u)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    odd = torch.zeros(5 * 4099 + 1, dtype=torch.bfloat16, device=device)[1:].view(5, 4099)
    odd.copy_(wide)
    a, b = wa.sample_logits(odd, u), wa.sample_logits(wide.bfloat16().to(device), u)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    none = wa.sample_logits(wide[:0].to(device), u[:0])
    assert none[0].shape == none[1].shape == (0,)


def test_repeats_streams_and_graphs(device):
    rng = np.random.default_rng(14)
    R, V = 24, 40000
    logits = head(rng, R, V).to(device)
    u, temp = torch.rand(R, device=device), torch.rand(R, device=device) + 0.3
    k, p = torch.randint(0, 100, (R,), device=device, dtype=torch.int32), torch.rand(R, device=device)
    call = lambda: wa.sample_logits(logits, u, temp, k, p)   # noqa: E731
    eager = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [call() for _ in range(3)]
    here = [call() for _ in range(3)]
    side.synchronize()
    for t, lp in other + here:
        assert torch.equal(t, eager[0]) and torch.equal(lp, eager[1])
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for step in range(3):
        u.uniform_()
        p.uniform_()
        k.random_(0, 3000)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = call()
        for _, (t, lp) in graphs:
            assert torch.equal(t, want[0]) and torch.equal(lp, want[1]), step


def test_past_32_bits(device):
    """The last rows of more than 2^31 logits."""
    R, V = 17000, 129280
    logits = torch.empty(R, V, dtype=torch.bfloat16, device=device)
    logits.fill_(-1.0)
    logits[-3:].normal_(std=3.0)
    u = torch.rand(R, device=device)
    tokens, logp = wa.sample_logits(logits, u)
    t, lp = wa.sample_logits(logits[-3:].clone(), u[-3:].clone())
    assert torch.equal(tokens[-3:], t) and torch.equal(logp[-3:], lp)
    same = (u[:-3].double() * V).floor().int()
    assert (tokens[:-3] - same).abs().max() <= 1


@pytest.mark.parametrize("R,V", [(3, 2048), (3, 2049), (1023, 2050), (1024, 2049), (1025, 2051), (2050, 2060)])
def test_sets_of_rows(device, R, V):
    """Around the vocabularies of one launch a row, and the rows of one set of launches."""
    rng = np.random.default_rng([R, V])
    temp = rng.uniform(0.3, 1.6, R)
    temp[R // 2] = 0.0
    v = values(rng, R, V, RULES["kpm"])
    v["k"][-1], v["p"][0] = 20, 1.0
    check(device, head(rng, R, V), rng.random(R).astype(np.float32), temp, **v)


@pytest.mark.parametrize("V", [2049, 4096, 8200, 70000])
def test_k_around_the_groups(device, V):
    """Cuts at and next to every k at which the way to the candidates changes; all of the largest logits in one group, or one in
    each; more equal logits in the groups than there is room for."""
    rng = np.random.default_rng(V)
    groups = V // 64
    ks = sorted({1, 2, 63, 64, 65, 255, 256, 257, groups * 3 // 4, groups * 3 // 4 + 1, groups, groups + 1, 511, 512, 513, V - 1, V})
    n = len(ks)
    rows = [head(rng, 1, V)[0] for _ in range(4)]
    rows[1][:64] += 40.0
    rows[2][::64] += 40.0
    rows[3] = torch.round(rows[3] * 0.2)                   # few values
    for l in rows:
        u = rng.random(n).astype(np.float32)
        check(device, l.repeat(n, 1), u, k=ks, least_clear=0.8)
        check(device, l.repeat(n, 1), u, k=ks, p=np.full(n, 0.83), m=np.full(n, 0.001), least_clear=0.8)


def test_rows_do_not_depend_on_their_batch(device):
    rng = np.random.default_rng(21)
    R, V = 40, 9000
    logits = head(rng, R, V).to(device)
    u, t = torch.rand(R, device=device), torch.rand(R, device=device) + 0.2
    k = torch.randint(0, 400, (R,), device=device, dtype=torch.int32)
    p = torch.rand(R, device=device)
    tokens, logp = wa.sample_logits(logits, u, t, k, p)
    for r in (0, 7, 39):
        a, b = wa.sample_logits(logits[r:r + 1], u[r:r + 1], t[r:r + 1], k[r:r + 1], p[r:r + 1])
        assert int(a) == int(tokens[r]) and float(b) == float(logp[r])
    many = 300
    a, b = wa.sample_logits(logits[3:4].repeat(many, 1), u[3:4].repeat(many), t[3:4].repeat(many), k[3:4].repeat(many), p[3:4].repeat(many))
    assert bool((a == tokens[3]).all()) and bool((b == logp[3]).all())
