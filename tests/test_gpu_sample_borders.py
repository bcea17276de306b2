"""Draws of which a deciding sum lies on its border (wm_sample_logits): the token is one of those that the border's two sides
give, is no masked one, and its log-probability is that of its side.

Bar: a sum of V weights is off by at most V 2^-s, s = 62 less the bits of the vocabulary (51 at most), and the fp64 reference's
by V 2^-52; where a sum is within twice of that (UNIT) of its border, either side may be taken.
"""
import math

import numpy as np
import pytest
import torch

import whallm_amd as wa
from test_gpu_sample_logits import RULES, head, values

MOST = 8   # sides that are looked at one by one; more of them differ by weights below the unit, and the sums between their ends do


def weights(l, temp):
    """Weights in the order of the logits, and that order."""
    l = l.astype(np.float64) + 0.0
    order = np.argsort(-l, kind="stable")
    with np.errstate(invalid="ignore"):
        d = np.where(l[order] == l[order[0]], 0.0, l[order] - l[order[0]])
        e = np.where(l[order] == -np.inf, 0.0, np.exp(d / temp))
    return e, order


def sides(l, u, temp, k, p, m, unit):
    """The numbers of tokens that may be left, lowest first, with the weights of the longest and their ids."""
    V = len(l)
    if not temp > 0:
        temp, k = 1.0, 1
    e, order = weights(l, temp)
    if 0 < k < V:
        e, order = e[:k], order[:k]
    low = high = len(e)
    if p < 1:
        want, before = max(p, 0.0) * e.sum(), np.cumsum(e) - e
        low, high = max(1, int((before < want - unit).sum())), max(1, int((before < want + unit).sum()))
    if m > 0:
        m = min(m, 1.0)
        near = np.where(e == 1.0, 0.0, 1e-15)   # a weight is good to 2^-51; the largest is 1
        low, high = min(low, int((e >= m + near).sum())), min(high, int((e >= m - near).sum()))
    return low, high, e[:high], order[:high]


def allowed(token, logp, l, u, rules, unit):
    low, high, e, order = sides(l, u, *rules, unit)
    u = min(u, 1 - 2.0 ** -24) if u > 0 else 0.0
    rank = np.flatnonzero(order == token)
    if len(rank) == 0 or not e[rank[0]] > 0:
        return False
    ids = np.argsort(order)
    at = int(np.flatnonzero(order[ids] == token)[0])
    one_by_one = high - low < MOST

    def run(n):
        w = np.where(ids < n, e[ids], 0.0)
        return np.cumsum(w), float(w[at])

    for n in range(low, high + 1) if one_by_one else [None]:
        (a, _), (b, mine) = (run(n), run(n)) if one_by_one else (run(low), run(high))
        if mine > 0 and b[at] > u * a[-1] - unit and a[at] - (mine if one_by_one or rank[0] < low else 0.0) <= u * b[-1] + unit:
            lp = math.log(e[rank[0]] / b[-1])
            if abs(logp - lp) <= 2.0 ** -23 * abs(lp) + 4 * unit + (b[-1] - a[-1]) / a[-1] + 1e-12:
                return True
    return False


def check_all(device, logits, u, temp=None, k=None, p=None, m=None):
    """Every row; returns the tokens and how many rows have more than one side."""
    R, V = logits.shape
    dev = lambda v, t: None if v is None else torch.as_tensor(np.asarray(v), dtype=t).to(device)   # noqa: E731
    tokens, logp = wa.sample_logits(logits.to(device), dev(u, torch.float32), dev(temp, torch.float32), dev(k, torch.int32),
                                    dev(p, torch.float32), dev(m, torch.float32))
    tokens, logp, host = tokens.cpu().numpy(), logp.cpu().numpy(), logits.float().cpu().numpy()
    unit = 2 * (V * 2.0 ** -min(62 - max(V - 1, 0).bit_length(), 51) + V * 2.0 ** -52)
    f32 = lambda v, r, d: d if v is None else float(np.float32(v[r]))   # noqa: E731
    borders = 0
    for r in range(R):
        rules = (f32(temp, r, 1.0), 0 if k is None else int(k[r]), f32(p, r, 1.0), f32(m, r, 0.0))
        if np.isnan(host[r]).any() or host[r].max() == -np.inf:
            assert tokens[r] == -1 and math.isnan(logp[r])
            continue
        assert 0 <= tokens[r] < V and host[r, tokens[r]] > -np.inf, (r, tokens[r])
        assert allowed(int(tokens[r]), float(logp[r]), host[r], f32(u, r, 0.0), rules, unit), (r, tokens[r], logp[r], rules, u[r])
        low, high, _, _ = sides(host[r], 0.0, *rules, unit)
        borders += high > low
    return tokens, borders


def test_the_bar_takes_both_sides_and_nothing_else():
    """Four equal weights, a smaller one and a masked token, without a GPU."""
    l = np.array([0.0, 0.0, -np.inf, 0.0, 0.0, -1.0], np.float32)
    unit, rest = 1e-12, math.exp(-1.0)
    ok = lambda token, logp, u, p: allowed(token, logp, l, u, (1.0, 5, p, 0.0), unit)   # noqa: E731
    quarter, third = math.log(0.25), math.log(1 / 3)
    at = 3 / (4 + rest)                                       # three of the weights are p of the sum
    assert ok(4, quarter, 0.99, 3.5 / (4 + rest)) and not ok(4, third, 0.99, 3.5 / (4 + rest)) and not ok(5, quarter, 0.99, 3.5 / (4 + rest))
    assert ok(3, third, 0.99, at) and ok(4, quarter, 0.99, at) and not ok(3, quarter, 0.99, at) and not ok(4, third, 0.99, at)
    assert not ok(2, quarter, 0.5, at) and not ok(0, third, 0.99, at) and not ok(5, math.log(rest / (4 + rest)), 0.99, at)
    assert ok(1, quarter, 0.5, 3.5 / (4 + rest)) and ok(3, quarter, 0.5, 3.5 / (4 + rest)) and not ok(0, quarter, 0.5, 3.5 / (4 + rest))


@pytest.mark.gpu
@pytest.mark.parametrize("rules", list(RULES))
@pytest.mark.parametrize("R,V", [(3, 1), (40, 500), (6, 8193), (5, 129280), (2, 300007)])
def test_every_row_of_the_rules(device, R, V, rules):
    rng = np.random.default_rng([R, V, len(rules), 1])
    temp = rng.uniform(0.3, 1.6, R)
    logits = head(rng, R, V)
    logits[0][torch.from_numpy(rng.random(V) < 0.4)] = -math.inf
    logits[0, V // 2] = 0.0
    check_all(device, logits, rng.random(R).astype(np.float32), temp, **values(rng, R, V, RULES[rules]))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [600, 2049, 30000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cuts_and_numbers_on_borders(device, V, dtype):
    """Rows of equal logits, p and u whole multiples of 1 / 64: sums lie on their borders where V i / 64 is whole, for some i below 64
    if V is even. The exact side is known: a token stays before which less than p lies, and is drawn where the running sum is above u."""
    n = 64
    logits = torch.full((n, V), -7.5).to(dtype)
    i = np.arange(n)
    p, u = ((i + 1) / n).astype(np.float32), (i[::-1] / n).astype(np.float32)
    tokens, borders = check_all(device, logits, u, p=p)
    assert (borders > 0) == (V % 2 == 0)
    exact = [int(math.floor(float(a) * min(math.ceil(float(b) * V), V))) for a, b in zip(u, p)]
    assert tokens.tolist() == exact
    k = 1 + (i * 9) % (V - 1)
    tokens, _ = check_all(device, logits, u, k=k, p=p)
    kept = [math.ceil(float(b) * int(c)) if b < 1 else int(c) for b, c in zip(p, k)]
    assert tokens.tolist() == [int(math.floor(float(a) * c)) for a, c in zip(u, kept)]


@pytest.mark.gpu
@pytest.mark.parametrize("V", [700, 5000, 40000])
def test_halves_and_masks(device, V):
    """Logits whose weights are powers of two, exactly on the borders of p, of m and of u, with masked tokens among them."""
    rng = np.random.default_rng(V)
    R = 48
    logits = torch.full((R, V), -math.inf)
    for r in range(R):
        ids = rng.choice(V, 12, replace=False)
        logits[r, torch.from_numpy(ids)] = torch.from_numpy((-np.arange(12) * math.log(2.0)).astype(np.float32))
    u = (rng.integers(0, 16, R) / 16).astype(np.float32)
    for rules in (dict(p=rng.integers(1, 16, R) / 16), dict(m=2.0 ** -rng.integers(1, 12, R)), dict(k=rng.integers(1, 12, R)),
                  dict(k=rng.integers(1, 300, R), p=rng.integers(1, 16, R) / 16, m=2.0 ** -rng.integers(1, 12, R))):
        check_all(device, logits, u, **rules)


@pytest.mark.gpu
@pytest.mark.parametrize("rules", ["none", "k", "p", "kpm"])
def test_rows_whose_cut_holds_thousands_of_tokens(device, rules):
    """bf16 logits between 8 and 32, 1/16 to 1/8 apart, so that thousands of tokens share the value at which a cut falls; rows
    that have more candidates than the sort has room for among rows that do not."""
    rng = np.random.default_rng(5)
    for V, mean, std in ((130001, -10.0, 1.5), (60000, 20.0, 0.3), (9000, -25.0, 0.05)):
        logits = torch.from_numpy((rng.standard_normal((6, V)) * std + mean).astype(np.float32)).bfloat16()
        v = values(rng, 6, V, RULES[rules])
        if v["k"] is not None:
            v["k"] = rng.integers(1, V, 6)
        logits[4] = head(rng, 1, V)[0]
        check_all(device, logits, rng.random(6).astype(np.float32), rng.uniform(0.5, 2.0, 6), **v)
