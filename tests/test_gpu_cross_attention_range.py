"""sy_cross_attention where scores are far from zero or leave float32, and hidden states of every form.

Queries and keys are small integers times powers of two, so that scores are exact in any order of summation: two of them
are equal, or so far apart that the smaller one's weight is 0.  A row is then the mean of the values of its largest score's
states: `count` equal weights, their sum and the weighted values' (count partial sums each), the quotient and what a
three-part product leaves out are off by (count + 16) halves of a step together."""
import numpy as np
import pytest

import _blocks as R
import _layers as L
from test_gpu_cross_attention import MANY, check, run, scaled, tensors

pytestmark = pytest.mark.gpu

# n, queries, states, heads, key heads, key dim, head dim, whether the states are taken in pieces
FORMS = {
    "few": (2, 1, 300, 8, 8, 32, 32, False), "few, wide": (2, 2, 90, 4, 2, 128, 100, False),
    "few, pieces": (1, 1, 3001, 4, 2, 64, 64, True), "alone": (2, 40, 77, 2, 2, 32, 32, False),
    "pieces": (1, 300, 900, 2, 2, 32, 32, True), "pieces, wide": (1, 300, 2100, 2, 1, 128, 128, True),
    "many": (2, 2100, 1100, 8, 8, 64, 64, None), "short": (8, 1100, 77, 8, 8, 64, 64, False),
}


def means(s, v, seen):
    """The mean of the values of the largest visible scores, and its bound; s [rows, states], v [states, hd]."""
    s = np.where(seen, s, -np.inf)
    best = (s == s.max(1, keepdims=True)) & seen
    count = best.sum(1, keepdims=True)
    share = best / np.maximum(count, 1)
    return share @ v, (share @ np.abs(v)) * (count + 16) * L.UNIT + L.TINY * s.shape[1]


def compare(hip, form, q, k, scale, masked, seed):
    n, tq, tk, heads, kv, kd, hd, split = FORMS[form]
    g = R.rng(seed)
    v = g.standard_normal((n, tk, kv, hd)).astype(np.float32)
    lengths = [tk - 7 * b for b in range(n)]
    mask = (g.random((n, 1, tq, tk)) < 0.6).astype(np.uint8) if masked else None
    if masked:
        mask[:, :, tq // 2] = 0
    for b, e in enumerate(lengths):
        v[b, e:] = np.nan
    got = run(hip, q, k, v, lengths, mask, scale=scale, split=split)
    rows = np.unique(np.r_[0, tq // 2, tq - 1, g.integers(0, tq, 12)])
    for b, e in enumerate(lengths):
        for h in range(heads):
            kg, vg = (a[b, :e, h // (heads // kv)].astype(np.float64) for a in (k, v))
            s = q[b, rows, h].astype(np.float64) @ kg.T
            exp, bound = means(s, vg, np.ones(s.shape, bool) if mask is None else mask[b, 0, rows, :e] != 0)
            check(got[b, rows, h], exp, bound)
    if masked:
        assert (got[:, tq // 2] == 0).all()


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("size", [2e8, 1e9, 1e10, 1e11, 1e12, 1e20, 1e33])
@pytest.mark.parametrize("form", FORMS)
def test_large_scores(hip, form, size, masked):
    """Scaled scores up to about size / 4 to size, which is where rounding the largest alone may leave no weight at all."""
    n, tq, tk, heads, kv, kd, hd, _ = FORMS[form]
    g = R.rng(51)
    q = g.integers(-100, 101, (n, tq, heads, kd)).astype(np.float32)
    k = g.integers(-100, 101, (n, tk, kv, kd)).astype(np.float32)
    q[:, :, :, 0] = 100
    scale, most = 2.0 ** -3, 100.0 * 100 * kd ** 0.5
    q *= np.float32(2.0 ** np.floor(np.log2(size / most / scale)))
    compare(hip, form, q, k, scale, masked, 52)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("scale", [1.0, 0.125])
@pytest.mark.parametrize("most", [95, 124])
@pytest.mark.parametrize("form", FORMS)
def test_scores_at_the_end_of_float32(hip, form, most, scale, sign):
    """Scaled scores of up to 2.5e38 and 3.3e38 (times log2 e past float32), which are sums of one product; with a scale
    below 1 the product itself is past it.  sign -1: the largest scores are -2^121 (and so far from the others)."""
    n, tq, tk, heads, kv, kd, hd, _ = FORMS[form]
    g = R.rng(53)
    q = np.zeros((n, tq, heads, kd), np.float32)
    q[..., 5 % kd] = np.float32(sign * 2.0 ** 121 / scale)
    k = g.integers(-4, 5, (n, tk, kv, kd)).astype(np.float32)
    k[..., 5 % kd] = g.integers(1, most + 1, (n, tk, kv))
    k[:, ::3, :, 5 % kd] = most
    compare(hip, form, q, k, scale, False, 54)


@pytest.mark.parametrize("case", MANY[:2] + MANY[4:6], ids=str)
def test_a_huge_query(hip, case):
    """A row of huge scores beside ordinary ones takes the state of its largest."""
    q, k, v = tensors(*case, seed=14)
    q[0, 77, 1] = 1e30
    got = run(hip, q, k, v)[0, 77, 1]
    g = 1 // (case[3] // case[4])
    k64 = k[0, :, g].astype(np.float64)
    s = k64.sum(1)
    order = np.argsort(s)
    # Far enough apart for any order of summation in float32: weights other than the first's are 0.
    assert s[order[-1]] - s[order[-2]] > 2 * 140 * L.UNIT * np.abs(k64).sum(1).max()
    exp = v[0, order[-1], g].astype(np.float64)
    assert (np.abs(got - exp) <= 17 * L.UNIT * np.abs(exp)).all()


# Forms whose hidden states the masks of few rows, of many rows and of pieces have to keep out
HIDDEN = {name: FORMS[name] for name in ("few", "few, wide", "few, pieces", "pieces, wide", "many", "short")}


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf, np.finfo(np.float32).max, np.finfo(np.float32).min])
@pytest.mark.parametrize("form", HIDDEN)
def test_masked_states_hold_anything(hip, form, what):
    """Keys and values of masked states that no query, or only half of the heads, may see."""
    n, tq, tk, heads, kv, kd, hd, split = HIDDEN[form]
    q, k, v = tensors(n, tq, tk, heads, kv, kd, hd, 55)
    mask = np.ones((1, heads, 1, tk), np.uint8)
    mask[:, :, :, 7::11] = 0
    mask[:, heads // 2:, :, 3::11] = 0
    clean = k.copy(), v.copy()
    k[:, 7::22], v[:, 18::22] = what, what
    k[:, 3::22], v[:, 14::22] = what, what
    got = run(hip, q, k, v, None, mask, split=split)
    rows = np.unique(np.r_[0, tq - 1, R.rng(56).integers(0, tq, 6)])
    exp, bound = L.cross(q[:, rows], *clean, scaled(q, k), None, mask)
    keep = np.s_[:, :, heads // 2:]
    check(got[:, rows][keep], exp[keep], bound[keep])
