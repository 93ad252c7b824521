"""Rows of sy_gated_run that are multiplied in plain float32, and the rows beside them."""
import numpy as np
import pytest

import _blocks as R
import _layers as L
from simdyolo_amd import _native as N
from test_gpu_gated import check, rows_of, run, weights

pytestmark = pytest.mark.gpu

# rows, input channels, output channels: few rows, a middling number of tiles, many of long rows, short ones of each layout
FORMS = [(7, 320, 70), (30, 1100, 40), (200, 600, 70), (300, 700, 690), (3000, 1100, 300), (3000, 530, 50), (3000, 250, 2100),
         (200, 320, 200), (13100, 40, 300), (33000, 64, 60), (33000, 200, 70)]


def spread(g, *shape):
    """Magnitudes from 1/2 to 1."""
    return (g.uniform(0.5, 1, shape) * g.choice([-1, 1], shape)).astype(np.float32)


def plain(x, w):
    """No activation, in plain float32: every product that is not 0 and every sum with one rounds once, then the sum with the
    bias and the product of both."""
    sums, x64 = [], x.astype(np.float64)
    terms = (x != 0).sum(1)[:, None]
    for m, b in zip(w[:2], w[2:]):
        m = m.astype(np.float64)
        s = x64 @ m.T + (0 if b is None else b)
        sums.append((s, np.abs(x64) @ np.abs(m).T * 2 * terms * L.UNIT + np.abs(s) * L.UNIT))
    (a, a_off), (u, u_off) = sums
    return a * u, a_off * (np.abs(u) + u_off) + np.abs(a) * u_off + np.abs(a * u) * L.UNIT + L.TINY


def one_channel(g, rows, ic, size):
    """Rows with one element of about `size` (in one of the first 16 even channels), so that no sum hides its products."""
    x = np.zeros((rows, ic), np.float32)
    x[np.arange(rows), 2 * g.integers(0, 8, rows)] = spread(g, rows) * np.float32(size)
    return x


@pytest.mark.parametrize("size", FORMS, ids=str)
def test_tiny_weights_beside_an_uneven_row(hip, size):
    """Output channels whose weights are below 2^-112, rows of about 1e30, some of them with an element far below."""
    rows, ic, oc = size
    g = R.rng(61)
    x, w = spread(g, rows, ic) * np.float32(1e30), [spread(g, oc, ic) * np.float32(1e-30) for _ in range(2)]
    w[0][::3] *= np.float32(1e-5)
    w[1][::2] *= np.float32(1e-5)
    x[3::40, 2] = 1e-3
    check(run(hip, x, w + [None, None], N.ACT_NONE), *L.gated(x, *w, None, None, N.ACT_NONE))


@pytest.mark.parametrize("size", FORMS, ids=str)
def test_plain_rows_meet_whole_weights(hip, size):
    """Even weights with elements down to 2^-30 of their row's largest: a row that is multiplied in plain float32, here for
    an element far below its largest, takes all their bits."""
    rows, ic, oc = size
    g = R.rng(62)
    x, w = one_channel(g, rows, ic, 2.0 ** 29), [spread(g, oc, ic) for _ in range(2)]
    for m in w:
        m[:, ::2] *= np.float32(2.0 ** -29)
    x[:, 3] = np.float32(2.0 ** -60)
    w += [g.standard_normal(oc).astype(np.float32), None]
    check(run(hip, x, w, N.ACT_NONE), *plain(x, w))


@pytest.mark.parametrize("far", [33, 60])
@pytest.mark.parametrize("size", FORMS, ids=str)
def test_uneven_weights_are_multiplied_plainly(hip, size, far):
    rows, ic, oc = size
    g = R.rng(63)
    x, w = one_channel(g, rows, ic, 2.0 ** far), [spread(g, oc, ic) for _ in range(2)]
    for m in w:
        m[:, ::2] *= np.float32(2.0 ** -far)
    w += [None, g.standard_normal(oc).astype(np.float32)]
    check(run(hip, x, w, N.ACT_NONE), *plain(x, w))


@pytest.mark.parametrize("what", [np.nan, np.inf, 1e-20, 1e12])
@pytest.mark.parametrize("size", FORMS, ids=str)
def test_rows_keep_their_bits_beside_any_row(hip, size, what):
    """Rows of a tile in which others are infinite, NaN or uneven."""
    rows, ic, oc = size
    x, w = rows_of(rows, ic, 64), weights(oc, ic, 65)
    layer = hip.gated_create(*w)
    one = run(hip, x, w, layer=layer)
    odd = np.unique(np.r_[2, 5:rows:37, rows - 1])
    x[odd, R.rng(66).integers(0, ic, len(odd))] = what
    two = run(hip, x, w, layer=layer)
    keep = np.setdiff1d(np.arange(rows), odd)
    np.testing.assert_array_equal(one[keep], two[keep])
    if np.isfinite(what):
        check(two[odd], *L.gated(x[odd], *w, N.ACT_SILU))
    else:
        assert not np.isfinite(two[odd]).any()


@pytest.mark.parametrize("ic", [1, 2, 3])
@pytest.mark.parametrize("rows,oc", [(1, 1), (5, 33), (40, 300), (5000, 40), (66000, 20)])
def test_rows_of_fewer_than_four_elements(hip, rows, oc, ic):
    x, w = rows_of(rows, ic, 67), weights(oc, ic, 68)
    check(run(hip, x, w, N.ACT_NONE), *plain(x, w))
