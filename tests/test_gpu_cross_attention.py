"""sy_cross_attention against float64 (bounds: _layers.cross)."""
import numpy as np
import pytest

import _blocks as R
import _layers as L
from simdyolo_amd import SyError, Tensor
from simdyolo_amd import _native as N
from simdyolo_amd.device import HipContext

pytestmark = pytest.mark.gpu


def tensors(n, tq, tk, heads, kv, kd, hd, seed=0):
    g = R.rng(seed)
    return (1.5 * g.standard_normal((n, tq, heads, kd)).astype(np.float32),
            g.standard_normal((n, tk, kv, kd)).astype(np.float32), g.standard_normal((n, tk, kv, hd)).astype(np.float32))


def config(heads, kv, kd, hd, strides=(0, 0, 0), scale=None):
    return N.CrossConfig(heads, kv, kd, hd, *strides, kd ** -0.5 if scale is None else scale)


def run(hip, q, k, v, lengths=None, mask=None, scale=None, pads=True, qh=1, kh=1, split=None):
    """mask: [n or 1, heads or 1, tq or 1, tk] bytes.  split: whether the states have to be taken in pieces."""
    n, tq, heads, kd = q.shape
    tk, kv, hd = v.shape[1:]
    gap, before = (4, 8) if pads else (0, 0)
    with R.Device(hip) as d:
        vq, sq, _ = d.view(q, qh, tq // qh, gap=gap, before=before)
        vk, sk, _ = d.view(k, kh, tk // kh, gap=2 * gap, pad=before)
        vv, sv, _ = d.view(v, kh, tk // kh, gap=gap, before=gap)
        vo, _, read = d.view(np.full((n, tq, heads, hd), np.nan, np.float32), qh, tq // qh, pad=gap, before=before)
        m = None
        if mask is not None:
            room = 3 if pads else 0  # rows of odd length
            full = np.full(mask.shape[:3] + (tk + room,), 255, np.uint8)
            full[..., :tk] = mask
            step = [int(np.prod(full.shape[i + 1:])) if full.shape[i] > 1 else 0 for i in range(3)]
            m = N.KeyMask(d.put(full), *step)
        hip.profile_enable(True)
        try:
            hip.cross_attention(config(heads, kv, kd, hd, (sq, sk, sv), scale), vq, vk, vv, vo, d.ints(lengths), m)
            hip.flush()
            names = set(hip.profile_read())
        finally:
            hip.profile_enable(False)
        assert names <= {"cross_attention", "cross_join"} and (split is None or ("cross_join" in names) == split)
        return read()


def check(got, exp, bound):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(exp))
    fine = np.isfinite(exp)
    assert (np.abs(got - exp)[fine] <= bound[fine]).all(), (np.abs(got - exp)[fine] / np.maximum(bound[fine], 1e-37)).max()


def scaled(q, k):
    return q.shape[-1] ** -0.5


# n, queries, states, heads, key heads, key dim, head dim, whether the states are taken in pieces
CASES = [
    (1, 1, 1, 1, 1, 4, 4, False), (2, 3, 2, 2, 1, 8, 12, False), (1, 1, 31, 1, 1, 32, 32, False),
    (1, 5, 33, 3, 3, 36, 20, False), (2, 1, 700, 8, 8, 64, 64, True), (1, 1, 3001, 16, 2, 128, 128, True),
    (1, 2, 5000, 3, 1, 80, 100, True), (1, 40, 77, 8, 8, 32, 32, False), (3, 400, 77, 2, 2, 64, 64, False),
    (1, 65, 129, 4, 4, 128, 128, None), (1, 300, 900, 2, 2, 32, 32, True), (2, 33, 65, 6, 2, 16, 128, None),
    (1, 129, 64, 1, 1, 128, 4, None), (1, 64, 96, 5, 1, 4, 64, None), (1, 257, 31, 2, 1, 100, 36, None),
    (8, 200, 40, 8, 8, 32, 64, False), (1, 7, 4097, 1, 1, 68, 32, True),
]


@pytest.mark.parametrize("pads", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_shapes(hip, case, pads):
    n, tq, tk, heads, kv, kd, hd, split = case
    q, k, v = tensors(n, tq, tk, heads, kv, kd, hd)
    check(run(hip, q, k, v, pads=pads, split=split), *L.cross(q, k, v, scaled(q, k)))


@pytest.mark.parametrize("case", CASES, ids=str)
def test_lengths(hip, case):
    """Ragged lengths, none and more than all among them; what stands behind them is NaN."""
    _, tq, tk, heads, kv, kd, hd, _ = case
    n = 5
    tq = min(tq, 70)
    q, k, v = tensors(n, tq, tk, heads, kv, kd, hd, 1)
    lengths = [tk // 2, 0, tk + 9, 1, -3]
    exp, bound = L.cross(q, k, v, scaled(q, k), lengths)
    for b, e in enumerate(lengths):
        k[b, max(e, 0):], v[b, max(e, 0):] = np.nan, np.nan
    got = run(hip, q, k, v, lengths)
    check(got, exp, bound)
    assert (got[1] == 0).all() and (got[4] == 0).all()


@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 1, 1), (1, 4, 1), (1, 1, 50), (2, 1, 50), (2, 4, 50)], ids=str)
@pytest.mark.parametrize("tk,pads", [(1, True), (64, False), (75, True), (900, False), (901, True)])
def test_masks(hip, shape, tk, pads):
    """Masks of every sharing; queries that see nothing, one state, all; any byte but 0 shows."""
    q, k, v = tensors(2, 50, tk, 4, 2, 32, 64, 2)
    g = R.rng(3)
    mask = (g.random(shape + (tk,)) < 0.3).astype(np.uint8) * g.integers(1, 256, shape + (tk,)).astype(np.uint8)
    mask[..., -1, :] = 0
    if shape[2] > 2:
        mask[..., 0, :] = 1
        mask[..., 1, :] = np.arange(tk) == tk - 1
    for lengths in (None, [tk, max(tk - 5, 0)]):
        got = run(hip, q, k, v, lengths, mask, pads=pads)
        check(got, *L.cross(q, k, v, scaled(q, k), lengths, mask))


@pytest.mark.parametrize("tk", [40, 900])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf, np.finfo(np.float32).max, np.finfo(np.float32).min])
def test_hidden_states_hold_anything(hip, tk, what):
    """States that some queries see and others do not: those that do not see them keep their bits' worth."""
    q, k, v = tensors(1, 70, tk, 2, 2, 32, 32, 4)
    mask = np.ones((1, 1, 70, tk), np.uint8)
    mask[:, :, :35, 7::11] = 0
    clean = L.cross(q, k, v, scaled(q, k), None, mask)
    k[:, 7::22], v[:, 18::22] = what, what
    got = run(hip, q, k, v, None, mask)
    check(got[:, :35], clean[0][:, :35], clean[1][:, :35])


# n, queries, states, heads, key heads, key dim, head dim: enough rows for a state's parts to be used many times
MANY = [(8, 1100, 77, 8, 8, 64, 64), (16, 700, 40, 24, 8, 32, 36), (4, 2500, 33, 8, 8, 100, 128), (40, 300, 1, 6, 6, 20, 8),
        (2, 2100, 1100, 8, 8, 64, 64), (1, 3000, 1300, 12, 4, 128, 128), (2, 2000, 500, 8, 4, 32, 20)]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("case", MANY, ids=str)
def test_many_rows(hip, case, masked):
    """Ragged lengths, with and without a mask for each query, states behind them NaN; some of the rows, from every
    image, are compared, and the rest must be as finite."""
    n, tq, tk, heads, kv, kd, hd = case
    q, k, v = tensors(*case, seed=12)
    g = R.rng(13)
    lengths = g.integers(tk // 2, tk + 1, n)
    lengths[0] = tk
    if n > 2:
        lengths[2] = 0
    mask = (g.random((n, 1, tq, tk)) < 0.3).astype(np.uint8) if masked else None
    for b in range(n):
        k[b, lengths[b]:], v[b, lengths[b]:] = np.nan, np.nan
    got = run(hip, q, k, v, lengths, mask)
    assert np.isfinite(got).all()
    rows = np.unique(np.r_[0:3, tq - 3:tq, g.integers(0, tq, 12)])
    exp, bound = L.cross(q[:, rows], k, v, scaled(q, k), lengths, None if mask is None else mask[:, :, rows])
    check(got[:, rows], exp, bound)


@pytest.mark.parametrize("case", MANY[:2] + MANY[4:6], ids=str)
def test_rows_beside_odd_ones(hip, case):
    """A row whose query is infinite, and one whose query is huge, leave every other row's bits alone."""
    q, k, v = tensors(*case, seed=14)
    one = run(hip, q, k, v)
    q[0, 40, 0, 3], q[0, 77, 1] = np.inf, 1e30
    two = run(hip, q, k, v)
    keep = np.ones(one.shape[:3], bool)
    keep[0, 40, 0] = keep[0, 77, 1] = False
    np.testing.assert_array_equal(one[keep], two[keep])
    assert np.isnan(two[0, 40, 0]).all() and np.isfinite(two[0, 77, 1]).all()


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1.0, 30.0])
@pytest.mark.parametrize("tk", [50, 1500])
def test_scales(hip, tk, scale):
    q, k, v = tensors(1, 40, tk, 2, 1, 64, 64, 5)
    check(run(hip, q, k, v, scale=scale), *L.cross(q, k, v, scale))


@pytest.mark.parametrize("tq", [20, 200])
@pytest.mark.parametrize("size", [1e-12, 1e12, 1e36])
def test_values_of_any_size(hip, tq, size):
    """Values that are far from each other, channel by channel and state by state."""
    q, k, v = tensors(1, tq, 120, 2, 2, 32, 64, 6)
    v[..., ::2] *= np.float32(size)
    v[:, 60:] *= np.float32(1e-6)
    check(run(hip, q, k, v), *L.cross(q, k, v, scaled(q, k)))


@pytest.mark.parametrize("tq", [20, 200])
def test_uneven_channels(hip, tq):
    """Channels of queries and keys 2^40 apart, whose products are not."""
    q, k, v = tensors(1, tq, 120, 2, 2, 64, 32, 7)
    q[..., ::2] *= np.float32(2.0 ** 20)
    k[..., ::2] *= np.float32(2.0 ** -20)
    q[..., 1::2] *= np.float32(2.0 ** -20)
    k[..., 1::2] *= np.float32(2.0 ** 20)
    check(run(hip, q, k, v), *L.cross(q, k, v, scaled(q, k)))


@pytest.mark.parametrize("tk", [40, 1000])
def test_visible_non_finite(hip, tk):
    """A visible NaN makes the rows that weigh it NaN; scores past float32 before the scale are formed again."""
    q, k, v = tensors(1, 40, tk, 1, 1, 32, 32, 8)
    v[0, 3, 0, 5] = np.nan
    got = run(hip, q, k, v)
    assert np.isnan(got[..., 5]).all() and np.isfinite(np.delete(got, 5, -1)).all()
    q, k, v = tensors(1, 40, tk, 1, 1, 32, 32, 9)
    q, k, scale = q * np.float32(1e20), k * np.float32(1e19), 1e-39
    scale = float(np.float32(1.2e-38))
    q *= np.float32(0.1)
    check(run(hip, q, k, v, scale=scale), *L.cross(q, k, v, scale))


@pytest.mark.parametrize("qh,kh", [(5, 6), (20, 1), (1, 30)])
def test_maps(hip, qh, kh):
    q, k, v = tensors(2, 100, 90, 2, 2, 32, 32, 10)
    check(run(hip, q, k, v, qh=qh, kh=kh), *L.cross(q, k, v, scaled(q, k)))


def test_keys_and_values_of_one_projection(hip):
    n, tq, tk, heads, kd, hd = 2, 60, 77, 4, 32, 64
    q, k, v = tensors(n, tq, tk, heads, heads, kd, hd, 11)
    both = np.concatenate([k.reshape(n, tk, -1), v.reshape(n, tk, -1)], -1)
    with R.Device(hip) as d:
        p, ld = d.put(both), both.shape[-1]
        vq, _, _ = d.view(q, 1, tq)
        vo, _, read = d.view(np.zeros((n, tq, heads, hd), np.float32), 1, tq)
        hip.cross_attention(config(heads, heads, kd, hd), vq, Tensor(p, n, heads * kd, 1, tk, ld, 0),
                            Tensor(p + 4 * heads * kd, n, heads * hd, 1, tk, ld, 0), vo)
        check(read(), *L.cross(q, k, v, scaled(q, k)))


def test_graphs():
    """Captured calls that share the context's scratch, replayed on new inputs, lengths and masks."""
    with HipContext(0) as ctx, R.Device(ctx) as d:
        calls = []
        for n, tq, tk, heads, kv, dim in ((2, 30, 900, 4, 2, 32), (3, 1, 2000, 8, 8, 64), (1, 200, 60, 2, 2, 32)):
            q, k, v = tensors(n, tq, tk, heads, kv, dim, dim, tq)
            views = [d.view(a, 1, a.shape[1])[0] for a in (q, k, v)]
            vo, _, read = d.view(np.zeros((n, tq, heads, dim), np.float32), 1, tq)
            ln, m = d.ints([tk] * n), d.put(np.ones((n, tq, tk), np.uint8))
            calls.append((lambda views=views, vo=vo, ln=ln, m=N.KeyMask(m, tq * tk, 0, tk), c=config(heads, kv, dim, dim):
                          ctx.cross_attention(c, *views, vo, ln, m), views, ln, m, read, (n, tq, tk, heads, kv, dim, dim)))
        graphs = []
        for c in calls:
            c[0]()
        for c in calls:
            ctx.graph_begin()
            c[0]()
            graphs.append(ctx.graph_end())
        for turn in range(3):
            for i, (call, views, ln, m, read, shape) in enumerate(calls):
                n, tq, tk = shape[:3]
                new = tensors(*shape, 50 + 10 * turn + i)
                lengths = R.rng(turn).integers(0, tk + 1, n).astype(np.int32)
                mask = (R.rng(turn + 9).random((n, tq, tk)) < 0.7).astype(np.uint8)
                for view, a in zip(views, new):
                    ctx.h2d(view.data, a)
                ctx.h2d(ln, lengths)
                ctx.h2d(m, mask)
                calls[i - 1][0]()
                ctx.graph_launch(graphs[i])
                check(read(), *L.cross(*new, shape[5] ** -0.5, lengths, mask[:, None]))


def test_overlaps_are_refused(hip):
    with R.Device(hip) as d:
        vq, _, _ = d.view(np.zeros((1, 6, 2, 32), np.float32), 1, 6)
        vk, _, _ = d.view(np.zeros((1, 9, 2, 32), np.float32), 1, 9)
        vv, _, _ = d.view(np.zeros((1, 9, 2, 32), np.float32), 1, 9)
        for o in (vq, Tensor(vk.data, 1, 64, 1, 6, 64, 0), Tensor(vv.data + 16, 1, 64, 1, 6, 64, 0)):
            with pytest.raises(SyError, match="overlaps"):
                hip.cross_attention(config(2, 2, 32, 32), vq, vk, vv, o)


@pytest.mark.parametrize("kd,hd", [(36, 68), (48, 96), (52, 36), (68, 100), (80, 80), (84, 64), (96, 96), (100, 72), (32, 92), (64, 80)])
@pytest.mark.parametrize("case", [(2, 40, 77, 2, 2), (8, 1300, 33, 8, 8), (1, 900, 1300, 6, 2), (2, 5, 2100, 2, 1), (2, 2, 700, 3, 3)],
                         ids=str)
def test_head_dims(hip, case, kd, hd):
    """Every number of steps of 16 channels and tiles of 32, in each form: some of the rows of large cases are compared."""
    n, tq, tk, heads, kv = case
    q, k, v = tensors(n, tq, tk, heads, kv, kd, hd, 21)
    lengths = [tk - 5 * b for b in range(n)]
    got = run(hip, q, k, v, lengths)
    assert np.isfinite(got).all()
    rows = np.unique(np.r_[0:min(tq, 3), tq - min(tq, 3):tq, R.rng(22).integers(0, tq, 12)])
    exp, bound = L.cross(q[:, rows], k, v, scaled(q, k), lengths)
    check(got[:, rows], exp, bound)
