"""sy_gated_create and sy_gated_run against float64 (bounds: _layers.gated)."""
import numpy as np
import pytest

import _blocks as R
import _layers as L
from simdyolo_amd import SyError, Tensor
from simdyolo_amd import _native as N
from simdyolo_amd.device import HipContext

pytestmark = pytest.mark.gpu


def weights(oc, ic, seed, bias=True):
    g = R.rng(seed)
    w = [(g.standard_normal((oc, ic)) * ic ** -0.5).astype(np.float32) for _ in range(2)]
    return w + [g.standard_normal(oc).astype(np.float32) * np.float32(0.3) if bias else None for _ in range(2)]


def run(hip, x, w, act=N.ACT_SILU, shape=None, pad=0, before=0, layer=None):
    rows, ic = x.shape
    n, h, width = shape or (1, 1, rows)
    oc = len(w[0])
    if layer is None:
        layer = hip.gated_create(*w, act=act)
    with R.Device(hip) as d:
        vx, _, _ = d.view(x.reshape(n, h * width, 1, ic), h, width, pad=pad, before=before)
        vy, _, read = d.view(np.full((n, h * width, 1, oc), np.nan, np.float32), h, width, pad=before, before=pad)
        hip.gated(layer, vx, vy)
        return read().reshape(rows, oc)


def check(got, exp, bound):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(exp))
    fine = np.isfinite(exp)
    assert (np.abs(got - exp)[fine] <= bound[fine]).all(), (np.abs(got - exp)[fine] / bound[fine]).max()


def rows_of(rows, ic, seed):
    return R.rng(seed).standard_normal((rows, ic)).astype(np.float32)


SIZES = [(1, 1, 1), (1, 64, 32), (2, 15, 33), (3, 16, 31), (5, 257, 100), (16, 100, 65), (31, 300, 40), (32, 512, 96),
         (33, 1, 2), (34, 32, 64), (64, 33, 32), (65, 64, 97), (127, 31, 5), (128, 128, 128), (129, 200, 130),
         (300, 255, 690), (1000, 17, 33), (257, 600, 64), (4100, 48, 1100), (3000, 1100, 300), (9000, 40, 33), (12, 1500, 20),
         (40, 1500, 100)]


@pytest.mark.parametrize("pad,before", [(0, 0), (4, 8), (3, 1)])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(hip, size, pad, before):
    rows, ic, oc = size
    x, w = rows_of(rows, ic, 1), weights(oc, ic, 2, bias=pad == 4)
    check(run(hip, x, w, pad=pad, before=before), *L.gated(x, *w, N.ACT_SILU))


@pytest.mark.parametrize("act", L.ACTS, ids=str)
@pytest.mark.parametrize("rows", [3, 90])
def test_activations(hip, rows, act):
    x, w = rows_of(rows, 64, 3), weights(48, 64, 4)
    w[0] *= np.float32(6)
    check(run(hip, x, w, L.ACTS[act]), *L.gated(x, *w, L.ACTS[act]))


@pytest.mark.parametrize("rows", [7, 200, 3000])
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e25])
def test_rows_of_any_size(hip, rows, size):
    """Rows far apart beside each other, against weights that bring them back."""
    x, w = rows_of(rows, 96, 5), weights(70 if rows < 1000 else 400, 96, 6, bias=False)
    x[::2] *= np.float32(size)
    w[0] *= np.float32(min(1 / size, 1e12))
    check(run(hip, x, w, N.ACT_NONE), *L.gated(x, *w, N.ACT_NONE))


@pytest.mark.parametrize("rows", [7, 200, 3000])
@pytest.mark.parametrize("far", [20, 27, 32, 40, 60])
def test_uneven_channels(hip, rows, far):
    """Channels 2^far below the others of their row, whose weights are as far above the others of theirs; and such rows
    alone, where the large channels' weights are 0."""
    x, w = rows_of(rows, 64, 7), weights(40 if rows < 1000 else 400, 64, 8)
    x[:, ::2] *= np.float32(2.0 ** -far)
    w[0][:, ::2] *= np.float32(2.0 ** far)
    w[1][:, 1::2] = 0
    exp, _ = L.gated(x, *w, N.ACT_NONE)
    near = np.abs(x.astype(np.float64)) @ np.abs(w[0].astype(np.float64)).T, np.abs(x.astype(np.float64)) @ np.abs(
        w[1].astype(np.float64)).T
    a, b = x.astype(np.float64) @ w[0].astype(np.float64).T + w[2], x.astype(np.float64) @ w[1].astype(np.float64).T + w[3]
    # An element down to 2^-32 of its row's largest is off by 2^-50 of that, 2^-18 of itself; so are the weights.
    off = [(m * (64 + 16) * L.UNIT + m * 2.0 ** -17) + np.abs(s) * 2 * L.UNIT for m, s in zip(near, (a, b))]
    bound = off[0] * np.abs(b) + off[1] * (np.abs(a) + off[0]) + np.abs(exp) * L.UNIT + L.TINY
    got = run(hip, x, w, N.ACT_NONE)
    assert (np.abs(got - exp) <= bound).all(), (np.abs(got - exp) / bound).max()


@pytest.mark.parametrize("rows", [7, 200, 3000])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_non_finite(hip, rows, what):
    """An infinity or NaN in a row spoils that row alone, in the weights that channel alone."""
    x, w = rows_of(rows, 64, 9), weights(70 if rows < 1000 else 400, 64, 10)
    exp, bound = L.gated(x, *w, N.ACT_NONE)
    x[5, 3] = what
    w[1][40, 6] = what
    got = run(hip, x, w, N.ACT_NONE)
    assert not np.isfinite(got[5]).any() and not np.isfinite(got[:, 40]).any()
    fine = np.ones(got.shape, bool)
    fine[5], fine[:, 40] = False, False
    assert (np.abs(got - exp) <= bound)[fine].all()


@pytest.mark.parametrize("rows", [4, 100])
def test_zeros(hip, rows):
    x, w = rows_of(rows, 64, 11), weights(33, 64, 12)
    x[1] = 0
    x[:, 16:] = 0
    w[0][3], w[1][4] = 0, 0
    check(run(hip, x, w), *L.gated(x, *w, N.ACT_SILU))
    check(run(hip, x * 0, w), *L.gated(x * 0, *w, N.ACT_SILU))


@pytest.mark.parametrize("shape", [(2, 5, 7), (3, 1, 4)], ids=str)
def test_maps(hip, shape):
    n, h, w = shape
    x, p = rows_of(n * h * w, 40, 13), weights(50, 40, 14)
    check(run(hip, x, p, N.ACT_GELU, shape, pad=4), *L.gated(x, *p, N.ACT_GELU))


@pytest.mark.parametrize("rows,oc", [(200, 64), (3000, 400)])
def test_a_row_does_not_depend_on_the_others(hip, rows, oc):
    """Rows of other sizes beside it, and plain ones in another panel."""
    x, w = rows_of(rows, 96, 15), weights(oc, 96, 16)
    layer = hip.gated_create(*w)
    one = run(hip, x, w, layer=layer)
    x[::2] *= np.float32(1e8)
    x[7, 3] = np.nan
    two = run(hip, x, w, layer=layer)
    keep = np.r_[33:rows:2]
    np.testing.assert_array_equal(one[keep], two[keep])


def test_graphs():
    """Captured calls of two layers that share the context's scratch, replayed on new inputs."""
    with HipContext(0) as ctx, R.Device(ctx) as d:
        calls = []
        for rows, ic, oc in ((200, 64, 96), (700, 33, 40), (5, 100, 64)):
            w = weights(oc, ic, rows)
            layer = ctx.gated_create(*w, act=N.ACT_GELU)
            vx, _, _ = d.view(rows_of(rows, ic, 0).reshape(1, rows, 1, ic), 1, rows)
            vy, _, read = d.view(np.zeros((1, rows, 1, oc), np.float32), 1, rows)
            calls.append((lambda layer=layer, vx=vx, vy=vy: ctx.gated(layer, vx, vy), vx, read, w, rows, ic))
        graphs = []
        for c in calls:
            c[0]()
        for c in calls:
            ctx.graph_begin()
            c[0]()
            with pytest.raises(SyError, match="capture"):
                ctx.gated_create(*weights(4, 4, 0))
            graphs.append(ctx.graph_end())
        for turn in range(3):
            for i, (call, vx, read, w, rows, ic) in enumerate(calls):
                x = rows_of(rows, ic, 20 + 3 * turn + i)
                if turn == 1:
                    x[2, 5] = 1e-30  # a row that is computed plainly, and again not
                ctx.h2d(vx.data, x)
                calls[i - 1][0]()
                ctx.graph_launch(graphs[i])
                check(read().reshape(rows, -1), *L.gated(x, *w, N.ACT_GELU))


def test_refusals(hip):
    layer = hip.gated_create(*weights(8, 12, 0))
    with R.Device(hip) as d:
        vx, _, _ = d.view(np.zeros((1, 6, 1, 12), np.float32), 2, 3, pad=8)
        vy, _, _ = d.view(np.zeros((1, 6, 1, 8), np.float32), 2, 3)
        for x, y, match in [(vy, vy, "views have"), (vx, vx, "views have"), (vx, Tensor(vy.data, 1, 8, 3, 2, 8, 0), "mismatch"),
                            (vx, Tensor(vx.data + 16, 1, 8, 2, 3, vx.ldc, 0), "overlaps"),
                            (Tensor(vx.data + 2, 1, 12, 2, 3, vx.ldc, 0), vy, "aligned")]:
            with pytest.raises(SyError, match=match):
                hip.gated(layer, x, y)
        for handle in (0, layer + 1000):
            with pytest.raises(SyError, match="unknown gated"):
                hip.gated(handle, vx, vy)
        hip.gated(layer, vx, Tensor(vx.data + 48, 1, 8, 2, 3, vx.ldc, 0))
    with pytest.raises(ValueError):
        hip.gated_create(np.zeros((4, 5), np.float32), np.zeros((4, 6), np.float32))


# rows, input channels, output channels: few rows, a middling number of tiles, many of long rows, of short ones
FORMS = [(7, 320, 70), (200, 320, 70), (3000, 320, 400), (3000, 250, 2100), (300, 900, 130), (3000, 530, 400), (13100, 40, 300), (33000, 64, 60), (33000, 200, 70)]


@pytest.mark.parametrize("size", [(33000, 250, 70), (33001, 120, 130), (13000, 250, 300), (3000, 200, 900), (3000, 256, 2100),
                                  (200, 256, 40), (5000, 3, 40), (66000, 2, 20), (40000, 5, 9), (35000, 130, 500), (1300, 511, 200), (700, 258, 690)], ids=str)
@pytest.mark.parametrize("pad", [0, 3])
def test_many_short_rows(hip, size, pad):
    rows, ic, oc = size
    x, w = rows_of(rows, ic, 31), weights(oc, ic, 32)
    check(run(hip, x, w, N.ACT_GELU, pad=pad), *L.gated(x, *w, N.ACT_GELU))


@pytest.mark.parametrize("size", FORMS, ids=str)
@pytest.mark.parametrize("far", [32, 60])
def test_uneven_channels_of_every_form(hip, size, far):
    """As above, with some ordinary rows beside them."""
    rows, ic, oc = size
    x, w = rows_of(rows, ic, 33), weights(oc, ic, 34)
    x[rows // 3:, ::2] *= np.float32(2.0 ** -far)
    w[0][:, ::2] *= np.float32(2.0 ** far)
    w[1][:, 1::2] = 0
    exp, _ = L.gated(x, *w, N.ACT_NONE)
    x64 = x.astype(np.float64)
    near = [np.abs(x64) @ np.abs(m.astype(np.float64)).T for m in w[:2]]
    a, b = (x64 @ w[i].astype(np.float64).T + w[2 + i] for i in range(2))
    off = [(m * (ic + 16) * L.UNIT + m * 2.0 ** -17) + np.abs(s) * 2 * L.UNIT for m, s in zip(near, (a, b))]
    bound = off[0] * np.abs(b) + off[1] * (np.abs(a) + off[0]) + np.abs(exp) * L.UNIT + L.TINY
    got = run(hip, x, w, N.ACT_NONE)
    assert (np.abs(got - exp) <= bound).all(), (np.abs(got - exp) / bound).max()


@pytest.mark.parametrize("size", FORMS, ids=str)
@pytest.mark.parametrize("what", [np.nan, -np.inf])
def test_non_finite_of_every_form(hip, size, what):
    """An infinity or NaN in the first, a middle and the last row, and in a weight of the first and the last channel."""
    rows, ic, oc = size
    x, w = rows_of(rows, ic, 35), weights(oc, ic, 36)
    exp, bound = L.gated(x, *w, N.ACT_NONE)
    bad = [0, rows // 2, rows - 1]
    x[bad[0], 0], x[bad[1], ic // 2], x[bad[2], ic - 1] = what, what, what
    fine = np.ones(exp.shape, bool)
    fine[bad] = False
    got = run(hip, x, w, N.ACT_NONE)
    assert not np.isfinite(got[bad]).any() and (np.abs(got - exp) <= bound)[fine].all()
    w[1][0, ic - 1] = w[0][oc - 1, 0] = what
    fine[:, [0, oc - 1]] = False
    got = run(hip, x, w, N.ACT_NONE)
    assert not np.isfinite(got[:, [0, oc - 1]]).any() and (np.abs(got - exp) <= bound)[fine].all()


def test_graphs_that_share_the_scratch():
    """Captured calls whose rows are split into the context's scratch, of two layers and beside another operator's."""
    with HipContext(0) as ctx, R.Device(ctx) as d:
        calls = []
        for rows, ic, oc in ((3000, 540, 400), (5000, 600, 300)):
            w = weights(oc, ic, rows)
            layer = ctx.gated_create(*w)
            vx, _, _ = d.view(rows_of(rows, ic, 0).reshape(1, rows, 1, ic), 1, rows)
            vy, _, read = d.view(np.zeros((1, rows, 1, oc), np.float32), 1, rows)
            calls.append((lambda layer=layer, vx=vx, vy=vy: ctx.gated(layer, vx, vy), vx, read, w, rows, ic))
        big = d.view(rows_of(9000, 64, 1).reshape(1, 9000, 1, 64), 90, 100)[0]
        norm = lambda: ctx.group_norm(big, big, 2)
        graphs = []
        for c in calls + [(norm,)]:
            c[0]()
        for c in calls + [(norm,)]:
            ctx.graph_begin()
            c[0]()
            graphs.append(ctx.graph_end())
        for turn in range(3):
            for i, (call, vx, read, w, rows, ic) in enumerate(calls):
                x = rows_of(rows, ic, 40 + 3 * turn + i)
                if turn == 1:
                    x[2, 5] = 1e-30
                ctx.h2d(vx.data, x)
                calls[i - 1][0]()
                ctx.graph_launch(graphs[2])
                ctx.graph_launch(graphs[i])
                check(read().reshape(rows, -1), *L.gated(x, *w, N.ACT_SILU))
