"""sy_group_norm against float64 (bounds: _layers.group_norm)."""
import numpy as np
import pytest

import _blocks as R
import _layers as L
from simdyolo_amd import SyError, Tensor
from simdyolo_amd.device import HipContext

pytestmark = pytest.mark.gpu


def run(hip, x, h, w, groups, gamma=None, beta=None, eps=1e-5, act=0, pad=0, before=0, in_place=False):
    n, t, c = x.shape
    with R.Device(hip) as d:
        vx, _, read = d.view(x[:, :, None], h, w, pad=pad, before=before)
        vy = vx
        if not in_place:
            vy, _, read = d.view(np.full((n, t, 1, c), np.nan, np.float32), h, w, pad=before, before=pad)
        g, b = (None if a is None else d.put(a) for a in (gamma, beta))
        hip.group_norm(vx, vy, groups, gamma=g, beta=b, eps=eps, act=act)
        return read()[:, :, 0]


def data(n, t, c, seed, mean=1.0, spread=1.0):
    g = R.rng(seed)
    x = g.standard_normal((n, t, c)) * spread + mean * g.standard_normal((n, 1, c))
    return x.astype(np.float32), (1 + 0.3 * g.standard_normal(c)).astype(np.float32), \
        (0.3 * g.standard_normal(c)).astype(np.float32)


def check(got, exp, bound):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(exp))
    fine = np.isfinite(exp)
    assert (np.abs(got - exp)[fine] <= bound[fine]).all(), (np.abs(got - exp)[fine] / bound[fine]).max()


# n, h, w, channels, groups
SHAPES = [
    (1, 1, 1, 1, 1), (3, 1, 1, 2, 1), (1, 1, 2, 3, 3), (5, 1, 1, 256, 1), (70, 1, 1, 36, 1), (3, 1, 1, 1000, 1),
    (2, 1, 1, 4096, 1), (2, 1, 1, 4097, 1), (2, 1, 1, 9000, 2), (3, 4, 4, 32, 8), (1, 7, 9, 40, 5), (2, 7, 9, 35, 7),
    (1, 20, 20, 256, 32), (2, 20, 20, 512, 32), (2, 13, 17, 108, 12), (1, 45, 75, 27, 3), (1, 40, 40, 64, 1),
    (1, 60, 60, 96, 96), (1, 80, 80, 64, 8), (2, 65, 63, 24, 2), (1, 70, 70, 1040, 2), (1, 100, 100, 10, 1),
    (1, 80, 80, 7, 7), (1, 3, 5, 8200, 1), (1, 1, 3000, 512, 512), (2, 33, 31, 640, 20), (3, 60, 50, 36, 6), (1, 90, 80, 20, 20), (2, 70, 61, 140, 4), (1, 70, 80, 72, 24),
    (1, 64, 70, 1020, 4), (2, 50, 90, 44, 4), (1, 61, 70, 12, 2), (9, 100, 90, 60, 4), (3, 130, 120, 100, 20),
]


@pytest.mark.parametrize("pad,before", [(0, 0), (4, 8), (3, 1)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(hip, shape, pad, before):
    """Dense views, channel slices that can be read four at a time, and ones that cannot."""
    n, h, w, c, groups = shape
    x, gamma, beta = data(n, h * w, c, 1)
    check(run(hip, x, h, w, groups, gamma, beta, pad=pad, before=before), *L.group_norm(x, groups, gamma, beta, 1e-5, 0))


@pytest.mark.parametrize("act", L.ACTS, ids=str)
@pytest.mark.parametrize("shape", [(4, 1, 1, 64, 1), (2, 10, 12, 64, 16), (1, 90, 70, 96, 8)], ids=str)
def test_activations(hip, shape, act):
    n, h, w, c, groups = shape
    x, gamma, beta = data(n, h * w, c, 2)
    gamma = gamma * 6  # far into both tails
    check(run(hip, x, h, w, groups, gamma, beta, act=L.ACTS[act]), *L.group_norm(x, groups, gamma, beta, 1e-5, L.ACTS[act]))


@pytest.mark.parametrize("gamma,beta", [(True, False), (False, True), (False, False)])
def test_without_weights(hip, gamma, beta):
    x, g, b = data(2, 60, 32, 3)
    g, b = g if gamma else None, b if beta else None
    check(run(hip, x, 6, 10, 4, g, b, eps=1e-3), *L.group_norm(x, 4, g, b, 1e-3, 0))


@pytest.mark.parametrize("shape", [(3, 1, 1, 64, 1), (2, 20, 20, 64, 16), (1, 90, 70, 96, 8)], ids=str)
@pytest.mark.parametrize("mean,spread", [(1e4, 1.0), (1e6, 1.0), (0.0, 1e-12), (0.0, 1e15), (1e30, 1e28)])
def test_scales(hip, shape, mean, spread):
    """Means far from zero, spreads whose squares leave float32."""
    n, h, w, c, groups = shape
    x, gamma, beta = data(n, h * w, c, 4, mean, spread)
    check(run(hip, x, h, w, groups, gamma, beta), *L.group_norm(x, groups, gamma, beta, 1e-5, 0))


@pytest.mark.parametrize("shape", [(2, 1, 1, 64, 1), (1, 20, 20, 64, 16), (1, 90, 70, 96, 8)], ids=str)
def test_constant_groups(hip, shape):
    """No variance: the bias alone, exactly."""
    n, h, w, c, groups = shape
    x, gamma, beta = data(n, h * w, c, 5)
    x[:] = np.float32(12345.678)
    np.testing.assert_array_equal(run(hip, x, h, w, groups, gamma, beta), np.broadcast_to(beta, x.shape))


@pytest.mark.parametrize("shape", [(4, 1, 1, 64, 1), (2, 20, 20, 64, 16), (2, 90, 70, 96, 8)], ids=str)
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_non_finite(hip, shape, what):
    """An infinity or a NaN spoils its group alone."""
    n, h, w, c, groups = shape
    x, gamma, beta = data(n, h * w, c, 6)
    x[1, -1, c // 2] = what
    got = run(hip, x, h, w, groups, gamma, beta)
    g = c // 2 // (c // groups)
    bad = np.zeros(x.shape, bool)
    bad[1, :, g * (c // groups):(g + 1) * (c // groups)] = True
    np.testing.assert_array_equal(np.isnan(got), bad)
    x[1, -1, c // 2] = 0
    exp, bound = L.group_norm(x, groups, gamma, beta, 1e-5, 0)
    assert (np.abs(got - exp) <= bound)[~bad].all()


@pytest.mark.parametrize("shape", [(4, 1, 1, 64, 1), (2, 20, 20, 64, 16), (2, 90, 70, 96, 8)], ids=str)
def test_in_place_is_the_same(hip, shape):
    n, h, w, c, groups = shape
    x, gamma, beta = data(n, h * w, c, 7)
    out = run(hip, x, h, w, groups, gamma, beta, act=1)
    np.testing.assert_array_equal(out, run(hip, x, h, w, groups, gamma, beta, act=1, in_place=True, pad=4))


def test_graphs(hip):
    """Two captured calls that share the context's scratch, replayed on new inputs with eager work between."""
    shapes = [(2, 90, 70, 96, 8), (1, 120, 100, 64, 16), (2, 20, 20, 64, 16)]
    with HipContext(0) as ctx, R.Device(ctx) as d:
        calls = []
        for i, (n, h, w, c, groups) in enumerate(shapes):
            x, gamma, beta = data(n, h * w, c, i)
            vx, _, _ = d.view(x[:, :, None], h, w)
            vy, _, read = d.view(np.zeros((n, h * w, 1, c), np.float32), h, w)
            calls.append((lambda vx=vx, vy=vy, g=groups, ga=d.put(gamma), be=d.put(beta):
                          ctx.group_norm(vx, vy, g, ga, be, act=1), vx, read, gamma, beta, (n, h * w, c), groups))
        graphs = []
        for c in calls:
            c[0]()
        for c in calls:
            ctx.graph_begin()
            c[0]()
            graphs.append(ctx.graph_end())
        for turn in range(3):
            for i, (call, vx, read, gamma, beta, shape, groups) in enumerate(calls):
                x = data(*shape, 10 * turn + i)[0]
                ctx.h2d(vx.data, x)
                calls[i - 1][0]()
                ctx.graph_launch(graphs[i])
                check(read()[:, :, 0], *L.group_norm(x, groups, gamma, beta, 1e-5, 1))


def test_overlaps_are_refused(hip):
    with R.Device(hip) as d:
        v, _, _ = d.view(np.zeros((1, 6, 1, 32), np.float32), 2, 3, pad=32)
        for bad in (Tensor(v.data + 16, 1, 32, 2, 3, v.ldc, 0), Tensor(v.data, 1, 32, 2, 3, 32, 0)):
            with pytest.raises(SyError, match="overlaps"):
                hip.group_norm(v, bad, 4)
        with pytest.raises(SyError, match="weights"):
            hip.group_norm(v, v, 4, gamma=v.data)
        hip.group_norm(Tensor(v.data, 1, 32, 2, 3, v.ldc, 0), Tensor(v.data + 128, 1, 32, 2, 3, v.ldc, 0), 4)


def test_more_rows_than_a_grid_of_pixels(hip):
    """Many images of few values."""
    x, gamma, beta = data(70001, 1, 4, 8)
    check(run(hip, x, 1, 1, 1, gamma, beta), *L.group_norm(x, 1, gamma, beta, 1e-5, 0))
