"""sy_group_norm at the ends of float32: differences past its largest value, spreads below its smallest normal one."""
import numpy as np
import pytest

import _blocks as R
import _layers as L
from test_gpu_group_norm import check, run

pytestmark = pytest.mark.gpu

# n, h, w, channels, groups: tokens, one kernel, two kernels, groups that are not of whole quads
SHAPES = [(5, 1, 1, 256, 1), (3, 1, 1, 6, 1), (2, 20, 20, 64, 16), (3, 1, 1, 2000, 1), (1, 90, 70, 96, 8), (1, 45, 75, 27, 3),
          (9, 100, 90, 60, 4)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("low,high", [(-3e38, 3e38), (1e38, 3.3e38), (-2e38, 1e37)])
def test_values_near_the_largest(hip, shape, low, high):
    """One element in 20 at one end of the range, the others about the other: some differences from the mean are past
    float32."""
    n, h, w, c, groups = shape
    g = R.rng(71)
    x = np.where(g.random((n, h * w, c)) < 0.05, high, low) * g.uniform(0.9, 1, (n, h * w, c))
    x[:, 0, 0], x = high, x.astype(np.float32)
    beta = g.standard_normal(c).astype(np.float32)
    got = run(hip, x, h, w, groups, None, beta)
    assert np.isfinite(got).all()
    check(got, *L.group_norm(x, groups, None, beta, 1e-5, 0))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("spread,mean", [(1e-41, 0.0), (1e-38, 3e-38), (1e-33, 0.0), (1e-31, 1e-27)])
def test_spreads_below_float32(hip, shape, spread, mean):
    """No eps: x counts relative to its spread, however small that is."""
    n, h, w, c, groups = shape
    g = R.rng(72)
    x = (g.standard_normal((n, h * w, c)) * spread + mean).astype(np.float32)
    gamma = (1 + 0.3 * g.standard_normal(c)).astype(np.float32)
    got = run(hip, x, h, w, groups, gamma, None, eps=0.0)
    assert np.isfinite(got).all()
    check(got, *L.group_norm(x, groups, gamma, None, 0.0, 0))
