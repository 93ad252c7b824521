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
