"""sy_block_attention on operands of far apart sizes, against float64 (bounds: _blocks.attend)."""
import numpy as np
import pytest

import _blocks as R
from test_gpu_block_attention import check, choice, run, tensors

pytestmark = pytest.mark.gpu

FEW, MANY = 1, 700  # queries: pair by pair, as tiles


@pytest.mark.parametrize("tq", [FEW, MANY])
@pytest.mark.parametrize("where", ["own block", "same block", "both"])
@pytest.mark.parametrize("light,heavy", [(1e-10, 1e27), (1e-15, 1e25), (1e-22, 1e24), (1e-33, 1e35)])
def test_far_values_without_weight(hip, tq, where, light, heavy):
    """Keys that weigh nothing (scores 280 below the others, e^-280 = 2^-400 and so nothing in float32 either), with
    values 2^123 to 2^225 above the others': the others' keep their precision, as the products with an exact 0 do."""
    cfg, kd, hd, w = R.shape(2, 1, 1, 32, 3), 32, 64, 128
    q, k, v = tensors(1, tq, w, cfg, kd, hd, 5)
    q[..., 0], k[..., 0] = 40.0, 0.0
    far = {"own block": range(32, 64), "same block": (3, 20), "both": (*range(32, 64), 3, 20)}[where]
    k[:, far, 0, 0] = -40.0
    size = np.full((w, 1, 1), light, np.float32)
    size[list(far)] = heavy
    v *= size
    blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
    blocks[..., 0], blocks[..., 1], blocks[..., 2] = 0, 1, np.maximum(blocks[..., 2], 2)
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    assert (np.abs(exp) < 10 * light).all()
    check(run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == MANY), exp, bound)


@pytest.mark.parametrize("tq", [FEW, MANY])
@pytest.mark.parametrize("selected", [3, 40])
@pytest.mark.parametrize("gap", [30.0, 60.0])
def test_far_values_of_little_weight(hip, tq, selected, gap):
    """Weights down to e^-30 and e^-60 (2^-87) on values that make up for it, fall short of it and outdo it, block by block;
    with 40 blocks the join takes its slots in more than one go."""
    cfg, kd, hd, w = R.shape(2, 1, 1, 16, selected), 32, 36, 16 * 48
    q, k, v = tensors(1, tq, w, cfg, kd, hd, 6)
    q[..., 0], k[..., 0] = 8.0, 0.0
    block = np.arange(w) // 16
    step = (block % 3).astype(np.float32)[:, None, None]  # each a gap below the one before
    k[..., 0] -= step[..., 0] * np.float32(gap / 8 * kd ** 0.5 / 2)
    v *= np.exp(step * np.float32(gap / 2) * (1 + 0.5 * (block % 2)[:, None, None] - 0.25)).astype(np.float32)
    blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    check(run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == MANY), exp, bound)
