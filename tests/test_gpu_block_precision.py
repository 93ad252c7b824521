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


@pytest.mark.parametrize("tq", [FEW, MANY])
@pytest.mark.parametrize("far", ["q", "k"])
@pytest.mark.parametrize("dims", [(32, 64), (64, 32), (128, 128)], ids=str)
@pytest.mark.parametrize("r", [8, 12, 16, 20, 40])
def test_uneven_channels_of_queries_and_keys(hip, tq, far, dims, r):
    """One channel of the queries 2^r above the others and of the keys as far below, another the other way round: their
    products are of the others' size.  far: the same on one side alone, whose products decide."""
    (kd, hd), w = dims, 96
    cfg = R.shape(2, 2, 1, 16, 4)
    q, k, v = tensors(1, tq, w, cfg, kd, hd, 5)
    up, down = np.float32(2.0 ** r), np.float32(2.0 ** -r)
    q[..., 0] *= up
    k[..., 0] *= down
    if far == "q":
        q[..., kd // 2] *= down
        k[..., kd // 2] *= up
    else:  # what is small on one side meets what is small on the other: nothing is lost with it
        k[..., kd // 2] *= down
    blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    check(run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == MANY), exp, bound)


@pytest.mark.parametrize("tq", [FEW, MANY])
@pytest.mark.parametrize("keys", ["alike", "of many sizes"])
@pytest.mark.parametrize("r", [8, 16, 20, 24, 28, 32, 60])
def test_uneven_channels_of_values(hip, tq, keys, r):
    """Channels of the values 2^r below the others, in every key: as precise as the others."""
    cfg, kd, hd, w = R.shape(4, 2, 1, 48, 3, causal=1), 32, 64, 200
    q, k, v = tensors(2, tq, w, cfg, kd, hd, 5)
    v[..., 3] *= np.float32(2.0 ** -r)
    v[..., 40:48] *= np.float32(2.0 ** -(r // 2))
    v[..., 63] = 0
    if keys == "of many sizes":
        v *= np.exp2(5.0 * (np.arange(w) % 7)).astype(np.float32)[:, None, None]
    blocks = choice(2, tq, cfg, 1, w, 8, 0.0)
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    check(run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == MANY), exp, bound)


@pytest.mark.parametrize("tq", [FEW, MANY])
@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 11, 2.0 ** 14])
def test_large_scores(hip, tq, size):
    """Queries and keys whose products come to 2^16 and more, on both sides of where the matrix cores are left, cancelled
    to ordinary scores by a second channel; garbage behind the last token, far above the keys, that no row sees."""
    cfg, kd, hd, w = R.shape(2, 1, 1, 32, 3, causal=1), 16, 16, 1000
    q, k, v = tensors(1, tq, w, cfg, kd, hd, 5)
    q[..., 0] = q[..., 1] = k[..., 0] = np.float32(size)
    k[..., 1] = np.float32(-size)
    blocks = choice(1, tq, cfg, 1, w, 8, 0.0)
    blocks[..., 0] = 0
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5)
    k[:, max(tq, 32):] *= np.float32(2.0 ** 60)
    check(run(hip, cfg, q, k, v, blocks, 1, w, sort=tq == MANY), exp, bound)


@pytest.mark.parametrize("dims", [(32, 20), (64, 64), (128, 128)], ids=str)
@pytest.mark.parametrize("group", [1, 3])
def test_channels_of_values_with_powers_of_their_own(hip, dims, group):
    """Channels from 2^-21 to 2^-115 of the others, one that is so in the keys of one block alone, one of zeros, one with
    an infinity in a key that some rows see."""
    (kd, hd), w = dims, 300
    cfg = R.shape(2 * group, 2, 1, 70, 3, causal=1)
    q, k, v = tensors(2, 500, w, cfg, kd, hd, 5)
    for c, r in enumerate((21, 30, 44, 60, 76, 92, 103, 115)):
        v[..., c] *= np.float32(2.0 ** -r)
    v[:, 70:140, :, 8] *= np.float32(2.0 ** -50)
    v[..., 9] = 0
    blocks = choice(2, 500, cfg, 1, w, 8, 0.0)
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5, (0, -40))
    check(run(hip, cfg, q, k, v, blocks, 1, w, starts=(0, -40), sort=True), exp, bound + 2.0 ** -140)
    v[0, 75, 1, 3] = np.inf
    with np.errstate(invalid="ignore"):
        exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5, (0, -40))
    got = run(hip, cfg, q, k, v, blocks, 1, w, starts=(0, -40), sort=True)
    np.testing.assert_array_equal(np.isfinite(got), np.isfinite(exp))
    fine = np.isfinite(exp)
    assert (np.abs(got[fine] - exp[fine]) <= bound[fine] + 2.0 ** -140).all()


def test_a_dead_channel_costs_little_more(hip):
    """A channel of the values at 1e-12 of the others in every key: 1.7 times the ordinary call, not plain float32 (170
    times)."""
    cfg, h, w, kd, hd = R.shape(2, 2, 8, 8, 8), 120, 120, 32, 64
    q, k, v = tensors(1, h * w, h * w, cfg, kd, hd, 5)
    blocks = R.rng(3).integers(0, 225, (1, h * w, 2, 8)).astype(np.int32)
    took = []
    for size in (1.0, 1e-12):
        v[..., 7] *= np.float32(size)
        with R.Device(hip) as d:
            vq, vk, vv = (d.view(a, h, w)[0] for a in (q, k, v))
            vo, _, read = d.view(np.full((1, h * w, 2, hd), np.nan, np.float32), h, w)
            p, cf, least = d.put(blocks), R.config(cfg, kd, hd), np.inf
            for _ in range(5):
                hip.timer_start()
                hip.block_attention(cf, vq, vk, vv, p, vo)
                least = min(least, hip.timer_stop())
            got = read()
        took.append(least)
        keep = R.rng(4).integers(0, h * w, 100)
        check(got[:, keep], *R.attend(cfg, q[:, keep], k, v, blocks[:, keep], h, w, kd ** -0.5))
    assert took[1] < 5 * took[0]


@pytest.mark.parametrize("hd", [4, 12, 64])
@pytest.mark.parametrize("bw", [3, 64])
def test_uneven_channels_and_uneven_keys(hip, hd, bw):
    """A channel 2^-41 of the others, which a few keys have hardly anything of: these keys' rows are scaled up, and the small
    channel of the other keys is as precise as without them."""
    cfg, kd, w = R.shape(2, 1, 1, bw, 9, causal=1), 20, 8 * bw + 2
    q, k, v = tensors(2, 700, w, cfg, kd, hd, 5)
    v[..., 1] *= np.float32(2.0 ** -41)
    v[..., [0, *range(2, hd)]] *= np.where(np.arange(w) % 7 == 3, np.float32(2.0 ** -16), np.float32(1))[:, None, None]
    blocks = choice(2, 700, cfg, 1, w, 8, 0.0)
    exp, bound = R.attend(cfg, q, k, v, blocks, 1, w, kd ** -0.5, (0, 30))
    check(run(hip, cfg, q, k, v, blocks, 1, w, starts=(0, 30), sort=True), exp, bound)
