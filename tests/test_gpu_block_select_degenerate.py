"""sy_block_select on padded queries, empty and constant areas: inputs whose scores are many times alike."""
import numpy as np
import pytest

import _blocks as R
from test_gpu_block_select import FEW, MANY, run_select, some

pytestmark = pytest.mark.gpu


def compare(hip, cfg, q, m, starts=None, lengths=None, every=1, many=True):
    got = run_select(hip, cfg, q, m, 1, m.shape[1] * cfg["block_w"], starts, lengths, many=many)
    for i in range(0, q.shape[1], every):
        at = [s + i for s in (starts or [0] * q.shape[0])]
        np.testing.assert_array_equal(got[:, i:i + 1], R.select(cfg, q[:, i:i + 1], m, at, lengths), err_msg=str(i))


@pytest.mark.parametrize("kv,kd,selected", [(2, 32, 8), (2, 64, 16), (2, 128, 3), (2, 32, 33), (2, 64, 1), (20, 32, 9)])
def test_zero_queries(hip, kv, kd, selected):
    """Padded rows among others of their wave, sums of heads that cancel, and subnormal queries, which are no zeros."""
    cfg, tq, blocks = R.shape(2 * kv, kv, 1, 4, selected, causal=1), 1300, 350
    q = R.rng(1).standard_normal((2, tq, 2 * kv, kd)).astype(np.float32)
    m = R.rng(2).standard_normal((2, blocks, kv, kd)).astype(np.float32)
    q[:, 5::7] = 0
    q[:, 6::7, 1::2] = -q[:, 6::7, ::2]
    q[:, 4::7] *= np.float32(2.0 ** -140)
    q[0, 640:800] = -0.0
    compare(hip, cfg, q, m, (0, 90), (1100, 1390), 11)
    m[0, 40, 0, 3], m[1, 50, 0, 5] = np.nan, np.inf  # 0 times these is NaN
    compare(hip, cfg, q, m, (0, 90), None, 31)


@pytest.mark.parametrize("kv,kd,selected", [(2, 32, 8), (2, 64, 16), (2, 32, 33), (20, 64, 5)])
@pytest.mark.parametrize("causal", [0, 1])
def test_zero_means(hip, kv, kd, selected, causal):
    """All of them zeros, but for the one of the last token; subnormal ones, whose squares are zeros."""
    cfg, tq, blocks = R.shape(2 * kv, kv, 1, 4, selected, causal), 1300, 330
    q = R.rng(1).standard_normal((2, tq, 2 * kv, kd)).astype(np.float32)
    m = np.zeros((2, blocks, kv, kd), np.float32)
    if causal:
        m[:, tq // 4 - 1:] = 3.0
    compare(hip, cfg, q, m, every=29)
    m[:, :90] = (R.rng(3).standard_normal((2, 90, kv, kd)) * 2.0 ** -130).astype(np.float32)
    compare(hip, cfg, q, m, every=29)
    q[:, 29, 0, 2], q[:, 58], q[:, 87, 1, 0] = np.nan, np.inf, np.nan
    compare(hip, cfg, q, m, every=29)


def least_ms(hip, cfg, q, m, h, w, by, bx, kd):
    with R.Device(hip) as d:
        vq, _, _ = d.view(q, h, w)
        vm, _, _ = d.view(m.reshape(m.shape[0], by * bx, 1, -1), by, bx)
        out = d.put(np.zeros((q.shape[0], h * w, cfg["kv_heads"], cfg["selected"]), np.int32))
        least = np.inf
        for _ in range(6):
            hip.timer_start()
            for _ in range(4):
                hip.block_select(R.config(cfg, kd, 4), vq, vm, out)
            least = min(least, hip.timer_stop())
    return least


def test_zeros_cost_no_more(hip):
    """A third of the queries zeros, or all means: no 64-bit scores for them (which took 7 and 20 times as long)."""
    cfg, n, h, w, kd = R.shape(4, 4, 8, 8, 8), 2, 160, 160, 32
    q = R.rng(1).standard_normal((n, h * w, 4, kd)).astype(np.float32)
    m = R.rng(2).standard_normal((n, 400, 4, kd)).astype(np.float32)
    plain = least_ms(hip, cfg, q, m, h, w, 20, 20, kd)
    padded = q.copy()
    padded[:, ::3] = 0
    assert least_ms(hip, cfg, padded, m, h, w, 20, 20, kd) < 2 * plain
    assert least_ms(hip, cfg, q, 0 * m, h, w, 20, 20, kd) < 2 * plain


@pytest.mark.parametrize("kd,selected", [(32, 8), (64, 16), (128, 5), (32, 40)])
@pytest.mark.parametrize("tq", [FEW, MANY])
def test_constant_area(hip, tq, kd, selected):
    """A third of the blocks alike in every bit (a letterbox's bars), and queries that are alike, too: the lower ones."""
    cfg, blocks = R.shape(2, 2, 1, 1, selected), 360
    q = R.rng(1).standard_normal((1, tq, 2, kd)).astype(np.float32)
    m = R.rng(2).standard_normal((1, blocks, 2, kd)).astype(np.float32)
    m[:, 200:300] = m[:, :1]
    m[:, 20:40] = m[:, :1]
    q[:, tq // 2:] = m[:, 0][:, None]
    got = run_select(hip, cfg, q, m, 1, blocks, many=tq == MANY)
    few, got = some(q, got)
    np.testing.assert_array_equal(got, R.select(cfg, few, m))


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 20, 2.0 ** 38])
def test_one_long_mean(hip, size):
    """A mean far longer than the others widens the bound for all: the choice stays."""
    cfg, kd, blocks = R.shape(2, 2, 1, 1, 8), 32, 300
    q = R.rng(1).standard_normal((1, MANY, 2, kd)).astype(np.float32)
    m = R.rng(2).standard_normal((1, blocks, 2, kd)).astype(np.float32)
    m[:, 7] *= np.float32(size)
    got = run_select(hip, cfg, q, m, 1, blocks, many=True)
    few, got = some(q, got)
    np.testing.assert_array_equal(got, R.select(cfg, few, m))


@pytest.mark.parametrize("kd,selected", [(32, 8), (128, 16), (64, 40)])
def test_alike_queries_of_a_row(hip, kd, selected):
    """Causal queries of a few kinds, alike in runs, on means that are nearly all alike: each sees another end."""
    cfg, tq, blocks = R.shape(4, 2, 1, 4, selected, causal=1), 1300, 330
    q = R.rng(1).standard_normal((2, 6, 4, kd)).astype(np.float32)[:, (np.arange(tq) // 9) % 6]
    q[:, ::50] = np.nan
    m = np.repeat(R.rng(2).standard_normal((2, 1, 2, kd)), blocks, 1).astype(np.float32)
    m[:, 100::45] = R.rng(3).standard_normal((2, len(range(100, blocks, 45)), 2, kd))
    compare(hip, cfg, q, m, (0, 13), (1290, 1200), 10)


def test_bars_cost_little_more(hip):
    """Bars above and below the picture, a third of the map, where keys and queries are constants: the queries there, in
    doubt between blocks that are alike, are ranked once for a run of them (one by one 9 times the ordinary call)."""
    cfg, n, h, w, kd = R.shape(4, 4, 8, 8, 8), 2, 160, 160, 32
    q = R.rng(1).standard_normal((n, h, w, 4, kd)).astype(np.float32)
    m = R.rng(2).standard_normal((n, 400, 4, kd)).astype(np.float32)
    plain = least_ms(hip, cfg, q.reshape(n, h * w, 4, kd), m, h, w, 20, 20, kd)
    q[:, :24] = q[:, 136:] = q[:, :1, :1]
    m[:, :60] = m[:, 340:] = q[:, 0, :1]
    assert least_ms(hip, cfg, q.reshape(n, h * w, 4, kd), m, h, w, 20, 20, kd) < 3 * plain
