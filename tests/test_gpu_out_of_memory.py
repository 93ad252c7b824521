"""A call that the device has no memory for fails by itself, and nothing after it."""
import numpy as np
import pytest

import _blocks as R
from simdyolo_amd import SyError, Tensor
from simdyolo_amd import _native as N
from simdyolo_amd.device import HipContext

pytestmark = pytest.mark.gpu


def beyond_memory(ctx):
    """Means of 16 images of 8 heads of 128 channels in 2^24 - 1 blocks, whose operands take 1.1 TB: refused when that is
    asked for, before anything is launched (the addresses stand for nothing)."""
    q = Tensor(1 << 44, 16, 1024, 1, 64, 1024, 0)
    m = Tensor(2 << 44, 16, 1024, 1, (1 << 24) - 1, 1024, 0)
    with pytest.raises(SyError) as e:
        ctx.block_select(R.config(R.shape(8, 8, 1, 1, 4), 128, 4), q, m, 3 << 44)
    assert e.value.code == N.SY_ENOMEM


def attention(ctx, d):
    cfg = R.shape(2, 2, 4, 4, 3)
    q, k, v = (R.rng(i).standard_normal((1, 400, 2, 32)).astype(np.float32) for i in range(3))
    blocks = np.tile(np.array([0, 7, 24], np.int32), (1, 400, 2, 1))
    vq, vk, vv = (d.view(a, 20, 20)[0] for a in (q, k, v))
    vo, _, read = d.view(np.full((1, 400, 2, 32), np.nan, np.float32), 20, 20)
    p = d.put(blocks)
    exp, bound = R.attend(cfg, q, k, v, blocks, 20, 20, 32 ** -0.5)

    def run():
        ctx.block_attention(R.config(cfg, 32, 32), vq, vk, vv, p, vo)

    def check():
        assert (np.abs(read() - exp) <= bound).all()
    return run, check


def test_next_call_works():
    with HipContext(0) as ctx, R.Device(ctx) as d:
        run, check = attention(ctx, d)
        beyond_memory(ctx)
        run()
        check()


def test_graphs_of_before_are_refused():
    """The scratch that a graph was captured with is gone with the call that wanted more of it."""
    with HipContext(0) as ctx, R.Device(ctx) as d:
        run, check = attention(ctx, d)
        run()
        ctx.graph_begin()
        run()
        graph = ctx.graph_end()
        ctx.graph_launch(graph)
        check()
        beyond_memory(ctx)
        with pytest.raises(SyError, match="capture it again"):
            ctx.graph_launch(graph)
        run()
        check()
