"""Captured prompt attention: one recording replayed with other lengths and other
ranges of rows, eager calls and infinite values between."""
import numpy as np
import pytest

import paged_ref as R
from fuel_amd.hiprt import HipRuntime
from paged_ref import BF16, F16, F32
from test_gpu_paged import Case, say, seed

pytestmark = pytest.mark.gpu


# 16-row tiles whole and cut, 64-row tiles, 128-row tiles, cut 128-row tiles
@pytest.mark.parametrize("act,cache,H,hk,D,past,new", [
    (F16, F16, 4, 2, 128, [60, 0, 7], [9, 30, 20]), (F32, F16, 4, 2, 64, [3000, 20, 700], [3, 1, 2]),
    (BF16, BF16, 32, 2, 128, [0, 30, 0], [170, 60, 70]), (F32, BF16, 20, 20, 64, [0, 70, 0], [330, 260, 130]),
    (F16, F16, 32, 2, 128, [2200, 2000, 0], [150, 100, 40])])
def test_prompts_captured_and_replayed(dev, act, cache, H, hk, D, past, new):
    say("captured prompts", act, cache, H, D, past)
    rng = seed(50, act, H, D)
    c = Case(dev, rng, act, cache, H, hk, D, 16, past, new, pad=8)
    c.max_kv_len = int(max(c.kv))
    full, rows = c.kv.copy(), c.rows
    c.upload()
    page = int(c.pool.table[1, 0])
    clean = c.pool.v.copy()
    rt = HipRuntime()
    stream = rt.stream_create()
    dev.set_stream(stream)
    try:
        graph = rt.capture(stream, c.run)
        for t in range(5):
            # the rows split anew, each sequence with as many as it has positions
            cuts = np.sort(rng.integers(0, rows + 1, 2))
            n = np.minimum(np.diff(np.concatenate([[0], cuts, [rows]])), full)
            c.new = [int(x) for x in n]
            c.kv = np.array([rng.integers(x, k + 1) for x, k in zip(n, full)], np.int32)
            c.start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
            odd = t % 2 == 1 and c.kv[1] > 3
            c.pool.v[:] = clean
            if odd:
                c.pool.v[page, 0, 3, 5] = R.to_bits(np.float32(np.inf), cache)[0]
            c.v_dev.copy_from(c.pool.v)
            c.ints[1].copy_from(c.kv)
            c.ints[2].copy_from(c.start)
            c.out.copy_from(R.to_bits(np.full((rows, c.ldo), 7.0, np.float32), act))
            rt.graph_launch(graph, stream)
            rt.stream_sync(stream)
            c.check(skip=(1,) if odd else ())
            got = c.got()
            if odd:  # sequence 1, key 3 of its first KV head, dim 5
                r0, w = int(c.start[1]), H * D
                mine = got[r0:r0 + c.new[1], :w].reshape(c.new[1], H, D)
                pos = c.kv[1] - c.new[1] + np.arange(c.new[1])
                want = np.zeros(mine.shape, bool)
                want[pos >= 3, :H // hk, 5] = True
                np.testing.assert_array_equal(mine == np.inf, want)
                assert np.isfinite(mine[~want]).all()
            c.out.copy_from(R.to_bits(np.full((rows, c.ldo), 7.0, np.float32), act))
            c.run()  # eager, the same bits
            np.testing.assert_array_equal(c.got(), got)
        rt.graph_destroy(graph)
    finally:
        dev.set_stream(None)
        rt.stream_destroy(stream)
