"""Ranges of rows that overlap in the paged attention calls: sequences beside them
have their results, or the call writes nothing."""
import numpy as np
import pytest

import fuel_amd as F
import paged_ref as R
from paged_ref import BF16, F16
from test_gpu_paged import Case, put, say, seed

pytestmark = pytest.mark.gpu

# heads, KV heads, dims, cached, rows / 10: a wavefront a 16-row tile, four a tile, cut 16-row tiles, 64-row tiles,
# 128-row tiles, cut 128-row tiles
KINDS = [(4, 4, 128, 0, 1), (4, 2, 64, 200, 1), (4, 2, 128, 2000, 1), (64, 4, 64, 0, 3), (40, 20, 64, 0, 13),
         (32, 2, 128, 2200, 4)]


@pytest.mark.parametrize("H,hk,D,past,f", KINDS)
def test_overlapping_ranges_within_the_rows(dev, H, hk, D, past, f):
    """Rows 10 .. 20 are in two sequences, as many rows are in none: what is in one
    sequence has its result."""
    say("overlap", H, hk, D, past, f)
    c = Case(dev, seed(40, H, past), BF16, BF16, H, hk, D, 16, [past, 0, past], [20 * f, 0, 30 * f], tail=20 * f)
    c.start = np.array([0, 20 * f, 10 * f, 40 * f], np.int32)
    c.upload()
    c.run()
    got = c.got()
    assert (got[40 * f:] == 7.0).all()
    q = R.from_bits(R.to_bits(c.q, BF16), BF16)
    for s, row0, n, lo, hi in ((0, 0, 20 * f, 0, 10 * f), (2, 10 * f, 30 * f, 20 * f, 40 * f)):
        k, v = c.pool.get(s, past + n)
        want, A, B, V = R.attend(q[row0:row0 + n, :H * D].reshape(n, H, D), k, v, past + np.arange(n), c.scale)
        tol = R.bound(want, A, B, V, past + n, D, BF16, BF16, True)
        at = slice(lo - row0, hi - row0)
        assert (np.abs(got[lo:hi, :H * D].reshape(hi - lo, H, D) - want[at]) <= tol[at]).all()


@pytest.mark.parametrize("H,hk,D,past,f", KINDS)
@pytest.mark.parametrize("n", [5, 90])
def test_more_rows_in_ranges_than_rows(dev, H, hk, D, past, f, n):
    """The same rows in n sequences and others in one: no row is written."""
    say("over and over", H, hk, D, past, f, n)
    c = Case(dev, seed(41, H, past), F16, F16, H, hk, D, 16, [past] * 2, [20 * f, 10 * f], tail=1)
    table = c.pool.table
    c.pool.table = np.concatenate([table[[i % 2]] for i in range(2 * n + 1)])
    c.kv = np.concatenate([c.kv[[0, 1]]] * n + [c.kv[:1]]).astype(np.int32)
    c.start = np.array([0, 20 * f] * n + [0, 20 * f], np.int32)
    c.start[-1] = 30 * f  # (the last sequence: rows 0 .. 30 f)
    c.upload()
    for _ in range(2):
        c.run()
        assert (c.got() == 7.0).all()


@pytest.mark.parametrize("decode", [True, False])
def test_batches_without_pages(dev, decode):
    """max_pages 0 and no table: lengths of 0 give zeros, others are none."""
    say("no pages", decode)
    n, H, D = 5, 4, 128
    c = Case(dev, seed(42), F16, F16, H, 2, D, 16, [0] * n, [1] * n, decode=decode)
    c.kv = np.array([0, 0, 5, 0, -1], np.int32)
    c.upload()
    batch = F.PagedBatch(None, c.ints[1], n, 0, n, None if decode else c.ints[2])
    assert F.paged_attention_workspace(c.kvc, batch, H) == 0
    k, v = (put(dev, np.ones((n, 2 * D), np.float32), F16) for _ in range(2))
    before = c.k_dev.numpy()
    out = put(dev, np.full((n, H * D), 7.0, np.float32), F16)
    F.paged_append(c.kvc, batch, F16, H, c.q_dev, k, v, out)
    want = np.zeros((n, H * D), np.float32)
    want[[2, 4]] = np.nan
    np.testing.assert_array_equal(R.from_bits(out.numpy(), F16), want)
    np.testing.assert_array_equal(c.k_dev.numpy(), before)
    out.copy_from(R.to_bits(np.full((n, H * D), 7.0, np.float32), F16))
    attend = F.paged_attention_decode if decode else F.paged_attention_prefill
    attend(c.kvc, batch, F16, H, c.q_dev, out, c.scale)
    np.testing.assert_array_equal(R.from_bits(out.numpy(), F16), want)
