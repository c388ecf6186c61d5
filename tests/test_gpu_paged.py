"""The operators over a paged KV cache against their plain 64-bit forms
(paged_ref.py, where the bounds are derived): append bit-exact, attention within
its bound, over types, head layouts, page sizes, ragged lengths from none to
thousands, strides, pools full of NaN outside the sequences' own rows, and the
batch's malformed entries.
"""
import ctypes as C

import numpy as np
import pytest

import fuel_amd as F
import paged_ref as R
from fuel_amd.hiprt import HipRuntime
from paged_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu

TYPES = [(F32, F16), (F16, F16), (F32, BF16), (BF16, BF16)]
NP = {F32: np.float32, F16: np.uint16, BF16: np.uint16}


def say(*a):
    print(*a, flush=True)


def put(dev, a, dt=None):
    return dev.from_numpy(R.to_bits(a, dt) if dt is not None else np.ascontiguousarray(a))


class Case:
    """Sequences with `past` cached tokens and `new` rows each on the device."""

    def __init__(self, dev, rng, act, cache, H, hk, D, ps, past, new, row0=0, tail=0, pad=0, decode=False,
                 width=0, std=1.0, max_kv_len=0):
        self.dev, self.act, self.cache, self.H, self.hk, self.D = dev, act, cache, H, hk, D
        self.kv = np.array([p + n for p, n in zip(past, new)], np.int32)
        self.new = list(new)
        self.start = np.concatenate([[row0], row0 + np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.start[-1]) + tail
        self.pool = R.Pool(rng, self.kv, ps, hk, D, cache, width=width)
        for s, n in enumerate(self.kv):
            self.pool.fill(rng, s, n, std)
        self.ldq, self.ldo = H * D + pad, H * D + 2 * pad
        self.q = (rng.standard_normal((self.rows, self.ldq)) * std).astype(np.float32)
        self.decode = decode
        self.max_kv_len = max_kv_len
        self.scale = float(np.float32(1 / np.sqrt(D)))

    def upload(self):
        dev, p = self.dev, self.pool
        self.k_dev, self.v_dev = dev.from_numpy(p.k), dev.from_numpy(p.v)
        self.kvc = F.PagedKvCache(dev, p.n_pages, p.ps, self.hk, self.D, self.cache, self.k_dev, self.v_dev)
        self.ints = [dev.from_numpy(a) for a in (p.table, self.kv, self.start)]
        self.batch = F.PagedBatch(self.ints[0], self.ints[1], len(self.kv), p.table.shape[1], self.rows,
                                  None if self.decode else self.ints[2], max_kv_len=self.max_kv_len)
        self.q_dev = put(dev, self.q, self.act)
        self.out = put(dev, np.full((self.rows, self.ldo), 7.0), self.act)
        self.work = dev.alloc((max(16, F.paged_attention_workspace(self.kvc, self.batch, self.H)),), np.uint8)
        self.work.copy_from(np.full(self.work.nbytes, 0xff, np.uint8))  # (no initialization needed)

    def run(self, scale=None):
        fn = F.paged_attention_decode if self.decode else F.paged_attention_prefill
        fn(self.kvc, self.batch, self.act, self.H, self.q_dev, self.out, self.scale if scale is None else scale,
           self.work, ldq=self.ldq, ldo=self.ldo)

    def got(self):
        return R.from_bits(self.out.numpy(), self.act)

    def check(self, skip=(), scale=None):
        scale = self.scale if scale is None else scale
        got = self.got()
        w = self.H * self.D
        assert (got[:, w:] == 7.0).all()  # between the rows
        inside = np.zeros(self.rows, bool)
        q = R.from_bits(R.to_bits(self.q, self.act), self.act)
        worst = 0.0
        for s, n in enumerate(self.new):
            r0 = int(self.start[s])
            inside[r0:r0 + n] = True
            if s in skip or n == 0:
                continue
            k, v = self.pool.get(s, int(self.kv[s]))
            pos = int(self.kv[s]) - n + np.arange(n)
            qs = q[r0:r0 + n, :w].reshape(n, self.H, self.D)
            want, A, B, V = R.attend(qs, k, v, pos, scale)
            tol = R.bound(want, A, B, V, max(1, int(self.kv[s])), self.D, self.act, self.cache, not self.decode)
            g = got[r0:r0 + n, :w].reshape(want.shape)
            gone = np.argwhere(~np.isfinite(g))
            assert not len(gone), (s, gone[:3])
            err = np.abs(g - want)
            worst = max(worst, float(np.linalg.norm(err) / max(np.linalg.norm(want), 1e-30)))
            bad = np.argwhere(err > tol)
            assert not len(bad), (s, bad[:3], err.max())
        assert (got[~inside] == 7.0).all()  # rows of no sequence
        say("   relative error", "%.2g" % worst)
        return got


def seed(*a):
    return np.random.default_rng([int(x) for x in a])


# ---- append ----

@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,ps", [(4, 2, 128, 16), (7, 1, 64, 32)])
def test_append(dev, act, cache, H, hk, D, ps):
    """Ragged sequences (one empty, one whose first rows stand before position
    0, one with a length that is none, one with a page outside the pool), rows
    before and behind them, q, k and v as parts of one wide row."""
    say("append", act, cache, H, hk, D, ps)
    rng = seed(1, act, cache, D)
    past, new = [0, 5, 31, -3, 40, 0, 2, 20], [1, 30, 0, 9, 3, 65, 4, 7]
    c = Case(dev, rng, act, cache, H, hk, D, ps, past, new, row0=2, tail=3, width=8)
    c.pool.k[:], c.pool.v[:] = R.NAN[cache], R.NAN[cache]
    width = (H + 2 * hk) * D + 8
    qkv = rng.standard_normal((c.rows, width)).astype(np.float32)
    cos, sin = R.tables(60, D)  # (sequence 5 goes to position 64)
    c.kv[6] = 8 * ps + 1
    c.pool.table[7, 20 // ps] = c.pool.n_pages
    c.upload()
    x = put(dev, qkv, act)
    size = x.nbytes // x.shape[0] // x.shape[1]
    qo = put(dev, np.full((c.rows, H * D + 16), 7.0), act)
    cd, sd = dev.from_numpy(cos), dev.from_numpy(sin)
    F.paged_append(c.kvc, c.batch, act, H, x, x.ptr + H * D * size, x.ptr + (H + hk) * D * size, qo, ldq=width,
                   ldk=width, ldv=width, ldqo=H * D + 16, rope_cos=cd, rope_sin=sd, rope_rows=60)
    xq = R.from_bits(R.to_bits(qkv, act), act)
    want_q = np.full((c.rows, H * D + 16), 7.0, np.float32)
    for s, n in enumerate(new):
        for i in range(n):
            row, pos = int(c.start[s]) + i, int(c.kv[s]) - n + i
            q, k, v = (a.reshape(1, -1, D) for a in np.split(xq[row, :(H + 2 * hk) * D], [H * D, (H + hk) * D]))
            if s == 6 or pos >= 60:
                want_q[row, :H * D] = np.nan
                continue
            if pos < 0:
                want_q[row, :H * D] = 0
                continue
            want_q[row, :H * D] = R.rotate(q, cos[pos:pos + 1], sin[pos:pos + 1]).reshape(-1)
            if 0 <= c.pool.table[s, pos // ps] < c.pool.n_pages:
                c.pool.put(s, np.array([pos]), R.rotate(k, cos[pos:pos + 1], sin[pos:pos + 1]), v)
    got = qo.numpy()
    np.testing.assert_array_equal(np.isnan(R.from_bits(got, act)), np.isnan(want_q))
    ok = ~np.isnan(want_q)
    np.testing.assert_array_equal(got[ok], R.to_bits(want_q, act)[ok])
    np.testing.assert_array_equal(c.k_dev.numpy(), c.pool.k)
    np.testing.assert_array_equal(c.v_dev.numpy(), c.pool.v)


@pytest.mark.parametrize("act,cache", [(F32, F16), (BF16, BF16)])
def test_append_in_place_without_tables_and_without_q(dev, act, cache):
    rng = seed(2, act)
    H, hk, D, ps, n = 6, 3, 64, 16, 300
    c = Case(dev, rng, act, cache, H, hk, D, ps, [0] * n, [1] * n, decode=True)
    c.kv[:] = rng.integers(0, 16, n)
    c.pool.k[:], c.pool.v[:] = R.NAN[cache], R.NAN[cache]
    q, k, v = (rng.standard_normal((n, h * D)).astype(np.float32) for h in (H, hk, hk))
    c.upload()
    qd, kd, vd = (put(dev, a, act) for a in (q, k, v))
    cos, sin = R.tables(16, D)
    k, v = (R.from_bits(R.to_bits(a, act), act).reshape(n, hk, D) for a in (k, v))
    say("append without q and tables")
    F.paged_append(c.kvc, c.batch, act, H, None, kd, vd, None)
    for s in range(n):
        if c.kv[s]:
            c.pool.put(s, np.array([c.kv[s] - 1]), k[s:s + 1], v[s:s + 1])
    np.testing.assert_array_equal(c.k_dev.numpy(), c.pool.k)
    np.testing.assert_array_equal(c.v_dev.numpy(), c.pool.v)
    say("append in place")
    F.paged_append(c.kvc, c.batch, act, H, qd, kd, vd, qd, rope_cos=dev.from_numpy(cos), rope_sin=dev.from_numpy(sin),
                   rope_rows=16)
    q = R.from_bits(R.to_bits(q, act), act).reshape(n, H, D)
    pos = np.maximum(c.kv - 1, 0)
    want = R.rotate(q, cos[pos], sin[pos])
    want[c.kv == 0] = 0
    np.testing.assert_array_equal(qd.numpy(), R.to_bits(want.reshape(n, -1), act))


# ---- decode ----

LAYOUTS = [(4, 4, 128), (8, 2, 128), (16, 2, 64), (7, 1, 128), (20, 1, 64), (40, 2, 128)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D", LAYOUTS)
def test_decode(dev, act, cache, H, hk, D):
    say("decode", act, cache, H, hk, D)
    ps = 16 if H != 16 else 64
    lens = [1, 0, 2, 15, 16, 17, 31, 33, 127, 128, 129, 300, 0, 777]
    c = Case(dev, seed(3, act, cache, H), act, cache, H, hk, D, ps, [n - 1 for n in lens], [1] * len(lens), pad=8,
             decode=True)
    c.upload()
    c.run()
    a = c.check()
    c.run()
    np.testing.assert_array_equal(c.got(), a)  # the same call, the same bits


@pytest.mark.parametrize("act,cache,H,hk,D,lens", [
    (F32, F16, 2, 1, 128, [4097]), (F16, F16, 4, 1, 64, [20000]), (BF16, BF16, 8, 8, 128, [3000, 5, 1500]),
    (F16, F16, 4, 2, 128, [40] * 300), (F32, BF16, 5, 1, 128, [2500, 0, 2500]), (BF16, BF16, 34, 2, 64, [6001])])
def test_decode_long(dev, act, cache, H, hk, D, lens):
    say("decode_long", act, cache, H, hk, D, lens[:3])
    c = Case(dev, seed(4, H, D), act, cache, H, hk, D, 16, [n - 1 for n in lens], [1] * len(lens), decode=True)
    c.upload()
    c.run()
    c.check()


@pytest.mark.parametrize("ps", [16, 32, 128, 1024])
def test_decode_page_sizes_and_scales(dev, ps):
    say("decode page", ps)
    lens = [1, 1023, 1025, 500]
    c = Case(dev, seed(5, ps), F16, F16, 6, 2, 128, ps, [n - 1 for n in lens], [1] * 4, decode=True, width=70)
    c.upload()
    for scale in (c.scale, -0.3, 0.0):
        c.run(scale)
        c.check(scale=scale)


@pytest.mark.parametrize("act,cache", [(F32, F16), (BF16, BF16)])
def test_decode_values_far_apart(dev, act, cache):
    """Scores far above and below each other, q rows of very different size."""
    say("decode far", act, cache)
    rng = seed(6, act)
    c = Case(dev, rng, act, cache, 8, 2, 128, 16, [600, 90], [1, 1], decode=True)
    c.q *= np.repeat(10.0 ** np.array([-30, -4, 0, 1, 1.5, -1, -2, 2]), 128).astype(np.float32)
    c.upload()
    c.run()
    c.check()


def test_decode_many_small_weights(dev):
    """One key far above 30000 equal ones: their weights, 2^-27 each, are 2e-4 of
    the sum and all of dimension 0 of the output."""
    say("decode many small")
    n, D = 30001, 128
    for act, cache in TYPES:
        c = Case(dev, seed(7), act, cache, 1, 1, D, 16, [n - 1], [1], decode=True)
        k = np.zeros((n, 1, D), np.float32)
        v = np.zeros((n, 1, D), np.float32)
        k[17, 0, 0] = 32.0
        v[:, 0, 0] = 1.0
        v[17, 0, 0], v[17, 0, 1] = 0.0, 1.0
        c.pool.put(0, np.arange(n), k, v)
        c.q[:] = 0
        c.q[0, 0] = 27 * np.log(2.0) / 32 / 0.25
        c.upload()
        c.run(0.25)
        c.check(scale=0.25)


def test_malformed_batches_stay_in_bounds(dev):
    """Lengths that are none give NaN, a page outside the pool NaN for the rows
    that see it, ranges that are none leave the output alone."""
    rng = seed(8)
    say("malformed decode")
    c = Case(dev, rng, F16, F16, 4, 2, 128, 16, [40, 40, 40, 40, 40], [1] * 5, decode=True)
    c.kv[1], c.kv[2] = -1, 49
    c.pool.table[3, 1], c.pool.table[4, 2] = -1, c.pool.n_pages
    c.upload()
    c.run()
    got = c.check(skip=(1, 2, 3, 4))
    assert np.isnan(got[1:, :4 * 128]).all()
    say("malformed prefill")
    c = Case(dev, rng, BF16, BF16, 4, 2, 64, 16, [0, 0, 3, 0, 10], [20, 40, 5, 33, 6])
    c.pool.table[1, 1] = c.pool.n_pages          # rows 16 .. of sequence 1 see it
    c.kv[3] = 1 << 20
    c.start[5] = c.rows + 1                      # sequence 4 ends behind the rows
    c.upload()
    c.run()
    got, w = c.got(), 4 * 64
    c.new[4] = 0
    c.check(skip=(1, 3))
    s1, s3 = c.start[1], c.start[3]
    assert np.isnan(got[s1 + 16:s1 + 40, :w]).all() and np.isfinite(got[s1:s1 + 16, :w]).all()
    assert np.isnan(got[s3:s3 + 33, :w]).all()


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("H,hk,D,top", [(20, 20, 128, 100), (40, 20, 64, 250), (3, 3, 128, 31), (70, 2, 64, 30)])
def test_many_short_sequences(dev, act, cache, decode, H, hk, D, top):
    """A wavefront a tile: lengths of none, one and up to `top`, a length that is
    none, a page that is none, sequences of no rows, keys behind a row that are
    no numbers."""
    say("many short", act, cache, decode, H, D, top)
    rng = seed(18, act, cache, H, decode)
    kv = np.concatenate([[0, 1, 2, 16, 17, top, top, 25, 25], rng.integers(1, top + 1, 24)])
    new = [1] * len(kv) if decode else [0, 1, 2, 3, 17, 4, 0, 3, 9] + [int(n) for n in rng.integers(0, 4, 24)]
    c = Case(dev, rng, act, cache, H, hk, D, 16, [int(n) - m for n, m in zip(kv, new)], new, row0=0 if decode else 2,
             tail=0 if decode else 3, pad=8, decode=decode, max_kv_len=top)
    c.kv[7] = top + 1
    c.pool.table[8, 1] = -1  # (positions 16 ..: all rows of sequence 8)
    page, slot = c.pool.table[5, (top - 1) // 16], (top - 1) % 16
    c.pool.k[page, :, slot + 1:], c.pool.v[page, :, slot + 1:] = R.NAN[cache], R.NAN[cache]
    c.upload()
    c.run()
    got = c.check(skip=(7, 8))
    for s in (7, 8):
        assert np.isnan(got[c.start[s]:c.start[s] + new[s], :H * D]).all()
    c.run()
    np.testing.assert_array_equal(c.got(), got)


def test_ranges_over_and_over(dev):
    """Ranges of rows that overlap so often that their work cannot be counted:
    the call ends, and leaves rows outside of them alone."""
    say("overlapping ranges")
    for n, H, D, new, cap in ((6, 8, 64, 100, 4096), (5000, 64, 64, 475, 1 << 20)):
        c = Case(dev, seed(20, n), F16, F16, H, 1, D, 1024, [0], [new], tail=2)
        c.pool.table = np.zeros((n, cap // 1024), np.int32)
        c.kv = np.full(n, cap, np.int32)
        c.start = np.array([0, new] * (n // 2) + [0], np.int32)
        c.upload()
        c.run()
        got = c.got()
        assert (got[new:] == 7.0).all() and (got[:, H * D:] == 7.0).all()


# ---- prefill ----

@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D", LAYOUTS)
def test_prefill(dev, act, cache, H, hk, D):
    say("prefill", act, cache, H, hk, D)
    new = [1, 0, 17, 64, 3, 130, 31, 9]
    past = [0, 0, 0, 5, 100, 0, 33, -4]
    c = Case(dev, seed(9, act, cache, H), act, cache, H, hk, D, 16 if H != 8 else 32, past, new, row0=3, tail=5, pad=8)
    c.upload()
    c.run()
    a = c.check()
    c.run()
    np.testing.assert_array_equal(c.got(), a)


@pytest.mark.parametrize("act,cache,H,hk,D,past,new", [
    (BF16, BF16, 4, 1, 128, [0], [1100]), (F16, F16, 2, 2, 64, [0, 0], [700, 513]),
    (F32, F16, 2, 1, 128, [1000], [70]), (BF16, BF16, 8, 2, 128, [3000, 20, 777], [5, 1, 2]),
    (F32, BF16, 2, 2, 64, [0], [600]), (F16, F16, 3, 1, 128, [129] * 70, [2] * 70)])
def test_prefill_long(dev, act, cache, H, hk, D, past, new):
    say("prefill_long", act, cache, H, hk, D, past[:3], new[:3])
    c = Case(dev, seed(10, H, D), act, cache, H, hk, D, 16, past, new)
    c.upload()
    c.run()
    c.check()
    c.run(-0.2)
    c.check(scale=-0.2)


# batches that take the tiles of 128 rows: many rows times heads; with more than
# 2048 keys and few tiles these are cut
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,ps,past,new", [
    (32, 4, 128, 16, [0, 0, 5, 100, 0, 33, -4], [150, 0, 64, 3, 65, 31, 9]),
    (35, 5, 64, 64, [0, 700, 0, 1], [128, 100, 1, 63]),
    (64, 64, 64, 32, [0, 0], [129, 64]),
    (32, 2, 128, 16, [2100, 0, 2500, 0, -30], [140, 5, 100, 33, 40]),
    (40, 1, 64, 256, [5000], [230])])
def test_prefill_tiles(dev, act, cache, H, hk, D, ps, past, new):
    say("prefill tiles", act, cache, H, hk, D, past, new)
    c = Case(dev, seed(15, act, cache, H), act, cache, H, hk, D, ps, past, new, row0=3, tail=5, pad=8)
    c.upload()
    c.run()
    a = c.check()
    c.run()
    np.testing.assert_array_equal(c.got(), a)
    c.run(-0.2)
    c.check(scale=-0.2)
    c.run(0.0)
    c.check(scale=0.0)


def test_prefill_tiles_of_more_sequences_than_lanes(dev):
    say("prefill tiles, many sequences")
    for past, new in ((0, 5), (2100, 3)):
        n = 150
        c = Case(dev, seed(16, past), BF16, BF16, 64, 1, 64, 16, [past] * n, [new + i % 3 for i in range(n)])
        if past:
            c.kv[:-2] = [new + i % 3 for i in range(n - 2)]  # (most of them short)
        c.upload()
        c.run()
        c.check()


def test_prefill_cut_tiles_of_more_sequences_than_lanes(dev):
    say("cut tiles, many sequences")
    past = [0] * 70
    past[3], past[66] = 5900, 3100
    c = Case(dev, seed(18), F16, F16, 16, 1, 64, 16, past, [40 - i % 5 for i in range(70)])
    c.upload()
    c.run()
    c.check()


def test_prefill_tiles_malformed(dev):
    """As test_malformed_batches_stay_in_bounds, for the tiles of 128 rows."""
    for past in (0, 2300):
        say("malformed tiles", past)
        c = Case(dev, seed(17, past), F16, F16, 40, 2, 64, 16, [past, past, 3, 0, 10], [120, 140, 5, 33, 6])
        c.pool.table[1, (past + 50) // 16] = -7
        page = (past + 50) // 16 * 16 - past         # sequence 1's first row that sees it
        c.kv[3] = -1 << 20
        c.start[5] = c.rows + 1
        c.upload()
        c.run()
        got, w = c.got(), 40 * 64
        c.new[4] = 0
        c.check(skip=(1, 3))
        s1, s3 = c.start[1], c.start[3]
        assert np.isnan(got[s1 + page:s1 + 140, :w]).all() and np.isfinite(got[s1:s1 + page, :w]).all()
        assert np.isnan(got[s3:s3 + 33, :w]).all()


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", [(4, 2, 64, [0, -3], [20, 9]), (32, 8, 128, [0, 30], [300, 70]),
                                             (20, 20, 64, [0, 60], [200, 700])])
def test_prefill_scales(dev, act, cache, H, hk, D, past, new):
    """Scales of 0 (the mean of the values a row sees), below 0 and far from 1,
    infinite and NaN keys and values behind the last row."""
    say("prefill scales", act, cache, H, D)
    c = Case(dev, seed(21, act, cache, H), act, cache, H, hk, D, 16, past, new)
    for s, n in enumerate(c.kv):
        if n % 16:
            page = c.pool.table[s, n // 16]
            c.pool.k[page, :, n % 16:] = c.pool.v[page, :, n % 16:] = R.to_bits(np.float32(np.inf), cache)
            c.pool.k[page, :, n % 16 + 1:] = R.NAN[cache]
    c.upload()
    for scale in (0.0, -0.09, 0.5, -1e-30):
        c.run(scale=scale)
        c.check(scale=float(np.float32(scale)))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D", [(20, 20, 128), (40, 20, 64)])
def test_prefill_more_tiles_than_cus(dev, act, cache, H, hk, D):
    """Whole tiles of 128 rows: prompts and a chunk, a page that is none, a length
    that is none, keys and values that are no numbers from position 150 on."""
    say("prefill many tiles", act, cache, H, D)
    past, new = [0, 0, 70, 0, 3, 0, 5], [200, 1, 130, 60, 250, 0, 190]
    c = Case(dev, seed(19, act, cache, H), act, cache, H, hk, D, 16, past, new, row0=1, tail=4, pad=8)
    c.kv[3] = -5
    c.pool.table[4, 100 // 16] = c.pool.n_pages          # positions 96 ..
    at = 150
    k, v = c.pool.get(0, 200)
    k, v = k.copy(), v.copy()
    k[at::3], v[at::3], v[at + 1::3], k[at + 2::3] = np.nan, np.inf, np.nan, -np.inf
    clean = c.pool.get(0, at)
    c.pool.put(0, np.arange(200), k, v)
    c.upload()
    c.run()
    got, w = c.check(skip=(0, 3, 4)), H * D
    s0, s3, s4 = (int(c.start[s]) for s in (0, 3, 4))
    assert np.isnan(got[s3:s3 + 60, :w]).all()
    assert np.isnan(got[s4 + 93:s4 + 250, :w]).all() and np.isfinite(got[s4:s4 + 93, :w]).all()
    assert not np.isfinite(got[s0 + at:s0 + 200, :w]).any()
    q = R.from_bits(R.to_bits(c.q, act), act)[s0:s0 + at, :w].reshape(at, H, D)
    want, A, B, V = R.attend(q, *clean, np.arange(at), c.scale)
    tol = R.bound(want, A, B, V, at, D, act, cache, True)
    assert (np.abs(got[s0:s0 + at, :w].reshape(want.shape) - want) <= tol).all()


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new,ats", [
    (4, 2, 64, (0, 30), (170, 160), (1, 20, 63, 97, 150)), (4, 2, 128, (0, 30), (170, 160), (1, 20, 63, 97, 150)),
    (32, 2, 128, (0, 30), (170, 160), (1, 20, 97)), (48, 4, 64, (0, 30), (100, 90), (5, 64)),
    (64, 4, 64, (0, 30), (170, 160), (5, 97)),
    (32, 2, 128, (2200, 2000), (150, 140), (2250, 2100)), (40, 2, 64, (2200, 2000), (150, 140), (2230,))])
def test_prefill_keys_a_row_does_not_see_may_hold_anything(dev, act, cache, H, hk, D, past, new, ats):
    """NaN and infinite keys and values from some position on: the rows before
    it as if they were not there, whatever tile they share with the others."""
    say("prefill nan", act, cache, H, D, past)
    for at in ats:
        c = Case(dev, seed(11, act, at), act, cache, H, hk, D, 16, past, new)
        clean = [c.pool.get(s, min(at, int(c.kv[s]))) for s in range(2)]
        for s in range(2):
            n = int(c.kv[s])
            k, v = c.pool.get(s, n)
            k, v = k.copy(), v.copy()
            k[at::3], v[at::3] = np.nan, np.inf
            v[at + 1::3], k[at + 2::3] = np.nan, -np.inf
            c.pool.put(s, np.arange(n), k, v)
        c.upload()
        c.run()
        got, w = c.got(), H * D
        q = R.from_bits(R.to_bits(c.q, act), act)
        for s, p in enumerate(past):
            m = max(0, min(at - p, c.new[s]))
            r0 = int(c.start[s])
            # the rows that see them are no numbers
            assert not np.isfinite(got[r0 + m:r0 + c.new[s], :w]).any()
            if not m:
                continue
            want, A, B, V = R.attend(q[r0:r0 + m, :w].reshape(m, H, D), *clean[s], p + np.arange(m), c.scale)
            tol = R.bound(want, A, B, V, at, D, act, cache, True)
            err = np.abs(got[r0:r0 + m, :w].reshape(want.shape) - want)
            assert (err <= tol).all(), (at, s, np.argwhere(~(err <= tol))[:3])


# ---- the operators together, as a server runs them ----

@pytest.mark.parametrize("act,cache,H,hk,D", [(F32, F16, 4, 2, 128), (BF16, BF16, 8, 1, 64)])
def test_prompts_then_captured_tokens(dev, act, cache, H, hk, D):
    """Prompts in two chunks (append, prefill), then tokens by one captured
    append + decode that is replayed while lengths grow, with eager work between:
    every step's output against attention over all rotated keys so far."""
    rng = seed(12, act)
    say("together", act, cache)
    lens, chunk, steps, ps = [37, 5, 64], [20, 5, 33], 18, 16
    n, width = len(lens), 8
    total = [m + steps for m in lens]
    x = [rng.standard_normal((t, (H + 2 * hk) * D)).astype(np.float32) for t in total]
    cos, sin = R.tables(128, D)
    cd, sd = dev.from_numpy(cos), dev.from_numpy(sin)
    kvc = F.PagedKvCache(dev, 40, ps, hk, D, cache)
    table = rng.permutation(40)[:n * width].reshape(n, width).astype(np.int32)
    td, kv = dev.from_numpy(table), dev.from_numpy(np.zeros(n, np.int32))
    scale = float(np.float32(D ** -0.5))
    refs = []
    for s in range(n):
        r = R.from_bits(R.to_bits(x[s], act), act)
        q, k, v = (a.reshape(total[s], -1, D) for a in np.split(r, [H * D, (H + hk) * D], 1))
        p = np.arange(total[s])
        q = R.from_bits(R.to_bits(R.rotate(q, cos[p], sin[p]), act), act)
        k, v = (R.from_bits(R.to_bits(a, cache), cache) for a in (R.rotate(k, cos[p], sin[p]), v))
        want, A, B, V = R.attend(q, k, v, p, scale)
        refs.append((want, [R.bound(want, A, B, V, total[s], D, act, cache, f) for f in (False, True)]))

    def compare(got, s, lo, hi, prefill):
        want, tol = refs[s]
        err = np.abs(got.reshape(hi - lo, H, D) - want[lo:hi])
        assert (err <= tol[prefill][lo:hi]).all(), (s, lo, prefill)

    size, w = 4 if act == F32 else 2, (H + 2 * hk) * D
    for lo, hi in (([0] * n, chunk), (chunk, lens)):
        new = [b - a for a, b in zip(lo, hi)]
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        rows = int(start[-1])
        xd = put(dev, np.concatenate([x[s][lo[s]:hi[s]] for s in range(n)]), act)
        qd, od = put(dev, np.zeros((rows, H * D)), act), put(dev, np.zeros((rows, H * D)), act)
        kv.copy_from(np.array(hi, np.int32))
        st = dev.from_numpy(start)
        b = F.PagedBatch(td, kv, n, width, rows, st)
        work = dev.alloc((max(16, F.paged_attention_workspace(kvc, b, H)),), np.uint8)
        F.paged_append(kvc, b, act, H, xd, xd.ptr + H * D * size, xd.ptr + (H + hk) * D * size, qd, ldq=w, ldk=w,
                       ldv=w, rope_cos=cd, rope_sin=sd, rope_rows=128)
        F.paged_attention_prefill(kvc, b, act, H, qd, od, scale, work)
        got = R.from_bits(od.numpy(), act)
        for s in range(n):
            compare(got[start[s]:start[s + 1]], s, lo[s], hi[s], True)
    rt = HipRuntime()
    stream = rt.stream_create()
    b = F.PagedBatch(td, kv, n, width)
    work = dev.alloc((max(16, F.paged_attention_workspace(kvc, b, H)),), np.uint8)
    xd = put(dev, np.zeros((n, w)), act)
    qd, od = put(dev, np.zeros((n, H * D)), act), put(dev, np.zeros((n, H * D)), act)
    dev.synchronize()
    dev.set_stream(stream)
    try:
        def step():
            F.paged_append(kvc, b, act, H, xd, xd.ptr + H * D * size, xd.ptr + (H + hk) * D * size, qd, ldq=w, ldk=w,
                           ldv=w, rope_cos=cd, rope_sin=sd, rope_rows=128)
            F.paged_attention_decode(kvc, b, act, H, qd, od, scale, work)

        graph = rt.capture(stream, step)
        for t in range(steps):
            xd.copy_from(R.to_bits(np.stack([x[s][lens[s] + t] for s in range(n)]), act))
            kv.copy_from(np.array([m + t + 1 for m in lens], np.int32))
            rt.graph_launch(graph, stream)
            rt.stream_sync(stream)
            got = R.from_bits(od.numpy(), act)
            for s in range(n):
                compare(got[s], s, lens[s] + t, lens[s] + t + 1, False)
            od.copy_from(np.zeros_like(od.numpy()))
            if t % 3 == 0:  # eager work between the replays, the same values again
                step()
                np.testing.assert_array_equal(R.from_bits(od.numpy(), act), got)
        rt.graph_destroy(graph)
    finally:
        dev.set_stream(None)
        rt.stream_destroy(stream)


def test_pools_past_four_gib(dev):
    """Pages whose byte and element offsets pass 32 bits."""
    say("large pool")
    H, hk, D, ps, dt = 2, 2, 128, 1024, F16
    n_pages = (1 << 33) // (hk * ps * D) + 3  # 2^33 elements, 16 GiB a pool
    rng = seed(13)
    c = Case(dev, rng, F16, dt, H, hk, D, ps, [1500, 900], [3, 2])
    c.upload()
    big = [dev.alloc((n_pages, hk, ps, D), np.uint16) for _ in range(2)]
    page_bytes = hk * ps * D * 2
    new = c.pool.table.copy()
    for i, old in enumerate(np.unique(c.pool.table[c.pool.table < (1 << 30)])):
        to = n_pages - 1 - i if i % 2 == 0 else n_pages // 2 + i
        new[c.pool.table == old] = to
        for src, dst in ((c.pool.k, big[0]), (c.pool.v, big[1])):
            page = np.ascontiguousarray(src[old])
            F._native.check(F.lib().frq_memcpy_htod(dev.handle, C.c_void_p(dst.ptr + int(to) * page_bytes),
                                                    page.ctypes.data_as(C.c_void_p), page.nbytes))
    c.kvc = F.PagedKvCache(dev, n_pages, ps, hk, D, dt, big[0], big[1])
    c.ints[0].copy_from(new)
    c.run()
    c.check()
    one = F.PagedBatch(c.ints[0], c.ints[1], 2, new.shape[1])
    work = dev.alloc((max(16, F.paged_attention_workspace(c.kvc, one, H)),), np.uint8)
    out = put(dev, np.zeros((2, H * D)), F16)
    rows = c.start[1:] - 1
    q = put(dev, c.q[rows], F16)
    F.paged_attention_decode(c.kvc, one, F16, H, q, out, c.scale, work)
    got = R.from_bits(out.numpy(), F16)
    np.testing.assert_allclose(got, c.got()[rows], atol=2 ** -9, rtol=0)
    k = rng.standard_normal((2, hk * D)).astype(np.float32)
    kd = put(dev, k, F16)
    F.paged_append(c.kvc, one, F16, H, None, kd, kd, None)
    for s in range(2):
        p = int(c.kv[s]) - 1
        row = np.empty(D, np.uint16)
        at = ((int(new[s, p // ps]) * hk + 1) * ps + p % ps) * D * 2
        F._native.check(F.lib().frq_memcpy_dtoh(dev.handle, row.ctypes.data_as(C.c_void_p),
                                                C.c_void_p(big[1].ptr + at), row.nbytes))
        np.testing.assert_array_equal(row, R.to_bits(k, F16)[s, D:])


def test_two_handles_at_once(dev):
    """Two handles with their own streams, caches and workspaces, calls enqueued in turn."""
    say("two handles")
    other = F.RocmDevice(0)
    try:
        cs = [Case(d, seed(14, i), BF16, BF16, 8, 2, 128, 16, [2000 + 300 * i, 40], [1, 1], decode=True)
              for i, d in enumerate((dev, other))]
        for c in cs:
            c.upload()
        for _ in range(10):
            for c in cs:
                c.run()
        for c in cs:
            c.check()
        del c, cs
    finally:
        other.close()
