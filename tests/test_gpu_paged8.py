"""The operators over an 8-bit paged KV cache against their plain 64-bit forms
(paged8_ref.py): append bit-exact in codes and scales, attention within its bound,
over types, head layouts, page sizes, ragged lengths, strides, pools of NaN codes and
scales outside the sequences' own rows, and the batch's malformed entries.
"""
import ctypes as C

import numpy as np
import pytest

import fuel_amd as F
import paged8_ref as P
import paged_ref as R
from fuel_amd.hiprt import HipRuntime
from paged_ref import BF16, F16, F32

pytestmark = pytest.mark.gpu

TYPES = [F32, F16, BF16]


def say(*a):
    print(*a, flush=True)


def seed(*a):
    return np.random.default_rng([int(x) for x in a])


def put(dev, a, dt=None):
    return dev.from_numpy(R.to_bits(a, dt) if dt is not None else np.ascontiguousarray(a))


class Case:
    """Sequences with `past` cached tokens and `new` rows each on the device."""

    def __init__(self, dev, rng, act, H, hk, D, ps, past, new, row0=0, tail=0, pad=0, decode=False, width=0, std=1.0,
                 max_kv_len=0, fill=True):
        self.dev, self.act, self.H, self.hk, self.D = dev, act, H, hk, D
        self.kv = np.array([p + n for p, n in zip(past, new)], np.int32)
        self.new = list(new)
        self.start = np.concatenate([[row0], row0 + np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.start[-1]) + tail
        self.pool = P.Pool(rng, self.kv, ps, hk, D, width=width)
        for s, n in enumerate(self.kv):
            if fill:
                self.pool.fill(rng, s, n, std)
        self.ldq, self.ldo = H * D + pad, H * D + 2 * pad
        self.q = (rng.standard_normal((self.rows, self.ldq)) * std).astype(np.float32)
        self.decode, self.max_kv_len = decode, max_kv_len
        self.scale = float(np.float32(1 / np.sqrt(D)))

    def upload(self):
        dev, p = self.dev, self.pool
        self.cells = [dev.from_numpy(a) for a in (p.code[0], p.code[1], p.scale[0], p.scale[1])]
        self.kvc = F.PagedKvCache8(dev, p.n_pages, p.ps, self.hk, self.D, *self.cells)
        self.ints = [dev.from_numpy(a) for a in (p.table, self.kv, self.start)]
        self.batch = F.PagedBatch(self.ints[0], self.ints[1], len(self.kv), p.table.shape[1], self.rows,
                                  None if self.decode else self.ints[2], max_kv_len=self.max_kv_len)
        self.q_dev = put(dev, self.q, self.act)
        self.out = put(dev, np.full((self.rows, self.ldo), 7.0), self.act)
        self.work = dev.alloc((max(16, F.paged_attention_workspace(self.kvc, self.batch, self.H)),), np.uint8)
        self.work.copy_from(np.full(self.work.nbytes, 0xff, np.uint8))  # (no initialization needed)

    def check_cells(self):
        for w, (code, scale) in enumerate(zip(self.cells[:2], self.cells[2:])):
            bad = np.argwhere(~P.same(code.numpy(), self.pool.code[w]))
            assert not len(bad), ("kv"[w], len(bad), bad[:4])
            np.testing.assert_array_equal(scale.numpy(), self.pool.scale[w])

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
            tol = P.bound(want, A, B, V, max(1, int(self.kv[s])), self.D, self.act, not self.decode)
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


# ---- append ----

@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("H,hk,D,ps", [(4, 2, 128, 16), (7, 1, 64, 32), (40, 20, 128, 64)])
def test_append(dev, act, few, H, hk, D, ps):
    """Ragged sequences (one empty, one whose first rows stand before position 0, one
    with a length that is none, one with a page outside the pool), blocks that older
    rows are in, of a smaller and of a larger scale than the new, rows before and
    behind them, q, k and v as parts of one wide row."""
    say("append", act, few, H, hk, D, ps)
    rng = seed(1, act, H, D, few)
    past, new = [0, 5, 31, -3, 40, 0, 2, 20, 13, 47, 15], [1, 30, 0, 9, 3, 65, 4, 7, 1, 2, 50]
    if few:  # two rows a sequence at most in the mean
        past, new = past + [int(x) for x in rng.integers(0, 60, 109)], new + [int(x) for x in rng.integers(0, 2, 109)]
        new[50:53] = 12, 3, 17
        past[50:53] = 10, 30, 8
    c = Case(dev, rng, act, H, hk, D, ps, past, new, row0=2, tail=3, width=8 if ps < 64 else 0, fill=False)
    for s, p in enumerate(past):
        c.pool.fill(rng, s, p, std=[1.0, 0.01, 60.0][s % 3])
    width = (H + 2 * hk) * D + 8
    qkv = rng.standard_normal((c.rows, width)).astype(np.float32)
    cos, sin = R.tables(60, D)  # (sequences 5 and 10 go to position 64)
    c.kv[6] = c.pool.table.shape[1] * ps + 1
    c.pool.table[7, 20 // ps] = c.pool.n_pages
    c.upload()
    x = put(dev, qkv, act)
    size = x.nbytes // x.shape[0] // x.shape[1]
    qo = put(dev, np.full((c.rows, H * D + 16), 7.0), act)
    cd, sd = dev.from_numpy(cos), dev.from_numpy(sin)
    call = lambda: F.paged_append(  # noqa: E731
        c.kvc, c.batch, act, H, x, x.ptr + H * D * size, x.ptr + (H + hk) * D * size, qo, ldq=width, ldk=width,
        ldv=width, ldqo=H * D + 16, rope_cos=cd, rope_sin=sd, rope_rows=60)
    call()
    xq = R.from_bits(R.to_bits(qkv, act), act)
    want_q = np.full((c.rows, H * D + 16), 7.0, np.float32)
    for s, n in enumerate(new):
        if n == 0:
            continue
        pos = int(c.kv[s]) - n + np.arange(n)
        rows = xq[c.start[s]:c.start[s] + n]
        q, k, v = (a.reshape(n, -1, D) for a in np.split(rows[:, :(H + 2 * hk) * D], [H * D, (H + hk) * D], 1))
        at = np.clip(pos, 0, 59)
        turned = R.rotate(q, cos[at], sin[at])
        turned[pos < 0] = 0
        turned[pos >= 60] = np.nan
        if s == 6:
            turned[:] = np.nan
        want_q[c.start[s]:c.start[s] + n, :H * D] = turned.reshape(n, -1)
        if s == 6:
            continue
        on = (pos >= 0) & (pos < 60)
        c.pool.append(s, int(pos[on][0]), R.rotate(k, cos[at], sin[at])[on], v[on])
    got = qo.numpy()
    np.testing.assert_array_equal(np.isnan(R.from_bits(got, act)), np.isnan(want_q))
    ok = ~np.isnan(want_q)
    np.testing.assert_array_equal(got[ok], R.to_bits(want_q, act)[ok])
    c.check_cells()
    call()  # the same rows once more: the same cache
    c.check_cells()


@pytest.mark.parametrize("act,hk,D", [(F32, 3, 64), (BF16, 8, 128), (F16, 17, 64), (F32, 9, 128), (F16, 2, 128),
                                      (BF16, 1, 64)])
def test_append_tokens_one_by_one(dev, act, hk, D):
    """One row a sequence, from each position of a block on, magnitudes that grow and
    shrink from token to token; without tables, without q, and in place."""
    rng = seed(2, act, hk)
    H, ps, n = 2 * hk, 32, 70
    c = Case(dev, rng, act, H, hk, D, ps, [0] * n, [40] * n, decode=True, fill=False, width=3)
    c.new, c.rows = [1] * n, n
    c.q = rng.standard_normal((n, c.ldq)).astype(np.float32)
    c.kv = rng.integers(0, 17, n).astype(np.int32)
    c.kv[:3] = 0, -1, 97
    for s in range(3, n):
        c.pool.fill(rng, s, int(c.kv[s]), std=2.0 ** rng.integers(-8, 8))
    c.upload()
    cos, sin = R.tables(40, D)
    cd, sd = dev.from_numpy(cos), dev.from_numpy(sin)
    for step in range(18):
        c.kv[3:] += 1
        c.ints[1].copy_from(c.kv)
        k, v = ((rng.standard_normal((n, hk * D)) * 2.0 ** rng.integers(-9, 9, (n, 1))).astype(np.float32)
                for _ in range(2))
        kd, vd = put(dev, k, act), put(dev, v, act)
        k, v = (R.from_bits(R.to_bits(a, act), act).reshape(n, hk, D) for a in (k, v))
        pos = np.maximum(c.kv - 1, 0) % 40
        turned = R.rotate(k, cos[pos], sin[pos])
        if step % 3 == 0:
            say("append one", step)
            F.paged_append(c.kvc, c.batch, act, H, None, kd, vd, None)
            turned = k
        else:
            F.paged_append(c.kvc, c.batch, act, H, c.q_dev, kd, vd, c.q_dev if step == 17 else c.out, rope_cos=cd,
                           rope_sin=sd, rope_rows=40)
        for s in range(3, n):
            c.pool.append(s, int(c.kv[s]) - 1, turned[s:s + 1], v[s:s + 1])
        c.check_cells()
    q = R.from_bits(R.to_bits(c.q, act), act).reshape(n, H, D)
    want = R.rotate(q, cos[pos], sin[pos]).reshape(n, -1)
    want[0], want[1:3] = 0, np.nan
    got = c.q_dev.numpy()
    assert np.isnan(R.from_bits(got[1:3], act)).all()
    np.testing.assert_array_equal(got[[0, *range(3, n)]], R.to_bits(want[[0, *range(3, n)]], act))


@pytest.mark.parametrize("one", [False, True])
def test_append_extreme_values(dev, one):
    """Blocks of zeros, of the smallest and the largest numbers, of ties between codes,
    with infinite and NaN values, and older rows under a NaN scale."""
    say("append extremes", one)
    rng = seed(3)
    D, hk, H = 64, 1, 1
    big = np.float32(np.finfo(np.float32).max)
    blocks = [np.zeros(D), np.full(D, 1e-45), np.full(D, 1e-40), np.linspace(-big, big, D, dtype=np.float64),
              np.full(D, big), np.full(D, 448.0), np.full(D, np.nextafter(np.float32(448), np.float32(500))),
              np.r_[np.nan, np.inf, -np.inf, np.ones(D - 3)], np.full(D, np.nan), np.r_[-0.0, np.arange(1, D) / 7],
              (P.CODE[:126:2][:63][None] + P.CODE[1:127:2][:63][None])[0].tolist() + [448.0],
              np.r_[448.0, 2.0 ** -6 - 2.0 ** -11, 2.0 ** -10, 2.0 ** -9 * 1.5, np.zeros(D - 4)]]
    blocks = [np.asarray(b, np.float32) for b in blocks]
    blocks[10][:63] /= 2  # (means of neighbouring codes)
    n = len(blocks)
    past = [0] * n + [3] * n + [5] * n
    c = Case(dev, rng, F32, H, hk, D, 16, past, [1] * 3 * n, decode=one, fill=False)
    for s in range(n, 3 * n):
        c.pool.fill(rng, s, past[s], std=1.0 if s < 2 * n else 2.0 ** 100)
    page = c.pool.table[n + 4, 0]
    c.pool.scale[:, page] = 255
    x = np.stack(blocks * 3)
    c.upload()
    xd, yd = put(dev, x), put(dev, -x)
    F.paged_append(c.kvc, c.batch, F32, H, None, xd, yd, None)
    for s in range(3 * n):
        c.pool.append(s, past[s], x[s].reshape(1, 1, D), -x[s].reshape(1, 1, D))
    c.check_cells()
    k, _ = c.pool.get(4, 1)
    assert np.isfinite(k).all() and (np.abs(k) < 2.0 ** 128).all()


# ---- attention ----

LAYOUTS = [(4, 4, 128), (8, 2, 128), (16, 2, 64), (7, 1, 128), (20, 1, 64), (40, 2, 128)]


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("H,hk,D", LAYOUTS)
def test_decode(dev, act, H, hk, D):
    say("decode", act, H, hk, D)
    ps = 16 if H != 16 else 64
    lens = [1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300, 0, 777]
    c = Case(dev, seed(4, act, H), act, H, hk, D, ps, [n - 1 for n in lens], [1] * len(lens), pad=8, decode=True)
    c.upload()
    c.run()
    a = c.check()
    c.run()
    np.testing.assert_array_equal(c.got(), a)  # the same call, the same bits


@pytest.mark.parametrize("act,H,hk,D,lens", [
    (F32, 2, 1, 128, [4097]), (F16, 4, 1, 64, [20000]), (BF16, 8, 8, 128, [3000, 5, 1500]),
    (F16, 4, 2, 128, [40] * 300), (F32, 5, 1, 128, [2500, 0, 2500]), (BF16, 34, 2, 64, [6001]),
    (F32, 16, 16, 64, [1030, 1025, 1500, 3])])
def test_decode_long(dev, act, H, hk, D, lens):
    say("decode_long", act, H, hk, D, lens[:3])
    c = Case(dev, seed(5, H, D), act, H, hk, D, 16, [n - 1 for n in lens], [1] * len(lens), decode=True)
    c.upload()
    c.run()
    c.check()


@pytest.mark.parametrize("ps", [16, 32, 128, 1024])
def test_page_sizes_and_scales(dev, ps):
    say("decode page", ps)
    lens = [1, 1023, 1025, 500]
    c = Case(dev, seed(6, ps), F16, 6, 2, 128, ps, [n - 1 for n in lens], [1] * 4, decode=True, width=70)
    c.upload()
    for scale in (c.scale, -0.3, 0.0):
        c.run(scale)
        c.check(scale=scale)


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("decode", [True, False])
def test_scales_far_apart(dev, act, decode):
    """Blocks of keys and of values of very different size, beside blocks of zeros:
    each row's result keeps the digits of the blocks that it weighs."""
    say("scales far apart", act, decode)
    rng = seed(7, act, decode)
    H, hk, D, n = 4, 2, 128, 600
    new = [1, 1] if decode else [70, 1]
    c = Case(dev, rng, act, H, hk, D, 16, [n - new[0], 129], new, decode=decode, fill=False)
    for s, length in enumerate((n, 130)):
        k, v = rng.standard_normal((2, length, hk, D)).astype(np.float32)
        k *= 2.0 ** rng.integers(-12, 1, (length // 16 + 1)).repeat(16)[:length, None, None]
        v *= 2.0 ** rng.integers(-30, 30, (length // 16 + 1)).repeat(16)[:length, None, None]
        k[32:48], v[64:80] = 0, 0
        c.pool.append(s, 0, k.astype(np.float32), v.astype(np.float32))
    c.upload()
    c.run()
    # (f16 outputs past f16's range are infinite)
    if act == F16:
        got = c.got()
        assert not np.isnan(got).any()
    else:
        c.check()


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("H,hk,D", LAYOUTS)
def test_prefill(dev, act, H, hk, D):
    say("prefill", act, H, hk, D)
    new = [1, 0, 17, 64, 3, 130, 31, 9]
    past = [0, 0, 0, 5, 100, 0, 33, -4]
    c = Case(dev, seed(8, act, H, D), act, H, hk, D, 16 if H != 8 else 128, past, new, row0=1, tail=2, pad=8)
    c.upload()
    c.run()
    a = c.check()
    c.run()
    np.testing.assert_array_equal(c.got(), a)


@pytest.mark.parametrize("act,H,hk,D,past,new", [
    (BF16, 8, 2, 128, [0], [700]), (F32, 4, 1, 128, [300, 0], [333, 257]), (F16, 16, 1, 64, [0, 90], [513, 200]),
    (F32, 2, 2, 64, [1000, 3000], [64, 129]), (F16, 32, 4, 128, [2000], [100]), (BF16, 5, 5, 64, [0] * 9, [70] * 9),
    (BF16, 4, 4, 128, [6000, 0], [20, 1]), (F32, 1, 1, 128, [9000], [30])])
def test_prefill_long(dev, act, H, hk, D, past, new):
    say("prefill_long", act, H, hk, D, past[:3], new[:3])
    c = Case(dev, seed(9, H, D, act), act, H, hk, D, 16, past, new)
    c.upload()
    c.run()
    c.check()


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("H,hk,D,top", [(20, 20, 128, 100), (40, 20, 64, 250), (3, 3, 128, 31), (70, 2, 64, 30)])
def test_many_short_sequences(dev, act, H, hk, D, top):
    """Lengths of none, one and up to `top`, a length that is none, a page that is
    none, sequences of no rows, keys behind a row that are no numbers."""
    for decode in (True, False):
        say("many short", act, decode, H, D, top)
        rng = seed(10, act, H, decode)
        kv = np.concatenate([[0, 1, 2, 16, 17, top, top, 25, 25], rng.integers(1, top + 1, 24)])
        new = [1] * len(kv) if decode else [0, 1, 2, 3, 17, 4, 0, 3, 9] + [int(n) for n in rng.integers(0, 4, 24)]
        c = Case(dev, rng, act, H, hk, D, 16, [int(n) - m for n, m in zip(kv, new)], new, row0=0 if decode else 2,
                 tail=0 if decode else 3, pad=8, decode=decode, max_kv_len=top)
        c.kv[7] = top + 1
        c.pool.table[8, 1] = -1  # (positions 16 ..: all rows of sequence 8)
        c.upload()
        c.run()
        got = c.check(skip=(7, 8))
        for s in (7, 8):
            assert np.isnan(got[c.start[s]:c.start[s] + new[s], :H * D]).all()
        c.run()
        np.testing.assert_array_equal(c.got(), got)


def test_malformed_batches_stay_in_bounds(dev):
    """Lengths that are none give NaN, a page outside the pool NaN for the rows
    that see it, ranges that are none leave the output alone."""
    rng = seed(11)
    say("malformed decode")
    c = Case(dev, rng, F16, 4, 2, 128, 16, [40, 40, 40, 40, 40], [1] * 5, decode=True)
    c.kv[1], c.kv[2] = -1, 49
    c.pool.table[3, 1], c.pool.table[4, 2] = -1, c.pool.n_pages
    c.upload()
    c.run()
    got = c.check(skip=(1, 2, 3, 4))
    assert np.isnan(got[1:, :4 * 128]).all()
    for H, hk in ((4, 2), (64, 1)):
        say("malformed prefill", H)
        c = Case(dev, rng, BF16, H, hk, 64, 16, [0, 0, 3, 0, 10], [20, 40, 5, 33, 6])
        c.pool.table[1, 1] = c.pool.n_pages          # rows 16 .. of sequence 1 see it
        c.kv[3] = 1 << 20
        c.start[5] = c.rows + 1                      # sequence 4 ends behind the rows
        c.upload()
        c.run()
        got, w = c.got(), H * 64
        c.new[4] = 0
        c.check(skip=(1, 3))
        s1, s3 = c.start[1], c.start[3]
        assert np.isnan(got[s1 + 16:s1 + 40, :w]).all() and np.isfinite(got[s1:s1 + 16, :w]).all()
        assert np.isnan(got[s3:s3 + 33, :w]).all()


def _odd(c, kv_new):
    """What each row's result has to be where NaN values are among the cache's: NaN
    in the dims of the NaN values that it sees (of v), or in all (of k)."""
    got = c.got()[:, :c.H * c.D].reshape(c.rows, c.H, c.D)
    for s, n in enumerate(kv_new):
        k, v = c.pool.get(s, int(c.kv[s]))
        for i in range(n):
            pos = int(c.kv[s]) - n + i
            row = int(c.start[s]) + i
            for h in range(c.H):
                g = h * c.hk // c.H
                want = np.isnan(v[:pos + 1, g]).any(0) | np.isnan(k[:pos + 1, g]).any()
                np.testing.assert_array_equal(np.isnan(got[row, h]), want, err_msg=str((s, i, h)))
    return got


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("H,hk,new", [(4, 2, 1), (4, 2, 40), (64, 2, 90)])
def test_nan_codes_and_scales(dev, act, H, hk, new):
    """A NaN code of v, of k, and NaN scales of a block that only later rows see: the
    rows and dims that see them are NaN, the others the numbers of a cache without."""
    say("nan codes", act, H, new)
    rng = seed(12, act, H)
    D, n = 128, 333
    c = Case(dev, rng, act, H, hk, D, 16, [n - new] * 4, [new] * 4, decode=new == 1)
    clean = c.pool.code.copy(), c.pool.scale.copy()
    pg = lambda s, j: (c.pool.table[s, j // 16], j % 16)  # noqa: E731
    for s, (w, j, d) in enumerate([(1, 100, 7), (0, n - 5, 3), (1, n - 3, 120)]):
        page, i = pg(s, j)
        c.pool.code[w, page, 1, i, d] = 0xff if s else 0x7f
    page, i = pg(3, n - 2)  # the last block: rows before its first position see none of it
    c.pool.scale[1, page, 0] = 255
    c.upload()
    c.run()
    odd = _odd(c, [new] * 4)
    c.pool.code, c.pool.scale = clean
    c.upload()
    c.run()
    c.check()
    even = c.got()[:, :H * D].reshape(odd.shape)
    some = ~np.isnan(odd)
    # (a walk of other blocks: the same within both's bound, of the result's size at most)
    np.testing.assert_allclose(odd[some], even[some], rtol=2.0 ** -6, atol=2.0 ** -6)
