"""The paged attention calls beside infinities, NaN and values far apart: every
output against the definition in 64 bits, infinities and NaN where it has them
and only there, the rest within the bounds of paged_ref.py."""
import numpy as np
import pytest

import paged_ref as R
from paged_ref import BF16, F16, F32
from test_gpu_paged import TYPES, Case, say, seed

pytestmark = pytest.mark.gpu


def compare(got, want, tol):
    """NaN and infinities at the same places, finite values within tol."""
    odd = ~np.isfinite(want)
    np.testing.assert_array_equal(got[odd], want[odd])
    err = np.abs(got[~odd] - want[~odd])
    assert np.isfinite(got[~odd]).all(), np.argwhere(~np.isfinite(got) & ~odd)[:4]
    assert (err <= tol[~odd]).all(), (np.argwhere(~odd)[~(err <= tol[~odd])][:4], err.max())


def rows_of(c, s):
    n, r0 = c.new[s], int(c.start[s])
    q = R.from_bits(R.to_bits(c.q, c.act), c.act)[r0:r0 + n, :c.H * c.D].reshape(n, c.H, c.D)
    return q, int(c.kv[s]) - n + np.arange(n)


def got_of(c, s):
    return c.got()[int(c.start[s]):int(c.start[s + 1]), :c.H * c.D].reshape(c.new[s], c.H, c.D)


# heads, KV heads, dims, cached, new: 16-row tiles, 64-row tiles, 128-row tiles, cut 128-row tiles
PREFILL = [(4, 2, 64, [0, 30], [170, 160]), (4, 2, 128, [0, 30], [170, 160]), (20, 20, 128, [40] * 30, [9] * 30),
           (32, 2, 128, [0, 30], [170, 160]), (64, 4, 64, [0, 30], [170, 160]),
           (20, 20, 128, [0, 0, 70, 0, 3], [200, 260, 130, 60, 200]),
           (40, 20, 64, [0, 0, 70], [200, 260, 130]), (32, 2, 128, [2200, 2000], [150, 140]),
           (40, 2, 64, [2200, 2000], [150, 140])]


def put_values(c, s, odd):
    """odd: (key, KV head, dim, value) of sequence s's V, the last where several name
    one element; its keys, and V with zeros there."""
    k, v = c.pool.get(s, int(c.kv[s]))
    v, zeroed = v.copy(), v.copy()
    for j, g, d, x in odd:
        v[j, g, d], zeroed[j, g, d] = x, 0
    c.pool.put(s, np.arange(len(k)), k, v)
    return k, zeroed


def check_values(c, s, odd, k, zeroed, prefill):
    q, pos = rows_of(c, s)
    want, A, B, V = R.attend(q, k, zeroed, pos, c.scale)
    tol = R.bound(want, A, B, V, len(k), c.D, c.act, c.cache, prefill)
    grp = c.H // c.hk
    with np.errstate(invalid="ignore"):
        for (j, g, d), x in {o[:3]: o[3] for o in odd}.items():  # (weights are above 0 in 64 bits, and in f32 for rows like these)
            want[pos >= j, g * grp:(g + 1) * grp, d] += x
    compare(got_of(c, s), want, tol)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,lens", [(8, 2, 128, [5000, 1235]), (4, 1, 64, [9001]), (8, 8, 128, [2500, 40, 777])])
def test_decode_joins_infinite_pieces(dev, act, cache, H, hk, D, lens):
    """An infinite value in a sequence's last key: it is in the last of the pieces
    that are joined, which stands for those past it as well."""
    say("decode joins", act, cache, H, D, lens)
    c = Case(dev, seed(31, act, cache, H, D), act, cache, H, hk, D, 16, [n - 1 for n in lens], [1] * len(lens),
             decode=True)
    odds = [[(n - 1, 0, 4, np.inf), (n - 1, hk - 1, D - 3, -np.inf)] for n in lens]
    plain = [put_values(c, s, odd) for s, odd in enumerate(odds)]
    c.upload()
    c.run()
    for s, odd in enumerate(odds):
        check_values(c, s, odd, *plain[s], False)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", PREFILL)
def test_prefill_single_values_that_are_no_numbers(dev, act, cache, H, hk, D, past, new):
    """Single infinite and NaN elements of V, in even and odd dims, in early keys
    that all rows see, on the diagonal and behind it."""
    say("prefill single values", act, cache, H, D, past)
    c = Case(dev, seed(30, act, cache, H, D), act, cache, H, hk, D, 16, past, new, row0=1, tail=2, pad=8)
    inf, nan, g = np.inf, np.nan, hk - 1
    odds = []
    for s, (p, n) in enumerate(zip(past, new)):
        at = p + n // 2
        odds.append([(0, 0, 0, inf), (p + min(17, n - 1), g, 3, -inf), (at, 0, 6, nan), (at + 1, 0, 7, inf), (at + 1, g, 10, -inf),
                     (at + 2, 0, 7, -inf), (p + n - 1, g, D - 1, inf), (p + max(0, n - 20), 0, D - 2, nan)])
    plain = [put_values(c, s, odd) for s, odd in enumerate(odds)]
    c.upload()
    for _ in range(2):
        c.run()
        for s, odd in enumerate(odds):
            check_values(c, s, odd, *plain[s], True)


# 16-row tiles: cut over the workgroups, whole, a wavefront each
DECODE = [(8, 2, 128, [1500, 1235, 0, 40]), (4, 1, 64, [9001]), (8, 8, 128, [300, 1, 77, 130]), (6, 2, 64, [1] * 3 + [500]),
          (40, 20, 128, [20, 31, 2]), (64, 32, 64, [100] * 9 + [250] * 8)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,lens", DECODE)
def test_decode_single_values_that_are_no_numbers(dev, act, cache, H, hk, D, lens):
    """Single infinite and NaN elements of V early and late in a sequence: infinite
    where the definition is, whichever block of keys holds them."""
    say("decode single values", act, cache, H, D, lens[:4])
    c = Case(dev, seed(32, act, cache, H, D), act, cache, H, hk, D, 16, [n - 1 for n in lens], [1] * len(lens), pad=8,
             decode=True)
    inf, nan = np.inf, np.nan
    odds = [[(j, g % hk, d, x) for j, g, d, x in [(0, 0, 0, inf), (n // 3, 1, 3, -inf), (n // 2, 0, 8, nan), (n // 2, 0, 9, inf),
                                                  (n // 3, 0, 9, -inf), (n - 1, 1, D - 1, inf)]] if n else [] for n in lens]
    plain = [put_values(c, s, odd) for s, odd in enumerate(odds)]
    c.upload()
    for _ in range(2):
        c.run()
        for s, odd in enumerate(odds):
            check_values(c, s, odd, *plain[s], False)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new,decode", [(*x, False) for x in PREFILL] +
                         [(H, hk, D, [n - 1 for n in lens if n > 3], [1] * sum(n > 3 for n in lens), True)
                          for H, hk, D, lens in DECODE])
def test_keys_of_infinite_dims(dev, act, cache, H, hk, D, past, new, decode):
    """A key of -inf in one dim: a weight of 0 for the rows whose q is above 0
    there, no number for those below."""
    say("infinite keys", act, cache, H, D, past[:3])
    c = Case(dev, seed(33, act, cache, H, D), act, cache, H, hk, D, 16, past, new, decode=decode)
    keys = [min(2 + p + n // 2, p + n - 1) for p, n in zip(past, new)]
    plain = []
    for s, j in enumerate(keys):
        k, v = c.pool.get(s, int(c.kv[s]))
        plain.append((np.delete(k, j, 0), np.delete(v, j, 0)))
        k = k.copy()
        k[j, :, 5] = -np.inf
        c.pool.put(s, np.arange(len(k)), k, v)
    c.upload()
    c.run()
    for s, j in enumerate(keys):
        q, pos = rows_of(c, s)
        assert (q[..., 5] != 0).all() and j > 0
        want, A, B, V = R.attend(q, *plain[s], pos - (pos >= j), c.scale)
        tol = R.bound(want, A, B, V, int(c.kv[s]), D, act, cache, not decode)
        want[(pos >= j)[:, None] & (q[..., 5] < 0)] = np.nan
        compare(got_of(c, s), want, tol)


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("weight", [2.0 ** -30, 1e-9, 1e-10, 1e-8])
@pytest.mark.parametrize("H,rows", [(1, 1), (32, 2), (64, 20), (128, 300)])
def test_f32_rows_keep_small_weights(dev, H, rows, weight, decode):
    """A key far above all others, late or early: the weights of the others, 1e-10
    .. 1e-8 of its own, are all of dim 0 of the output.  f32 sums keep them to some
    n steps of f32; over f16 pages they are held to the parts' 2^-22, but those in
    a block or tile with the large one (64 keys), to 2^-40 of that one."""
    rows = 1 if decode else rows
    for n in (600, 9000 if H * rows > 10000 else 30001):
        say("f32 small weights", H, rows, weight, decode, n)
        D, at = 128, 17 if n == 600 else n - 2 * rows - 100
        c = Case(dev, seed(34), F32, F16, H, 1, D, 16, [n - rows], [rows], decode=decode)
        k, v = np.zeros((n, 1, D), np.float32), np.zeros((n, 1, D), np.float32)
        k[at, 0, 0] = 32.0
        v[:, 0, 0] = 1.0
        v[at, 0, 0], v[at, 0, 1] = 0.0, 1.0
        c.pool.put(0, np.arange(n), k, v)
        c.q[:] = 0
        c.q[:, ::D] = -np.log(weight) / 32 / 0.25
        c.upload()
        c.run(0.25)
        q, pos = rows_of(c, 0)
        want = R.attend(q, k, v, pos, 0.25)[0]
        got = got_of(c, 0)
        # the score 32 q 0.25 is rounded at most four times, where the weight's logarithm is some 23
        near = 64 * 2.0 ** -41 / weight / n
        tol = want[..., 0] * ((4 * 23 + 2 * n + 16) * R.U + 2.0 ** -22 + near)
        err = np.abs(got[..., 0] - want[..., 0])
        assert (err <= tol).all(), (err / want[..., 0]).max()
        assert np.abs(got[..., 1] - 1).max() < 1e-3 and (got[..., 2:] == 0).all()


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,past,new", [(4, 900, 1), (4, 700, 30), (64, 300, 60), (32, 4000, 150), (32, 0, 700)])
def test_scores_that_rise_and_fall(dev, act, cache, H, past, new):
    """Scores that rise and fall by far more than the weights' types hold, in runs
    of some tiles and of single keys, with a dim for each run's values."""
    say("rise and fall", act, cache, H, past, new)
    D, n = 128, past + new
    rng = seed(35, act, cache, H)
    c = Case(dev, rng, act, cache, H, 2, D, 16, [past], [new], decode=new == 1)
    k, v = (a.copy() for a in c.pool.get(0, n))
    run = np.arange(n) // 90
    k[:, :, 0] = np.array([0, 60, -10, 150, 40, 149, -30, 100])[run % 8][:, None]
    k[::37, :, 0] += 7
    c.q[:, ::D] = 1.0
    v[np.arange(n), :, run % 8] += 2.0
    c.pool.put(0, np.arange(n), k, v)
    for scale in (1.0, 0.125):
        c.upload()
        c.run(scale)
        c.check(scale=scale)


@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("H,past,new", [(4, 900, 1), (4, 700, 30), (64, 300, 60), (20, 0, 700), (32, 4000, 150)])
def test_f32_rows_keep_small_dims(dev, cache, H, past, new):
    """A dim of q of 2^20 that no key has: the scores are those of the other dims.
    The parts of these, in steps of 2^-40 of 2^20 .. 2^21, add 2^-20 |k| a dim at
    most, some 2^-17 in all: less than the bound's (D + 9) A u, A near 9 here."""
    say("f32 small dims", cache, H, past, new)
    D = 128
    c = Case(dev, seed(36, cache, H), F32, cache, H, 4, D, 16, [past], [new], decode=new == 1)
    k, v = (a.copy() for a in c.pool.get(0, past + new))
    k[:, :, 3] = 0
    c.pool.put(0, np.arange(past + new), k, v)
    c.q[:, 3::D] = 2.0 ** 20 * 1.375
    c.upload()
    c.run()
    c.check()


@pytest.mark.parametrize("act,cache", [(F32, F16), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("H,hk,D,past,new", [(4, 2, 128, [0, 4, 39, 1300], [1] * 4), (8, 2, 64, [0, 12], [7, 3]),
                                             (64, 4, 128, [0, 3], [60, 70]), (64, 2, 64, [0, 0], [150, 290]),
                                             (32, 2, 128, [3000], [140])])
def test_scores_far_below_zero(dev, act, cache, H, hk, D, past, new):
    """Scores of some -1e32 and lower: a row's weights are 1 for its largest and 0
    for the others, whose distances are far above 1.  f32 scores err by (D + 9) u A
    at most (paged_ref.py), A the largest of the row's, so that where its two largest
    are within twice that they may come out in either order: a few rows, of which one
    was seen (two scores 2.9e-8 A apart, u is 6e-8).  These only have to be finite."""
    say("far below zero", act, cache, H, D, past)
    rng = seed(37, act, cache, H)
    c = Case(dev, rng, act, cache, H, hk, D, 16, past, new, decode=new[0] == 1)
    for s, n in enumerate(c.kv):
        k, v = c.pool.get(s, int(n))
        c.pool.put(s, np.arange(n), np.abs(k) + 0.25, v)
    c.q = -(np.abs(c.q) + 0.25) * np.float32(1e32)
    c.upload()
    c.run()
    for s, n in enumerate(c.kv):
        q, pos = rows_of(c, s)
        k, v = c.pool.get(s, int(n))
        want, A = R.attend(q, k, v, pos, c.scale)[:2]
        tol = np.abs(want) * (16 * R.U + (0 if act == F32 else R.HALF[act]))
        undecided = 0
        for h in range(H):
            x = np.where(np.arange(n)[None] <= pos[:, None], q[:, h].astype(float) @ k[:, h * hk // H].T.astype(float), -np.inf)
            x = np.sort(x * c.scale, 1)
            near = x[:, -1] - (x[:, -2] if n > 1 else -np.inf) < 2 * (D + 9) * R.U * A[:, h, 0]
            undecided += int(near.sum())
            tol[near, h] = 2 * np.abs(v).max()
        assert undecided <= max(1, q.shape[0] * H // 500)
        compare(got_of(c, s), want, tol)


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("H,hk,D,past,new", [(4, 2, 128, [0, 4, 39, 2300], [1] * 4), (8, 2, 64, [0, 12], [7, 3]),
                                             (64, 4, 128, [0, 3], [60, 70]), (64, 2, 64, [0, 0], [150, 290]),
                                             (20, 20, 128, [0, 0, 70], [200, 260, 130]), (32, 2, 128, [3000], [140])])
def test_values_at_the_end_of_the_range(dev, act, H, hk, D, past, new):
    """Values up to bf16's largest: their weighted mean is a number."""
    say("large values", act, H, D, past)
    rng = seed(38, act, H)
    c = Case(dev, rng, act, BF16, H, hk, D, 16, past, new, decode=new[0] == 1)
    for s, n in enumerate(c.kv):
        k, v = c.pool.get(s, int(n))
        c.pool.put(s, np.arange(n), k, rng.uniform(-3.3e38, 3.3e38, v.shape) * (np.arange(D) % 2 == 0) + v)
    c.upload()
    c.run()
    for scale in (c.scale, 0.0):
        c.run(scale)
        c.check(scale=scale)


# past the caches: one tile reads its keys alone, and they may be more than 256 MB
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,n,cap", [(4, 2, 128, 4, 65536), (4, 2, 64, 4, 131072),   # 16-row tiles, cut
                                          (16, 8, 128, 256, 256), (8, 8, 64, 500, 256)])  # a wavefront each
def test_decode_past_the_caches(dev, act, cache, H, hk, D, n, cap):
    say("past the caches", act, cache, H, D, n, cap)
    assert n * cap * hk * D * 4 > 256e6
    rng = seed(39, act, cache, D, n)
    kv = np.concatenate([[0, 1, 256, 17], rng.integers(1, 90, n - 4)]) if cap == 256 else np.array([3000, 0, 1234, 31])
    c = Case(dev, rng, act, cache, H, hk, D, 16, [int(x) - 1 for x in kv], [1] * n, pad=8, decode=True, width=cap // 16,
             max_kv_len=cap)
    c.upload()
    c.run()
    got = c.check()
    c.run()
    np.testing.assert_array_equal(c.got(), got)
