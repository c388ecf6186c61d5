"""The 8-bit paged KV cache as a server holds it: recorded prompts replayed with other
lengths and NaN codes between, pools past four GiB, two handles at once, and values
and scores at the ends of their ranges."""
import ctypes as C

import numpy as np
import pytest

import fuel_amd as F
import paged8_ref as P
import paged_ref as R
from fuel_amd.hiprt import HipRuntime
from paged_ref import BF16, F16, F32
from test_gpu_paged8 import Case, TYPES, put, say, seed

pytestmark = pytest.mark.gpu


# 16-row tiles whole and cut, 64-row tiles, 128-row tiles, cut 128-row tiles
@pytest.mark.parametrize("act,H,hk,D,past,new", [
    (F16, 4, 2, 128, [60, 0, 7], [9, 30, 20]), (F32, 4, 2, 64, [3000, 20, 700], [3, 1, 2]),
    (BF16, 32, 2, 128, [0, 30, 0], [170, 60, 70]), (F32, 20, 20, 64, [0, 70, 0], [330, 260, 130]),
    (F16, 32, 2, 128, [2200, 2000, 0], [150, 100, 40])])
def test_prompts_captured_and_replayed(dev, act, H, hk, D, past, new):
    say("captured prompts", act, H, D, past)
    rng = seed(20, act, H, D)
    c = Case(dev, rng, act, H, hk, D, 16, past, new, pad=8)
    c.max_kv_len = int(max(c.kv))
    full, rows = c.kv.copy(), c.rows
    c.upload()
    page = int(c.pool.table[1, 0])
    clean = c.pool.code.copy()
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
            c.pool.code[:] = clean
            if odd:
                c.pool.code[1, page, 0, 3, 5] = P.NAN
            c.cells[1].copy_from(c.pool.code[1])
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
                np.testing.assert_array_equal(np.isnan(mine), want)
            c.out.copy_from(R.to_bits(np.full((rows, c.ldo), 7.0, np.float32), act))
            c.run()  # eager, the same bits
            np.testing.assert_array_equal(c.got(), got)
        rt.graph_destroy(graph)
    finally:
        dev.set_stream(None)
        rt.stream_destroy(stream)


def test_pools_past_four_gib(dev):
    """Pages whose offsets pass 32 bits, appended to and read."""
    say("large pool")
    H, hk, D, ps = 2, 2, 128, 1024
    n_pages = (1 << 33) // (hk * ps * D) + 3  # 8 GiB a pool
    rng = seed(21)
    c = Case(dev, rng, F16, H, hk, D, ps, [1500, 900], [3, 2])
    c.upload()
    big = [dev.alloc((n_pages, hk, ps, D), np.uint8) for _ in range(2)]
    scales = [dev.alloc((n_pages, hk, ps // 16), np.uint8) for _ in range(2)]
    new = c.pool.table.copy()
    for i, old in enumerate(np.unique(c.pool.table[c.pool.table < (1 << 30)])):
        to = n_pages - 1 - i if i % 2 == 0 else n_pages // 2 + i
        new[c.pool.table == old] = to
        for src, dst in ((c.pool.code[0], big[0]), (c.pool.code[1], big[1]), (c.pool.scale[0], scales[0]),
                         (c.pool.scale[1], scales[1])):
            page = np.ascontiguousarray(src[old])
            F._native.check(F.lib().frq_memcpy_htod(dev.handle, C.c_void_p(dst.ptr + int(to) * page.nbytes),
                                                    page.ctypes.data_as(C.c_void_p), page.nbytes))
    c.kvc = F.PagedKvCache8(dev, n_pages, ps, hk, D, *big, *scales)
    c.ints[0].copy_from(new)
    c.run()
    c.check()
    one = F.PagedBatch(c.ints[0], c.ints[1], 2, new.shape[1])
    work = dev.alloc((max(16, F.paged_attention_workspace(c.kvc, one, H)),), np.uint8)
    out = put(dev, np.zeros((2, H * D)), F16)
    rows = c.start[1:] - 1
    q = put(dev, c.q[rows], F16)
    F.paged_attention_decode(c.kvc, one, F16, H, q, out, c.scale, work)
    np.testing.assert_allclose(R.from_bits(out.numpy(), F16), c.got()[rows], atol=2 ** -9, rtol=0)
    k = rng.standard_normal((2, hk * D)).astype(np.float32)
    kd = put(dev, k, F16)
    F.paged_append(c.kvc, one, F16, H, None, kd, kd, None)
    k = R.from_bits(R.to_bits(k, F16), F16).reshape(2, 1, hk, D)
    for s in range(2):
        p = int(c.kv[s]) - 1
        c.pool.append(s, p, k[s], k[s])
        old, i = c.pool.table[s, p // ps], p % ps
        row, byte = np.empty(D, np.uint8), np.empty(1, np.uint8)
        at = (int(new[s, p // ps]) * hk + 1) * ps + i
        for dst, base, off in ((row, big[1], at * D), (byte, scales[1], at // 16)):
            F._native.check(F.lib().frq_memcpy_dtoh(dev.handle, dst.ctypes.data_as(C.c_void_p),
                                                    C.c_void_p(base.ptr + off), dst.nbytes))
        np.testing.assert_array_equal(row, c.pool.code[1, old, 1, i])
        assert byte[0] == c.pool.scale[1, old, 1, i // 16]


def test_two_handles_at_once(dev):
    """Two handles with their own streams, caches and workspaces, calls enqueued in turn."""
    say("two handles")
    other = F.RocmDevice(0)
    try:
        cs = [Case(d, seed(22, i), BF16, 8, 2, 128, 16, [2000 + 300 * i, 40], [1, 1], decode=True)
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


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("new", [1, 70])
def test_values_at_the_ends_of_f32(dev, act, new):
    """Values of 2^-80 and of nearly f32's largest; f16 results past f16's range are
    infinite."""
    say("values", act, new)
    for std in (2.0 ** -80, 2.0 ** 120):
        rng = seed(23, act, new)
        c = Case(dev, rng, act, 32, 2, 64, 16, [400 - new, 90 - new], [new] * 2, decode=new == 1, fill=False)
        for s in range(2):
            k, v = rng.uniform(-1, 1, (2, int(c.kv[s]), 2, 64)).astype(np.float32)
            c.pool.append(s, 0, k, v * np.float32(std))
        c.upload()
        c.run()
        if act == F16 and std > 1:
            assert not np.isnan(c.got()).any()
        else:
            c.check()


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("new", [1, 70])
def test_scores_far_apart(dev, act, new):
    """Scores far above and below each other, q rows of very different size, one key
    far above the others, whose many small weights are half of the sum."""
    say("scores", act, new)
    rng = seed(24, act, new)
    c = Case(dev, rng, act, 32, 2, 128, 16, [900 - new, 90 - new], [new] * 2, decode=new == 1)
    c.q *= np.tile(np.repeat(10.0 ** np.array([-4 if act == F16 else -30, -4, 0, 1, 1.2, -1, -2, 1.5]), 128), 4).astype(np.float32)
    c.upload()
    c.run()
    c.check()
    n = 4000
    c = Case(dev, rng, act, 32, 2, 128, 16, [n - new], [new], decode=new == 1, fill=False)
    k, v = np.zeros((2, n, 2, 128), np.float32)
    k[17, :, 0], v[:, :, 0] = 32.0, 1.0
    v[17, :, 0], v[17, :, 1] = 0.0, 1.0
    c.pool.append(0, 0, k, v)
    c.q[:] = 0
    c.q[:, ::128] = np.log(float(n)) / 32 / 0.25
    c.upload()
    c.run(0.25)
    c.check(scale=0.25)


@pytest.mark.parametrize("act", TYPES)
def test_overlapping_ranges_end(dev, act):
    """Ranges of rows that overlap so often that their work cannot be counted: the
    calls end, and leave rows outside of them alone."""
    say("overlapping ranges", act)
    for n, H, D, new, cap in ((6, 8, 64, 100, 4096), (5000, 64, 64, 475, 1 << 20)):
        c = Case(dev, seed(25, n), act, H, 1, D, 1024, [0], [new], tail=2)
        c.pool.table = np.zeros((n, cap // 1024), np.int32)
        c.kv = np.full(n, cap, np.int32)
        c.start = np.array([0, new] * (n // 2) + [0], np.int32)
        c.upload()
        c.run()
        got = c.got()
        assert (got[new:] == 7.0).all() and (got[:, H * D:] == 7.0).all()
        k = put(dev, np.zeros((c.rows, D)), act)
        F.paged_append(c.kvc, c.batch, act, H, None, k, k, None)
        for code, was in zip(c.cells[:2], c.pool.code):  # pages but the tables'
            np.testing.assert_array_equal(code.numpy()[1:], was[1:])


# 16-row tiles, 64-row tiles, 128-row tiles, cut 128-row tiles
@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", [
    (4, 2, 128, [60, 0], [9, 30]), (32, 2, 128, [0, 30], [170, 60]), (20, 20, 64, [0, 70, 0], [330, 260, 130]),
    (32, 2, 128, [2200, 2000, 0], [150, 100, 40])])
@pytest.mark.parametrize("power", [12, 24, 45, 110])
def test_values_of_later_positions(dev, act, H, hk, D, past, new, power):
    """Values of a sequence's last positions 2^power times the others': no row before
    them loses anything, nor do blocks of zeros before them count."""
    say("later positions", act, H, D, past, power)
    rng = seed(26, act, H, D, power)
    c = Case(dev, rng, act, H, hk, D, 16, past, new, fill=False)
    cut = [int(k) - n // 2 for k, n in zip(c.kv, new)]
    for s, n in enumerate(c.kv):
        k, v = rng.standard_normal((2, n, hk, D)).astype(np.float32)
        v[cut[s]:] *= np.float32(2.0 ** power)
        if past[s]:
            v[:20] = 0
        c.pool.append(s, 0, k, v)
    c.upload()
    c.run()
    got, q = c.got(), R.from_bits(R.to_bits(c.q, act), act)
    for s, n in enumerate(new):
        r0 = int(c.start[s])
        k, v = c.pool.get(s, int(c.kv[s]))
        pos = int(c.kv[s]) - n + np.arange(n)
        want, A, B, _ = R.attend(q[r0:r0 + n].reshape(n, H, D), k, v, pos, c.scale)
        V = np.maximum.accumulate(np.abs(v).max((1, 2)))[pos][:, None, None]  # of the keys that the row sees
        tol = P.bound(want, A, B, V, int(c.kv[s]), D, act, True)
        err = np.abs(got[r0:r0 + n].reshape(want.shape) - want)
        ok = slice(0, n - n // 2) if act == F16 else slice(None)  # (f16 holds no results of the others)
        bad = np.argwhere(~(err[ok] <= tol[ok]))
        assert not len(bad), (s, bad[:3], err[ok].max())
