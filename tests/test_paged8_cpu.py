"""What the entry points of the 8-bit paged KV cache and of the plan of pages refuse,
before they touch a device (the calls name no device handle, so the arguments that
pass end in that refusal), and the reference codes against torch's e4m3."""
import ctypes as C

import numpy as np
import pytest
import torch

import fuel_amd as F
import paged8_ref as R
from fuel_amd._native import PagedBatch, PagedKv8, lib
from fuel_amd.backend import RocmStorage
from test_paged_cpu import BAD_BATCH, INVALID, MISALIGNED, P, UNSUPPORTED, WORKSPACE, batch, passes


def kv(**o):
    a = dict(n_pages=9, page_size=16, n_kv_heads=2, head_dim=128, k=P, v=P, k_scale=P, v_scale=P)
    a.update(o)
    return PagedKv8(*(a[n] for n, _ in PagedKv8._fields_))


def attend(fn="prefill", c=None, b=None, dtype=F.F16, n_heads=4, q=P, ldq=512, work=P, work_bytes=1 << 30, out=P,
           ldo=512):
    c, b = c or kv(), b or batch()
    return getattr(lib(), "frq_paged8_attention_" + fn)(None, C.byref(c), C.byref(b), dtype, n_heads, q, ldq, 0.1, work,
                                                        work_bytes, out, ldo)


def append(c=None, b=None, dtype=F.F16, n_heads=4, q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, cos=P, sin=P, rows=64,
           q_out=P, ldqo=512):
    c, b = c or kv(), b or batch()
    return lib().frq_paged8_append(None, C.byref(c), C.byref(b), dtype, n_heads, q, ldq, k, ldk, v, ldv, cos, sin, rows,
                                   q_out, ldqo)


def plan(**o):
    a = dict(n_seqs=3, max_pages=4, page_size=16, n_pages=9, rows=5, tokens=P, kv_len=P, kv_len_out=P, page_table=P,
             free_pages=P, n_free=P, n_free_out=P, row_start=P, slots=P, positions=P)
    a.update(o)
    return lib().frq_paged_plan(None, *a.values())


def test_good_arguments_reach_the_device_check():
    one = batch(rows=3, row_start=None)
    for dt in (F.F32, F.F16, F.BF16):
        assert passes(attend(dtype=dt)) and passes(append(dtype=dt))
        assert passes(attend("decode", b=one, dtype=dt)) and passes(attend(b=one)) and passes(append(b=one))
    assert passes(append(q=None, q_out=None)) and passes(append(cos=None, sin=None, rows=0))
    assert passes(attend(c=kv(head_dim=64), ldq=256, ldo=256)) and passes(attend(c=kv(k_scale=P + 1, v_scale=P + 3)))
    for b in (batch(n_seqs=0, rows=0, row_start=None), batch(rows=0)):  # nothing to do: buffers may be null
        assert passes(attend(b=b, q=None, out=None, work=None, work_bytes=0)) and passes(append(b=b, k=None, v=None))
    assert passes(plan()) and passes(plan(slots=None, positions=None)) and passes(plan(n_pages=0, free_pages=None))
    assert passes(plan(n_seqs=0, tokens=None, kv_len=None, kv_len_out=None, page_table=None, rows=0))


@pytest.mark.parametrize("how,code", [
    (dict(n_pages=0), INVALID), (dict(n_pages=1 << 31), INVALID), (dict(page_size=8), UNSUPPORTED),
    (dict(page_size=48), UNSUPPORTED), (dict(page_size=2048), UNSUPPORTED), (dict(n_kv_heads=0), INVALID),
    (dict(n_kv_heads=3), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(k=P + 8), MISALIGNED), (dict(v=P + 2), MISALIGNED), (dict(k_scale=None), INVALID),
    (dict(v_scale=None), INVALID)])
def test_refused_caches(how, code):
    assert attend(c=kv(**how)) == code and append(c=kv(**how)) == code
    assert attend("decode", c=kv(**how), b=batch(rows=3, row_start=None)) == code


@pytest.mark.parametrize("how,code", BAD_BATCH)
def test_refused_batches(how, code):
    assert attend(b=batch(**how)) == code and append(b=batch(**how)) == code


def test_refused_operands():
    for fn in ("decode", "prefill"):
        b = batch(rows=3, row_start=None)
        for how, code in [(dict(q=None), INVALID), (dict(out=None), INVALID), (dict(ldq=511), INVALID),
                          (dict(ldo=256), INVALID), (dict(ldq=516), MISALIGNED), (dict(q=P + 8), MISALIGNED),
                          (dict(n_heads=5), INVALID), (dict(n_heads=0), INVALID), (dict(dtype=F.Q8_0), UNSUPPORTED),
                          (dict(dtype=F.F32, ldq=514), MISALIGNED), (dict(dtype=99), UNSUPPORTED)]:
            assert attend(fn, b=b, **how) == code, (fn, how)
    assert attend("decode") == INVALID and b"row_start" in lib().frq_last_error()
    for how, code in [(dict(q=None), INVALID), (dict(q_out=None), INVALID), (dict(k=None), INVALID),
                      (dict(cos=None), INVALID), (dict(rows=0), INVALID), (dict(ldk=255), INVALID),
                      (dict(ldv=260), MISALIGNED), (dict(ldqo=128), INVALID), (dict(cos=P + 4), MISALIGNED),
                      (dict(dtype=F.Q4K), UNSUPPORTED), (dict(ldq=520, ldqo=512), INVALID)]:
        assert append(**how) == code, how
    L = lib()
    assert L.frq_paged8_attention_workspace(None, None, 4) == 0
    b = batch(rows=3, row_start=None, max_pages=1000)
    need = L.frq_paged8_attention_workspace(C.byref(kv()), C.byref(b), 4)
    assert need > 0 and attend("decode", b=b, work_bytes=need - 1) == WORKSPACE
    assert attend("decode", b=b, work=None) == INVALID and attend("decode", b=b, work=P + 8) == MISALIGNED
    assert passes(attend("decode", b=b, work_bytes=need))
    assert L.frq_paged8_append(None, None, C.byref(b), 0, 4, P, 512, P, 256, P, 256, P, P, 64, P, 512) == INVALID


def test_appends_end_at_the_grid():
    """A workgroup of 256 threads for a row's q (more of 64 heads and more), four
    wavefronts a workgroup for blocks of 16 rows."""
    most = (1 << 24) - 1
    c = kv(n_kv_heads=1)
    one = dict(c=c, n_heads=1, ldq=128, ldk=128, ldv=128, ldqo=128)
    assert append(b=batch(n_seqs=most, rows=most, row_start=None), **one) == UNSUPPORTED
    assert passes(append(b=batch(n_seqs=most // 2, rows=most // 2, row_start=None), **one))
    assert append(b=batch(n_seqs=1, rows=most // 2 + 1, row_start=P), n_heads=64, ldq=8192, ldqo=8192) == UNSUPPORTED


@pytest.mark.parametrize("how,code", [
    (dict(page_size=8), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED), (dict(page_size=2048), UNSUPPORTED),
    (dict(max_pages=1 << 27), UNSUPPORTED), (dict(n_seqs=(1 << 30) + 1), UNSUPPORTED),
    (dict(n_pages=(1 << 30) + 1), UNSUPPORTED), (dict(rows=(1 << 64) - 1), UNSUPPORTED), (dict(tokens=None), INVALID),
    (dict(kv_len=None), INVALID), (dict(kv_len_out=None), INVALID), (dict(page_table=None), INVALID),
    (dict(free_pages=None), INVALID), (dict(n_free=None), INVALID), (dict(n_free_out=None), INVALID),
    (dict(row_start=None), INVALID), (dict(tokens=P + 2), MISALIGNED), (dict(slots=P + 4), MISALIGNED),
    (dict(positions=P + 1), MISALIGNED), (dict(row_start=P + 3), MISALIGNED)])
def test_refused_plans(how, code):
    assert plan(**how) == code


def storage(dev, nbytes, dtype=np.uint8):
    s = RocmStorage.__new__(RocmStorage)
    s.dev, s.shape, s.dtype, s.nbytes, s.ptr = dev, (nbytes,), np.dtype(dtype), nbytes, P
    s.free = lambda: None
    return s


class Dev:
    ordinal, handle = 0, None


def test_python_checks_storages():
    dev = Dev()
    pages, scales = 9 * 2 * 16 * 128, 9 * 2
    ok = [storage(dev, n) for n in (pages, pages, scales, scales)]
    F.PagedKvCache8(dev, 9, 16, 2, 128, *ok)
    for i in range(4):
        with pytest.raises(F.FuelRocmError):
            F.PagedKvCache8(dev, 9, 16, 2, 128, *(storage(dev, s.nbytes - (i == j)) for j, s in enumerate(ok)))
        with pytest.raises(F.FuelRocmError):
            F.PagedKvCache8(dev, 9, 16, 2, 128, *(None if i == j else s for j, s in enumerate(ok)))
    i32 = lambda n, t=np.int32: storage(dev, n * np.dtype(t).itemsize, t)  # noqa: E731
    good = dict(tokens=i32(3), kv_len=i32(3), page_table=i32(12), free_pages=i32(9), n_free=i32(1), row_start=i32(4),
                slots=i32(5, np.int64), positions=i32(5))
    with pytest.raises(F.FuelRocmError, match="null device handle"):
        F.paged_plan(dev, 3, 4, 16, 9, 5, **good)
    for name, x in good.items():
        for bad in (i32(x.nbytes // x.dtype.itemsize - 1, x.dtype), storage(dev, x.nbytes, np.float32)):
            with pytest.raises(F.FuelRocmError, match=name):
                F.paged_plan(dev, 3, 4, 16, 9, 5, **{**good, name: bad})
        with pytest.raises(F.FuelRocmError, match="got list"):
            F.paged_plan(dev, 3, 4, 16, 9, 5, **{**good, name: [1, 2]})


def test_reference_codes():
    all_codes = torch.arange(256, dtype=torch.uint8)
    np.testing.assert_array_equal(R.CODE, all_codes.view(torch.float8_e4m3fn).double().numpy())
    rng = np.random.default_rng(1)
    mid = (R.CODE[:126] + R.CODE[1:127]) / 2
    x = np.concatenate([rng.uniform(-448, 448, 20000), rng.standard_normal(20000) * 2.0 ** rng.integers(-14, 6, 20000),
                        mid, np.nextafter(mid, 0), np.nextafter(mid, 500), [0.0, -0.0]]).astype(np.float32)
    np.testing.assert_array_equal(R.encode(x, 127), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    a = np.array([0, 448, 449, 224, 225, 1e-45, 3e38])
    b = R.byte(a)
    assert (a <= 448 * R.scale(b)).all() and ((a > 448 * R.scale(b - 1)) | (b == 0)).all()
