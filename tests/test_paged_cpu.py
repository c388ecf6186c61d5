"""What the paged KV cache entry points refuse, before they touch a device: the
calls name no device handle, so the arguments that pass end in that refusal."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import fuel_amd as F
from fuel_amd._native import PagedBatch, PagedKv, lib

OK, MISALIGNED, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3, 4
P = 1 << 20  # an address that nothing reads


def kv(**o):
    a = dict(dtype=F.F16, n_pages=9, page_size=16, n_kv_heads=2, head_dim=128, k=P, v=P)
    a.update(o)
    return PagedKv(*(a[n] for n, _ in PagedKv._fields_))


def batch(**o):
    a = dict(n_seqs=3, max_pages=4, rows=5, max_kv_len=0, page_table=P, kv_len=P, row_start=P)
    a.update(o)
    return PagedBatch(*(a[n] for n, _ in PagedBatch._fields_))


def attend(fn="prefill", c=None, b=None, dtype=F.F16, n_heads=4, q=P, ldq=512, work=P, work_bytes=1 << 30, out=P,
           ldo=512, dev=None):
    c, b = c or kv(), b or batch()
    return getattr(lib(), "frq_paged_attention_" + fn)(dev, C.byref(c), C.byref(b), dtype, n_heads, q, ldq, 0.1, work,
                                                       work_bytes, out, ldo)


def append(c=None, b=None, dtype=F.F16, n_heads=4, q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, cos=P, sin=P, rows=64,
           q_out=P, ldqo=512):
    c, b = c or kv(), b or batch()
    return lib().frq_paged_append(None, C.byref(c), C.byref(b), dtype, n_heads, q, ldq, k, ldk, v, ldv, cos, sin, rows,
                                  q_out, ldqo)


def passes(rc):
    return rc == INVALID and b"null device handle" in lib().frq_last_error()


def test_good_arguments_reach_the_device_check():
    assert passes(attend()) and passes(append())
    one = batch(rows=3, row_start=None)
    assert passes(attend("decode", b=one)) and passes(attend(b=one)) and passes(append(b=one))
    assert passes(append(q=None, q_out=None)) and passes(append(cos=None, sin=None, rows=0))
    for c, d in ((F.F16, F.F32), (F.BF16, F.F32), (F.BF16, F.BF16)):
        assert passes(attend(c=kv(dtype=c), dtype=d)), (c, d)
    # nothing to do: buffers may be null
    for b in (batch(n_seqs=0, rows=0, row_start=None), batch(rows=0)):
        assert passes(attend(b=b, q=None, out=None, work=None, work_bytes=0)) and passes(append(b=b, k=None, v=None))


BAD_CACHE = [(dict(dtype=F.F32), UNSUPPORTED), (dict(dtype=F.Q8_0), UNSUPPORTED), (dict(n_pages=0), INVALID),
             (dict(n_pages=1 << 31), INVALID), (dict(page_size=8), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED),
             (dict(page_size=0), UNSUPPORTED), (dict(page_size=2048), UNSUPPORTED), (dict(n_kv_heads=0), INVALID),
             (dict(n_kv_heads=3), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED),
             (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(k=P + 8), MISALIGNED), (dict(v=P + 2), MISALIGNED)]
BAD_BATCH = [(dict(row_start=None), INVALID), (dict(page_table=None), INVALID), (dict(kv_len=None), INVALID),
             (dict(kv_len=P + 2), MISALIGNED), (dict(row_start=P + 1), MISALIGNED), (dict(max_kv_len=65), INVALID),
             (dict(max_pages=1 << 28), UNSUPPORTED), (dict(rows=1 << 30), UNSUPPORTED),
             (dict(n_seqs=1 << 30), UNSUPPORTED), (dict(rows=(1 << 64) - 1), UNSUPPORTED)]


@pytest.mark.parametrize("how,code", BAD_CACHE)
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
                          (dict(ldo=256), INVALID), (dict(ldq=516), MISALIGNED), (dict(ldo=513), MISALIGNED),
                          (dict(q=P + 8), MISALIGNED), (dict(out=P + 4), MISALIGNED), (dict(ldq=1 << 31), INVALID),
                          (dict(n_heads=5), INVALID), (dict(n_heads=0), INVALID), (dict(n_heads=131072), INVALID),
                          (dict(dtype=F.F32, ldq=514), MISALIGNED), (dict(dtype=F.BF16), UNSUPPORTED),
                          (dict(dtype=F.Q8_0), UNSUPPORTED)]:
            assert attend(fn, b=b, **how) == code, (fn, how)
    assert attend("decode") == INVALID and b"row_start" in lib().frq_last_error()
    for how, code in [(dict(q=None), INVALID), (dict(q_out=None), INVALID), (dict(k=None), INVALID),
                      (dict(v=None), INVALID), (dict(cos=None), INVALID), (dict(sin=None), INVALID),
                      (dict(rows=0), INVALID), (dict(ldk=255), INVALID), (dict(ldv=260), MISALIGNED),
                      (dict(ldqo=128), INVALID), (dict(k=P + 8), MISALIGNED), (dict(cos=P + 4), MISALIGNED),
                      (dict(dtype=F.BF16), UNSUPPORTED)]:
        assert append(**how) == code, how


def test_null_structs_and_workspace():
    L = lib()
    assert L.frq_paged_attention_prefill(None, None, None, F.F16, 4, P, 512, 0.1, P, 0, P, 512) == INVALID
    assert L.frq_paged_attention_decode(None, None, None, F.F16, 4, P, 512, 0.1, P, 0, P, 512) == INVALID
    assert L.frq_paged_append(None, None, None, F.F16, 4, P, 512, P, 256, P, 256, P, P, 4, P, 512) == INVALID
    assert L.frq_paged_attention_workspace(None, None, 4) == 0
    c, b = kv(), batch(rows=3, row_start=None, max_pages=1 << 16)
    need = L.frq_paged_attention_workspace(C.byref(c), C.byref(b), 4)
    if need:
        assert attend("decode", b=b, work_bytes=need - 1) == WORKSPACE
        assert attend("decode", b=b, work=None, work_bytes=need) == INVALID
        assert attend("decode", b=b, work=P + 8, work_bytes=need) == MISALIGNED
        assert passes(attend("decode", b=b, work_bytes=need))


def test_python_wrappers_raise():
    with pytest.raises(F.FuelRocmError):
        F.PagedKvCache(None, 4, 16, 1, 64, k=P)


@pytest.mark.parametrize("ps", [16, 1024])
def test_positions_end_at_2_30(ps):
    most = (1 << 30) // ps
    one = dict(rows=3, row_start=None)
    for fn in ("decode", "prefill"):
        assert passes(attend(fn, c=kv(page_size=ps), b=batch(max_pages=most, **one)))
        assert attend(fn, c=kv(page_size=ps), b=batch(max_pages=most + 1, **one)) == UNSUPPORTED
    assert passes(append(c=kv(page_size=ps), b=batch(max_pages=most)))
    assert append(c=kv(page_size=ps), b=batch(max_pages=most + 1)) == UNSUPPORTED


HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_index_arithmetic_of_malformed_batches(tmp_path):
    """Pages, lengths and row ranges that are none lead no kernel out of the
    table, the pool or the rows (paged_index.cpp, the header's own functions)."""
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "paged_index.cpp")
    exe = str(tmp_path / "paged_index")
    subprocess.run([HIPCC, "-O1", "-std=c++17", "-x", "hip", "--offload-host-only", src, "-o", exe], check=True,
                   capture_output=True, timeout=300)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
