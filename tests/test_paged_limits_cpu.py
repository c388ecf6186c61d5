"""Refusals of the paged KV cache entry points at the ends of their ranges, and the
bounds that their grids and workspaces are sized by."""
import ctypes as C

import pytest

import fuel_amd as F
from fuel_amd._native import lib
from test_paged_cpu import INVALID, UNSUPPORTED, WORKSPACE, append, attend, batch, kv, passes


def test_append_in_place_keeps_its_rows_apart():
    for b in (batch(), batch(rows=3, row_start=None)):
        assert append(b=b, ldq=520, ldqo=512) == INVALID and b"in place" in lib().frq_last_error()
        assert append(b=b, ldq=512, ldqo=520) == INVALID
        assert passes(append(b=b, ldq=520, ldqo=520))
        assert passes(append(b=b, q=1 << 20, q_out=1 << 21, ldq=520, ldqo=512))


def test_launches_end_below_2_32_threads():
    """A row a workgroup of 256 threads in an append, a tile a workgroup or (short
    walks) a wavefront in an attention call: HIP's grids end below 2^32 threads."""
    most = (1 << 24) - 1
    for n, row_start in ((most, None), (most, 1 << 20)):
        b = dict(n_seqs=n, rows=n, row_start=row_start)
        assert passes(append(b=batch(**b)))
        b = dict(n_seqs=n, rows=n + 1, row_start=row_start) if row_start else dict(b, n_seqs=n + 1, rows=n + 1)
        assert append(b=batch(**b)) == UNSUPPORTED
    one = dict(c=kv(n_kv_heads=1), n_heads=1, ldq=128, ldo=128)
    for n, code in ((most, None), (most + 1, UNSUPPORTED)):  # 512 keys: four wavefronts a tile
        rc = attend("decode", b=batch(n_seqs=n, rows=n, max_pages=32, row_start=None), **one)
        assert rc == code or code is None and passes(rc)
    for n, code in ((4 * most, None), (4 * most + 1, UNSUPPORTED)):  # 32 keys: one
        rc = attend("decode", b=batch(n_seqs=n, rows=n, max_pages=2, row_start=None), **one)
        assert rc == code or code is None and passes(rc)
    rows = (1 << 31) - 1 - 1024
    for n, code in ((8, None), (9, UNSUPPORTED), (1024, UNSUPPORTED)):  # 128-row tiles: rows / 128 + n
        rc = attend(b=batch(n_seqs=n, rows=rows, max_pages=1 << 20), **one)
        assert rc == code or code is None and passes(rc), n


@pytest.mark.parametrize("heads,n_seqs,pages", [(4, 1, 100), (4, 3, 1 << 16), (32, 64, 512), (64, 128, 128)])
def test_long_decodes_need_a_workspace(heads, n_seqs, pages):
    c, b = kv(), batch(n_seqs=n_seqs, rows=n_seqs, row_start=None, max_pages=pages)
    need = lib().frq_paged_attention_workspace(C.byref(c), C.byref(b), heads)
    assert need > 0
    ld = heads * 128
    for fn in ("decode", "prefill"):
        assert attend(fn, b=b, n_heads=heads, ldq=ld, ldo=ld, work_bytes=need - 1) == WORKSPACE
        assert attend(fn, b=b, n_heads=heads, ldq=ld, ldo=ld, work=None, work_bytes=need) == INVALID
        assert passes(attend(fn, b=b, n_heads=heads, ldq=ld, ldo=ld, work_bytes=need))
    short = batch(n_seqs=n_seqs, rows=n_seqs, row_start=None, max_pages=pages, max_kv_len=200)
    assert lib().frq_paged_attention_workspace(C.byref(c), C.byref(short), heads) == 0


@pytest.mark.parametrize("new,past", [(16384, 0), (300, 6000)])
def test_long_prompts_in_tiles(new, past):
    """Whole tiles need no workspace, cut ones do."""
    c = kv(n_kv_heads=8)
    b = batch(n_seqs=1, rows=new, max_pages=(new + past + 15) // 16)
    need = lib().frq_paged_attention_workspace(C.byref(c), C.byref(b), 32)
    assert (need > 0) == (past > 0)
    if past:
        assert attend(c=c, b=b, n_heads=32, ldq=4096, ldo=4096, work_bytes=need - 1) == WORKSPACE
    assert passes(attend(c=c, b=b, n_heads=32, ldq=4096, ldo=4096, work_bytes=need))
