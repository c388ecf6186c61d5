"""What the Python mirror of the paged KV cache refuses before a call."""
import numpy as np
import pytest

import fuel_amd as F
from fuel_amd.backend import RocmStorage

P = 1 << 20  # an address that nothing reads


class Dev:
    """A device that no call reaches."""

    def __init__(self, ordinal=0):
        self.ordinal = ordinal

    @property
    def handle(self):
        return None


def storage(nbytes, dtype=np.uint16, dev=None):
    """A storage of that many bytes, without device memory."""
    s = object.__new__(RocmStorage)
    s.dev, s.dtype, s.nbytes, s.ptr = dev or DEV, np.dtype(dtype), nbytes, P
    s.shape = (nbytes // s.dtype.itemsize,)
    s.free = lambda: None
    return s


DEV = Dev()


def refused(f, *a, **k):
    with pytest.raises(F.FuelRocmError) as e:
        f(*a, **k)
    assert e.value.status != 0
    return str(e.value)


@pytest.mark.parametrize("x", [np.array([P]), np.array(P), 1.5, "1048576", True, [P], np.zeros(4, np.float32)])
def test_operands_that_are_no_addresses(x):
    """Arrays and tensors of one element have an int() of their value."""
    refused(F.PagedKvCache, DEV, 9, 16, 2, 128, F.F16, x, P)
    for name in ("page_table", "kv_len", "row_start"):
        refused(F.PagedBatch, **dict(dict(page_table=P, kv_len=P, n_seqs=3, max_pages=4, row_start=P), **{name: x}))
    cache, one = F.PagedKvCache(DEV, 9, 16, 2, 128, F.F16, P, P), F.PagedBatch(P, P, 3, 4)
    for name in ("q", "k", "v", "q_out", "rope_cos", "rope_sin"):
        a = dict(q=P, k=P, v=P, q_out=P, rope_cos=P, rope_sin=P)
        a[name] = x
        refused(F.paged_append, cache, one, F.F16, 4, rope_rows=4, **a)
    for fn in (F.paged_attention_decode, F.paged_attention_prefill):
        refused(fn, cache, one, F.F16, 4, x, P, 0.1)
        refused(fn, cache, one, F.F16, 4, P, x, 0.1)


def test_addresses_reach_the_library():
    cache, one = F.PagedKvCache(DEV, 9, 16, 2, 128, F.F16, np.int64(P), P), F.PagedBatch(P, np.uint64(P), 3, 4)
    assert cache.struct.k == P and one.struct.kv_len == P and one.struct.row_start is None
    assert "null device handle" in refused(F.paged_append, cache, one, F.F16, 4, P, P, P, P)


def test_workspace_is_a_storage_or_an_address_of_so_many_bytes():
    cache, one = F.PagedKvCache(DEV, 9, 16, 2, 128, F.F16, P, P), F.PagedBatch(P, P, 3, 1 << 16)
    need = F.paged_attention_workspace(cache, one, 4)
    assert need > 0
    for fn in (F.paged_attention_decode, F.paged_attention_prefill):
        args = (cache, one, F.F16, 4, P, P, 0.1)
        for work in (None, P, storage(need - 1, np.uint8)):
            assert "workspace" in refused(fn, *args, work)
        assert "workspace" in refused(fn, *args, P, work_bytes=need - 1)
        refused(fn, *args, np.zeros(need, np.uint8), work_bytes=need)
        assert "null device handle" in refused(fn, *args, P, work_bytes=need)
        assert "null device handle" in refused(fn, *args, storage(need, np.uint8))


def short(f, name, *a, **k):
    assert f": {name}: " in ": " + refused(f, *a, **k)


def test_storages_shorter_than_a_call_reaches():
    """q of 5 rows, 528 elements apart, 4 heads of 128; k and v of 2 heads."""
    H, hk, D, n, ld = 4, 2, 128, 5, 528
    pool = 9 * hk * 16 * D * 2
    for i in range(2):
        kv = [storage(pool), storage(pool)]
        kv[i] = storage(pool - 2)
        short(F.PagedKvCache, "kv"[i], DEV, 9, 16, hk, D, F.F16, *kv)
    cache = F.PagedKvCache(DEV, 9, 16, hk, D, F.F16, storage(pool), storage(pool))
    good = dict(page_table=storage(4 * 3 * 4, np.int32), kv_len=storage(4 * 3, np.int32), row_start=storage(4 * 4, np.int32))
    for name, s in good.items():
        short(F.PagedBatch, name, n_seqs=3, max_pages=4, rows=n, **dict(good, **{name: storage(s.nbytes - 4, np.int32)}))
        short(F.PagedBatch, name, n_seqs=3, max_pages=4, rows=n, **dict(good, **{name: storage(2 * s.nbytes, np.int64)}))
    batch = F.PagedBatch(n_seqs=3, max_pages=4, rows=n, **good)
    for dtype, size in ((F.F16, 2), (F.F32, 4)):
        wide, narrow, table = ((n - 1) * ld + H * D) * size, ((n - 1) * ld + hk * D) * size, 4 * 64 * D
        ops = dict(q=storage(wide), k=storage(narrow), v=storage(narrow), q_out=storage(wide),
                   rope_cos=storage(table, np.float32), rope_sin=storage(table, np.float32))
        lds = dict(ldq=ld, ldk=ld, ldv=ld, ldqo=ld, rope_rows=64)
        assert "null device handle" in refused(F.paged_append, cache, batch, dtype, H, **ops, **lds)
        for name, s in ops.items():
            short(F.paged_append, name, cache, batch, dtype, H, **dict(ops, **{name: storage(s.nbytes - 4, s.dtype)}), **lds)
        short(F.paged_append, "rope_cos", cache, batch, dtype, H, **dict(ops, rope_cos=storage(2 * table, np.float64)), **lds)
        q, work = storage(wide), storage(1 << 20, np.uint8)
        a = (cache, batch, dtype, H)
        assert "null device handle" in refused(F.paged_attention_prefill, *a, q, q, 0.1, work, ldq=ld, ldo=ld)
        short(F.paged_attention_prefill, "q", *a, storage(wide - 2), q, 0.1, work, ldq=ld, ldo=ld)
        short(F.paged_attention_prefill, "out", *a, q, storage(wide - 2), 0.1, work, ldq=ld, ldo=ld)
        one = F.PagedBatch(P, P, n, 4)
        assert "null device handle" in refused(F.paged_attention_decode, cache, one, dtype, H, q, q, 0.1, work, ldq=ld, ldo=ld)
        short(F.paged_attention_decode, "q", cache, one, dtype, H, storage(wide - 2), q, 0.1, work, ldq=ld, ldo=ld)
        short(F.paged_attention_decode, "out", cache, one, dtype, H, q, storage(wide - 2), 0.1, work, ldq=ld, ldo=ld)
    # a batch of no rows reaches none
    none = F.PagedBatch(storage(0, np.int32), storage(0, np.int32), 0, 0)
    assert "null device handle" in refused(F.paged_attention_decode, cache, none, F.F16, H, storage(0), storage(0), 0.1)


def test_storages_of_another_device():
    other, big = Dev(1), 1 << 20
    refused(F.PagedKvCache, DEV, 9, 16, 2, 128, F.F16, storage(big, dev=other), storage(big))
    refused(F.PagedBatch, storage(big, np.int32), storage(big, np.int32, other), 3, 4)
    cache = F.PagedKvCache(DEV, 9, 16, 2, 128, F.F16, P, P)
    one, far = F.PagedBatch(P, P, 3, 4), F.PagedBatch(storage(big, np.int32, other), P, 3, 4)
    here, there = storage(big), storage(big, dev=other)
    assert "device 1" in refused(F.paged_attention_decode, cache, far, F.F16, 4, here, here, 0.1)
    assert "device 1" in refused(F.paged_append, cache, far, F.F16, 4, here, here, here, here)
    for i in range(2):
        ops = [here, here]
        ops[i] = there
        assert "device 1" in refused(F.paged_attention_prefill, cache, one, F.F16, 4, *ops, 0.1)
    assert "device 1" in refused(F.paged_attention_prefill, cache, one, F.F16, 4, here, here, 0.1, there)
    for i in range(4):
        ops = [here] * 4
        ops[i] = there
        assert "device 1" in refused(F.paged_append, cache, one, F.F16, 4, *ops)
