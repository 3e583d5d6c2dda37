"""The paged cache's host side without a GPU: sizes, struct layouts and the
refusals of the C entry points, which come before any CUDA call."""
import ctypes

import pytest
import torch

from kvq import _lib


def paged(**kw):
    d = dict(pool=4096, status=4096, num_pages=4, page_size=16, kv_heads=2, head_dim=128, bits=4,
             group_size=64, dtype=_lib.DTYPE_FLOAT16, device=0)
    d.update(kw)
    return _lib.Paged(**d)


def batch(**kw):
    d = dict(page_table=4096, table_stride=8, seq_lens=4096, cu_rows=4096, batch=2, max_pages=8,
             rows=5)
    d.update(kw)
    return _lib.PagedBatch(**d)


S2 = (ctypes.c_int64 * 2)(256, 128)


def append(p, b, rope=None, q=None, q_heads=0, qs=None, q_out=None, k=4096, v=4096):
    return _lib.lib().kvq_paged_append(ctypes.byref(p), ctypes.byref(b), k, v, S2, S2,
                                       ctypes.byref(rope) if rope else None, q, q_heads, qs,
                                       q_out, None)


def sdpa(p, b, decode=False, q=4096, q_heads=8, window=0, sinks=0, out=4096, scale=1.0):
    fn = _lib.lib().kvq_paged_sdpa_decode if decode else _lib.lib().kvq_paged_sdpa_prefill
    return fn(ctypes.byref(p), ctypes.byref(b), q, q_heads, S2, scale, window, sinks, out, None, 0,
              None)


def error():
    return _lib.lib().kvq_last_error().decode()


@pytest.mark.parametrize("d,bits,gs,want", [
    (128, 4, 64, 2304), (128, 8, 64, 4352), (64, 4, 32, 1280), (256, 8, 128, 8448),
])
def test_tile_bytes(d, bits, gs, want):
    n = ctypes.c_size_t()
    p = paged(pool=None, status=None, head_dim=d, bits=bits, group_size=gs)
    assert _lib.lib().kvq_paged_tile_bytes(ctypes.byref(p), ctypes.byref(n)) == 0
    assert n.value == want == 2 * 16 * (d * bits // 8 + d // gs * 4)


def test_struct_layouts():
    assert ctypes.sizeof(_lib.Paged) == 48
    assert ctypes.sizeof(_lib.PagedBatch) == 48
    assert ctypes.sizeof(_lib.RopeArgs) == 32


@pytest.mark.parametrize("kw,word", [
    (dict(pool=None), "pool"), (dict(pool=4100), "aligned"), (dict(status=None), "status"),
    (dict(num_pages=0), "num_pages"), (dict(kv_heads=0), "kv_heads"), (dict(page_size=8), "page_size"),
    (dict(page_size=48), "page_size"), (dict(page_size=512), "page_size"),
    (dict(head_dim=96), "head_dim"), (dict(bits=3), "bits"), (dict(group_size=16), "group_size"),
    (dict(head_dim=64, group_size=128), "group_size"), (dict(dtype=10), "dtype"),
])
def test_bad_pools(kw, word):
    for rc in (append(paged(**kw), batch()), sdpa(paged(**kw), batch())):
        assert rc == _lib.ERR_ARG
        assert word in error()


@pytest.mark.parametrize("kw,word", [
    (dict(batch=-1), "batch"), (dict(rows=-1), "rows"), (dict(max_pages=-1), "max_pages"),
    (dict(seq_lens=None), "seq_lens"), (dict(page_table=None), "page_table"),
    (dict(table_stride=7), "table_stride"), (dict(cu_rows=None), "rows must equal batch"),
    (dict(max_pages=1 << 28, table_stride=1 << 28), "2^31"),
])
def test_bad_batches(kw, word):
    for rc in (append(paged(), batch(**kw)), sdpa(paged(), batch(**kw))):
        assert rc == _lib.ERR_ARG
        assert word in error()


def test_bad_rope_and_queries():
    r = _lib.RopeArgs(3, 0, 1e4, 1.0, 1.0, None)
    assert append(paged(), batch(), r) == _lib.ERR_ARG and "dims" in error()
    r = _lib.RopeArgs(130, 0, 1e4, 1.0, 1.0, None)
    assert append(paged(), batch(), r) == _lib.ERR_ARG and "dims" in error()
    r = _lib.RopeArgs(64, 0, 0.0, 1.0, 1.0, None)
    assert append(paged(), batch(), r) == _lib.ERR_ARG and "base" in error()
    assert append(paged(), batch(), q=4096, q_heads=0, qs=S2, q_out=4096) == _lib.ERR_ARG
    assert append(paged(), batch(), q=4096, q_heads=8, qs=S2) == _lib.ERR_ARG
    # in place needs a contiguous q: 8 heads of 128 are 1024 elements a row
    assert append(paged(), batch(), q=4096, q_heads=8, qs=S2, q_out=4096) == _lib.ERR_ARG
    assert "in place" in error()
    assert append(paged(), batch(), k=None) == _lib.ERR_ARG


def test_bad_attention_arguments():
    assert sdpa(paged(), batch(), q_heads=3) == _lib.ERR_ARG and "q_heads" in error()
    assert sdpa(paged(), batch(), q_heads=0) == _lib.ERR_ARG
    assert sdpa(paged(), batch(), window=-1) == _lib.ERR_ARG and "window" in error()
    assert sdpa(paged(), batch(), sinks=-1) == _lib.ERR_ARG
    assert sdpa(paged(), batch(), q=None) == _lib.ERR_ARG
    assert sdpa(paged(), batch(), scale=float("nan")) == _lib.ERR_ARG and "scale" in error()
    assert sdpa(paged(), batch(), scale=float("inf")) == _lib.ERR_ARG
    assert sdpa(paged(), batch(), out=None) == _lib.ERR_ARG
    assert sdpa(paged(), batch(), decode=True) == _lib.ERR_ARG  # 5 rows, 2 sequences
    assert "rows must equal batch" in error()


def test_no_rows_is_no_work():
    assert append(paged(), batch(rows=0)) == 0
    assert sdpa(paged(), batch(rows=0)) == 0
    assert sdpa(paged(), batch(rows=0, batch=0), decode=True) == 0


def test_python_refusals():
    import kvq
    with pytest.raises(ValueError):
        kvq.PagedQuantizedKVCache(2, 16, 2, 64, 32, 4, torch.float16, device="cpu")
    with pytest.raises(TypeError):
        kvq.PagedQuantizedKVCache.pool_shape(2, 16, 2, 64, 32, 4, torch.float32)
    with pytest.raises(kvq.KvqError):
        kvq.PagedQuantizedKVCache.pool_shape(2, 24, 2, 64, 32, 4, torch.float16)
    assert kvq.PagedQuantizedKVCache.pool_shape(3, 32, 2, 128, 64, 4) == (3, 2, 2, 576)


def test_overlapping_table_rows_are_refused():
    # a table that one row is broadcast into has the row stride 0: its rows
    # must not be taken for max_pages apart, behind the end of its memory
    import kvq
    cache = object.__new__(kvq.PagedQuantizedKVCache)
    cache._index = -1  # the device index of CPU tensors; no launch follows
    lens = torch.zeros(3, dtype=torch.int32)
    for table, stride in ((torch.zeros(1, 8, dtype=torch.int32).expand(3, 8), 0),
                          (torch.zeros(16, dtype=torch.int32).as_strided((3, 8), (4, 1)), 4),
                          (torch.zeros(1, 1, dtype=torch.int32).expand(3, 1), 0)):
        b = cache._batch(3, table, lens, None)
        assert b.table_stride == stride
        assert sdpa(paged(), b, decode=True) != 0 and "table_stride" in error()
        assert append(paged(), b) != 0 and "table_stride" in error()
    b = cache._batch(3, torch.zeros(3, 24, dtype=torch.int32)[:, :8], lens, None)
    assert (b.table_stride, b.max_pages) == (24, 8)
