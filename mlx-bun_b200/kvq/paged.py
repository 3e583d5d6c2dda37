"""Paged quantized KV cache: pages shared by many sequences, over libkvq.

``PagedQuantizedKVCache`` holds a pool of pages in the caches' affine
quantized format (kvq_paged, include/kvq.h).  Which pages a sequence owns is
the caller's page table; lengths and row offsets are device arrays, so a CUDA
graph of ``append`` + ``sdpa_decode`` serves every later step.  The same
(page_table, seq_lens, cu_rows) describe a step to all calls: ``seq_lens``
counts each sequence's tokens with the step's rows included.  Rows of
``page_table`` may share pages but not memory (a broadcast row is refused).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import check, lib
from .cache import dtype_code

TILE_ROWS = 16
_I64x2 = ctypes.c_int64 * 2
_byref = ctypes.byref


@dataclass
class Rope:
    """Rotary embedding of the first `dims` elements of a row (kvq_rope):
    angle (scale * position) * base^(-2i / dims), or / freqs[i] (device f32
    [dims / 2]); pairs (i, i + dims / 2), or (2i, 2i + 1) when traditional;
    pre_scale multiplies the rotated elements."""
    dims: int
    base: float = 10000.0
    scale: float = 1.0
    traditional: bool = False
    freqs: torch.Tensor | None = None
    pre_scale: float = 1.0

    def _struct(self, device: torch.device) -> _lib.RopeArgs:
        f = self.freqs
        if f is not None and (f.dtype != torch.float32 or f.device != device or
                              not f.is_contiguous() or f.numel() != self.dims // 2):
            raise ValueError("rope freqs must be contiguous float32 [dims / 2] on the cache's device")
        return _lib.RopeArgs(self.dims, int(self.traditional), self.base, self.scale,
                             self.pre_scale, f.data_ptr() if f is not None else None)


class PagedQuantizedKVCache:
    """A pool of `num_pages` pages of `page_size` token rows for every kv head.

    ``pool`` is the int32 tensor [num_pages, kv_heads, page_size / 16,
    tile_words] that holds them (allocated zeroed, or the caller's own); see
    ``keys`` / ``values`` for its parts."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 group_size: int = 64, bits: int = 8, dtype: torch.dtype = torch.float16,
                 device=None, pool: torch.Tensor | None = None):
        if pool is not None:
            dev = pool.device
        else:
            dev = torch.device("cuda" if device is None else device) \
                if not isinstance(device, int) else torch.device("cuda", device)
        if dev.type != "cuda":
            raise ValueError("the pool must be on a CUDA device")
        index = torch.cuda.current_device() if dev.index is None else dev.index
        self.device = torch.device("cuda", index)
        self.num_pages, self.page_size = num_pages, page_size
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self.group_size, self.bits, self.dtype = group_size, bits, dtype
        self._c = _lib.Paged(None, None, num_pages, page_size, kv_heads, head_dim, bits,
                             group_size, dtype_code(dtype), index)
        self.shape = self.pool_shape(num_pages, page_size, kv_heads, head_dim, group_size, bits,
                                     dtype)
        if pool is None:
            pool = torch.zeros(self.shape, dtype=torch.int32, device=self.device)
        elif pool.dtype != torch.int32 or tuple(pool.shape) != self.shape or \
                not pool.is_contiguous():
            raise ValueError(f"pool must be a contiguous int32 tensor {self.shape}")
        self.pool = pool
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._c.pool, self._c.status = pool.data_ptr(), self._status.data_ptr()
        self._index, self._ref = index, _byref(self._c)
        self._ws_bytes = {}

    @staticmethod
    def pool_shape(num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                   group_size: int = 64, bits: int = 8, dtype: torch.dtype = torch.float16):
        """Shape of the int32 pool tensor these pages need."""
        c = _lib.Paged(None, None, num_pages, page_size, kv_heads, head_dim, bits, group_size,
                       dtype_code(dtype), 0)
        n = ctypes.c_size_t()
        check(lib().kvq_paged_tile_bytes(ctypes.byref(c), ctypes.byref(n)))
        return (num_pages, kv_heads, page_size // TILE_ROWS, n.value // 4)

    def _half(self, part: int):
        """Codes [pages, heads, tiles, 16, words] and (scale, bias) pairs
        [pages, heads, tiles, 16, groups, 2] of K (0) or V (1), as views."""
        w, g = self.head_dim * self.bits // 32, self.head_dim // self.group_size
        o = part * TILE_ROWS * (w + g)
        codes = self.pool[..., o:o + TILE_ROWS * w].unflatten(-1, (TILE_ROWS, w))
        o += TILE_ROWS * w
        pairs = self.pool[..., o:o + TILE_ROWS * g].unflatten(-1, (TILE_ROWS, g))
        return codes, pairs.view(self.dtype).unflatten(-1, (g, 2))

    @property
    def keys(self):
        return self._half(0)

    @property
    def values(self):
        return self._half(1)

    # ------------------------------------------------------------- a step --

    def _batch(self, rows: int, page_table, seq_lens, cu_rows) -> _lib.PagedBatch:
        i32, dev = torch.int32, self._index
        B, pages = seq_lens.shape[0], page_table.shape
        if page_table.dtype is not i32 or len(pages) != 2 or pages[0] != B or \
                page_table.get_device() != dev or (pages[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table must be int32 [batch, max_pages] with contiguous rows on "
                             "the cache's device")
        if seq_lens.dtype is not i32 or seq_lens.dim() != 1 or seq_lens.get_device() != dev or \
                not seq_lens.is_contiguous():
            raise ValueError("seq_lens must be contiguous int32 [batch] on the cache's device")
        cu = None
        if cu_rows is not None:
            if cu_rows.dtype is not i32 or cu_rows.dim() != 1 or cu_rows.shape[0] != B + 1 or \
                    cu_rows.get_device() != dev or not cu_rows.is_contiguous():
                raise ValueError("cu_rows must be contiguous int32 [batch + 1] on the cache's device")
            cu = cu_rows.data_ptr()
        return _lib.PagedBatch(page_table.data_ptr(), page_table.stride(0),
                               seq_lens.data_ptr(), cu, B, pages[1], rows)

    def _rows(self, x: torch.Tensor, name: str, heads: int | None = None):
        """Check token rows [rows, heads, head_dim]; returns (shape, strides)."""
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be [rows, {heads or 'heads'}, {self.head_dim}]")
        if x.dtype is not self.dtype or x.get_device() != self._index:
            raise ValueError(f"{name} must be {self.dtype} on {self.device}")
        s = x.stride()
        if s[2] != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
        return shape, _I64x2(s[0], s[1])

    def _like(self, x: torch.Tensor, shape, name: str):
        if x.shape != shape or x.dtype is not self.dtype or x.get_device() != self._index or \
                not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor like q")

    def _stream(self, stream):
        # the raw handle of torch's current stream (or the caller's)
        return torch._C._cuda_getCurrentRawStream(self._index) if stream is None else stream

    def append(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
               seq_lens: torch.Tensor, cu_rows: torch.Tensor | None = None,
               rope: Rope | None = None, q: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None, stream=None):
        """Write the step's rows k, v [rows, kv_heads, head_dim] (any row and
        head strides) into their pages: K rotated by `rope` at its position,
        both quantized (kvq_paged_append).  q [rows, q_heads, head_dim]: its
        rotated rows go to q_out (allocated when None; q itself to rotate a
        contiguous q in place, otherwise apart from q, k and v), which is
        returned.  Padding rows (from cu_rows[batch] on) are not touched: a
        fresh q_out holds anything there."""
        shape, ks = self._rows(k, "k", self.kv_heads)
        vshape, vs = self._rows(v, "v", self.kv_heads)
        rows = shape[0]
        if vshape[0] != rows:
            raise ValueError("k and v must have the same rows")
        batch = self._batch(rows, page_table, seq_lens, cu_rows)
        qh, qs, qp, op = 0, None, None, None
        if q is not None:
            qshape, qs = self._rows(q, "q")
            if qshape[0] != rows:
                raise ValueError("q and k must have the same rows")
            qh = qshape[1]
            if q_out is None:
                q_out = torch.empty(qshape, dtype=q.dtype, device=q.device)
            else:
                self._like(q_out, qshape, "q_out")
            qp, op = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out needs q")
        r = _byref(rope._struct(self.device)) if rope is not None else None
        rc = lib().kvq_paged_append(self._ref, _byref(batch), k.data_ptr(), v.data_ptr(), ks, vs, r,
                                    qp, qh, qs, op, self._stream(stream))
        if rc:
            check(rc)
        return q_out

    def _sdpa(self, fn, q, page_table, seq_lens, cu_rows, scale, window, sinks, out, workspace,
              stream):
        shape, qs = self._rows(q, "q")
        batch = self._batch(shape[0], page_table, seq_lens, cu_rows)
        if out is None:
            out = torch.empty(shape, dtype=q.dtype, device=q.device)
        else:
            self._like(out, shape, "out")
        ws, wsb = None, 0
        if workspace is not None:
            if workspace.get_device() != self._index or not workspace.is_contiguous():
                raise ValueError("workspace must be a contiguous tensor on the cache's device")
            ws, wsb = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        elif stream is None:
            # torch's allocator orders it on the current stream and gives a
            # captured graph memory of its own; the size goes by the shapes
            key = (cu_rows is None, shape[0], batch.batch, shape[1])
            wsb = self._ws_bytes.get(key)
            if wsb is None:
                if len(self._ws_bytes) >= 4096:  # a server meets ever new counts of rows
                    self._ws_bytes.clear()
                wsb = self._ws_bytes[key] = self._workspace(batch, shape[1], cu_rows is None)
            workspace = torch.empty(wsb, dtype=torch.uint8, device=self.device)
            ws = workspace.data_ptr()
        rc = fn(self._ref, _byref(batch), q.data_ptr(), shape[1], qs, scale, window, sinks,
                out.data_ptr(), ws, wsb, self._stream(stream))
        if rc:
            check(rc)
        return out

    def sdpa_decode(self, q: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                    scale: float, window: int = 0, sinks: int = 0,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                    stream=None) -> torch.Tensor:
        """Attention of one query row per sequence, q [batch, q_heads,
        head_dim], at the sequences' last positions (kvq_paged_sdpa_decode).
        window > 0: the last `window` keys and the first `sinks` ones.  `out`
        may be a contiguous q itself, otherwise lies apart from it.
        workspace None: the call's own, safe with calls on other streams."""
        return self._sdpa(lib().kvq_paged_sdpa_decode, q, page_table, seq_lens, None, scale, window,
                          sinks, out, workspace, stream)

    def sdpa_prefill(self, q: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                     cu_rows: torch.Tensor, scale: float, window: int = 0, sinks: int = 0,
                     out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                     stream=None) -> torch.Tensor:
        """Causal attention of ragged query rows, q [rows, q_heads, head_dim]:
        sequence b's rows are cu_rows[b]..cu_rows[b + 1] and end at its last
        position (kvq_paged_sdpa_prefill).  Padding rows are not touched: a
        fresh `out` holds anything there.  Beyond rows * q_heads / kv_heads = 64
        * batch (rows of the buffer, padding included) K, V and the
        probabilities are rounded to the dtype before their products; below, K
        is exact, as in sdpa_decode (errors: include/kvq.h)."""
        return self._sdpa(lib().kvq_paged_sdpa_prefill, q, page_table, seq_lens, cu_rows, scale,
                          window, sinks, out, workspace, stream)

    def workspace_bytes(self, rows: int, q_heads: int, page_table: torch.Tensor,
                        seq_lens: torch.Tensor, cu_rows: torch.Tensor | None = None) -> int:
        """Bytes a caller's workspace needs for sdpa_decode (cu_rows None) or
        sdpa_prefill of these shapes."""
        return self._workspace(self._batch(rows, page_table, seq_lens, cu_rows), q_heads,
                               cu_rows is None)

    def _workspace(self, batch, q_heads: int, decode: bool) -> int:
        n = ctypes.c_size_t()
        check(lib().kvq_paged_sdpa_workspace(self._ref, _byref(batch), q_heads, int(decode),
                                             _byref(n)))
        return n.value

    def check(self, stream=None):
        """Synchronize and raise if a call met a row without a place, a page
        number outside the pool or a length beyond the page table."""
        check(lib().kvq_paged_check(ctypes.byref(self._c), self._stream(stream)))
