"""A paged key/value cache in 8 bits on the device, beside `ops.KVCache`: sequences of their own lengths whose tokens live in
pages, e4m3 codes with a power-of-two scale for each page and head (the format is described with `smc_paged_kv` in the C
header).  The reference's caches are contiguous (SharpMind.Model/IKVCache.cs); this one has no counterpart there.

The memory is three tensors of the caller's (`PagedKVCache.create` makes them), and which page belongs to which
sequence is the caller's too: every call takes the page table, the lengths (new tokens included) and, where sequences have
other than one row each, the rows' starts, all int32 tensors on the device.  No call waits for the device, and a captured
CUDA graph serves whatever these tensors hold when it is replayed.
"""
from __future__ import annotations

import ctypes as C

from . import ops


class _Kv(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("scales", C.c_void_p), ("pages", C.c_int), ("kv_heads", C.c_int), ("page", C.c_int),
                ("head_dim", C.c_int)]


class _Seqs(C.Structure):
    _fields_ = [("table", C.c_void_p), ("lengths", C.c_void_p), ("row_start", C.c_void_p), ("batch", C.c_int), ("width", C.c_int), ("rows", C.c_int)]


def _require(ok: bool, text: str):
    if not ok:
        raise ops.ArgumentException(text)


class PagedKVCache:
    """Pages of one attention layer: `k` [pages, kv_heads, page, head_dim] and `v` [pages, kv_heads, head_dim, page] float8_e4m3fn,
    `scales` [pages, kv_heads, 2] float32.  Work on the same pages goes to one stream, or is ordered by events."""

    def __init__(self, ctx: "ops.CudaContext", k, v, scales):
        import torch

        self.torch, self.ctx = torch, ctx
        _require(k.dim() == 4 and v.dim() == 4, "codes have four dimensions")
        self.pages, self.kv_heads, self.page, self.head_dim = k.shape
        if self.page not in (16, 32, 64):
            raise ops.NotSupportedException(f"pages of 16, 32 or 64 tokens, not {self.page}")
        if self.head_dim not in (64, 128):
            raise ops.NotSupportedException(f"heads of 64 or 128, not {self.head_dim}")
        _require(v.shape == (self.pages, self.kv_heads, self.head_dim, self.page), "values are [pages, kv_heads, head_dim, page]")
        _require(scales.shape == (self.pages, self.kv_heads, 2), "scales are [pages, kv_heads, 2]")
        _require(k.dtype == v.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32, "codes are float8_e4m3fn, scales float32")
        _require(k.is_contiguous() and v.is_contiguous() and scales.is_contiguous(), "the cache's tensors are contiguous")
        self.device = k.device
        _require(k.is_cuda and k.device == v.device == scales.device and k.device.index == ctx.device, "the cache lives on the context's device")
        self.k, self.v, self.scales = k, v, scales
        self._kv = _Kv(k.data_ptr(), v.data_ptr(), scales.data_ptr(), *k.shape)
        self._types = {torch.float32: 0, torch.bfloat16: 30}

    @classmethod
    def create(cls, ctx: "ops.CudaContext", pages: int, kv_heads: int, head_dim: int, page: int = 64) -> "PagedKVCache":
        import torch

        dev = torch.device("cuda", ctx.device)
        k = torch.zeros((pages, kv_heads, page, head_dim), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        v = torch.zeros((pages, kv_heads, head_dim, page), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        return cls(ctx, k, v, torch.zeros((pages, kv_heads, 2), dtype=torch.float32, device=dev))

    def _stream(self):
        return self.torch._C._cuda_getCurrentRawStream(self.ctx.device)

    def _type(self, x):
        t = self._types.get(x.dtype)
        if t is None:
            raise ops.NotSupportedException(f"activations of {x.dtype} (float32 and bfloat16 are served)")
        return t

    def _rows(self, x, heads, like, name):
        """Row stride of x [rows, heads, head_dim], whose rows may lie apart."""
        _require(x.dim() == 3 and x.shape[2] == self.head_dim and (heads is None or x.shape[1] == heads), f"{name} is [rows, heads, {self.head_dim}]")
        _require(x.device == self.device and x.dtype == like.dtype and x.shape[0] == like.shape[0], f"{name} is of another device, type or number of rows")
        _require((x.stride(2) == 1 and x.stride(1) == self.head_dim) or x.numel() == 0, f"the heads of a row of {name} are contiguous")
        return x.stride(0) if x.shape[0] > 1 else x.shape[1] * self.head_dim

    def _seqs(self, table, lengths, row_start, rows):
        i32 = self.torch.int32
        _require(table.dim() == 2 and table.dtype == i32 and table.is_contiguous() and table.device == self.device, "table is a contiguous int32 [batch, width] on the cache's device")
        batch, width = table.shape
        _require(lengths.shape == (batch,) and lengths.dtype == i32 and lengths.is_contiguous() and lengths.device == self.device, "lengths is an int32 [batch] on the cache's device")
        if row_start is None:
            _require(rows == batch, f"{rows} rows for {batch} sequences of one row")
            return _Seqs(table.data_ptr(), lengths.data_ptr(), None, batch, width, rows)
        _require(row_start.shape == (batch + 1,) and row_start.dtype == i32 and row_start.is_contiguous() and row_start.device == self.device,
                 "row_start is an int32 [batch + 1] on the cache's device")
        return _Seqs(table.data_ptr(), lengths.data_ptr(), row_start.data_ptr(), batch, width, rows)

    def Update(self, k, v, table, lengths, row_start=None, cos=None, sin=None, neox: bool = True, q=None, q_out=None):
        """Appends k, v [rows, kv_heads, head_dim], the last rows of every sequence.  With cos, sin [positions, rope_dim / 2] the keys are rotated to
        their positions on the way, and so are the queries q [rows, heads, head_dim]: returned in `q_out` (a new tensor without one)."""
        t, type_ = self.torch, self._type(k)
        ks, vs = self._rows(k, self.kv_heads, k, "k"), self._rows(v, self.kv_heads, k, "v")
        seqs = self._seqs(table, lengths, row_start, k.shape[0])
        _require((cos is None) == (sin is None), "cos and sin come together")
        half = rows_of = 0
        if cos is not None:
            _require(cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == t.float32 and cos.is_contiguous() and sin.is_contiguous()
                     and cos.device == sin.device == self.device, "cos and sin are contiguous float32 [positions, rope_dim / 2] on the cache's device")
            rows_of, half = cos.shape
            _require(0 < half <= self.head_dim // 2 and half % 4 == 0 and rows_of > 0, f"rotation of {2 * half} of {self.head_dim} dimensions: a multiple of 8 is served")
        qs = heads = 0
        if q is not None:
            qs, heads = self._rows(q, None, k, "q"), q.shape[1]
            if q_out is None:
                q_out = t.empty(q.shape, dtype=q.dtype, device=q.device)
            _require(q_out.shape == q.shape and q_out.dtype == q.dtype and q_out.device == q.device and q_out.is_contiguous(), "q_out is contiguous and of q's shape and type")
            _require(q_out.data_ptr() != q.data_ptr() or q.is_contiguous(), "queries in place are contiguous rows")
        rc = self.ctx.lib.smc_paged_update_dev(self.ctx.h, C.byref(self._kv), C.byref(seqs), type_, k.data_ptr(), ks, v.data_ptr(), vs,
                                               None if q is None else q.data_ptr(), qs, None if q is None else q_out.data_ptr(), heads,
                                               None if cos is None else cos.data_ptr(), None if sin is None else sin.data_ptr(), 2 * half, rows_of,
                                               1 if neox else 0, self._stream())
        if rc:
            self.ctx.check(rc)
        return q_out if q is not None else None

    def attention(self, q, table, lengths, scale: float, row_start=None, max_rows: int | None = None, max_len: int | None = None, window: int = 0, out=None):
        """Causal attention of q [rows, heads, head_dim], the last rows of every sequence, over the sequences' pages; the same shape and type.
        window > 0: a position sees itself and the window - 1 before it.  max_rows, max_len: the most rows and tokens that a sequence
        has (all rows, and what the table holds, where they are not given)."""
        t, type_ = self.torch, self._type(q)
        qs = self._rows(q, None, q, "q")
        rows, heads, _ = q.shape
        _require(heads > 0 and heads % self.kv_heads == 0, f"{heads} query heads on {self.kv_heads} key/value heads")
        seqs = self._seqs(table, lengths, row_start, rows)
        if out is None:
            out = t.empty(q.shape, dtype=q.dtype, device=q.device)
        _require(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device and out.is_contiguous(), "out is contiguous and of q's shape and type")
        most = 1 if row_start is None else rows if max_rows is None else max_rows
        long = seqs.width * self.page if max_len is None else max_len
        lib = self.ctx.lib
        n = lib.smc_paged_attention_work(self.ctx.h, C.byref(self._kv), seqs.batch, rows, heads, most, long)
        _require(n >= 0, f"max_rows {most} and max_len {long} do not describe a call")
        work = t.empty(n, dtype=t.uint8, device=self.device) if n else None
        rc = lib.smc_paged_attention_dev(self.ctx.h, C.byref(self._kv), C.byref(seqs), type_, q.data_ptr(), qs, out.data_ptr(), heads, scale, window, most, long,
                                         work.data_ptr() if n else None, n, self._stream())
        if rc:
            self.ctx.check(rc)
        return out

    def read(self, pages, dtype=None):
        """(keys, values) of the listed pages (int32), [n, page, kv_heads, head_dim] float32 or bfloat16."""
        t = self.torch
        dtype = dtype or t.float32
        _require(pages.dim() == 1 and pages.dtype == t.int32 and pages.is_contiguous() and pages.device == self.device, "pages is an int32 [n] on the cache's device")
        if dtype not in self._types:
            raise ops.NotSupportedException(f"values as {dtype} (float32 and bfloat16 are served)")
        shape = (pages.shape[0], self.page, self.kv_heads, self.head_dim)
        k, v = t.empty(shape, dtype=dtype, device=self.device), t.empty(shape, dtype=dtype, device=self.device)
        rc = self.ctx.lib.smc_paged_read_dev(self.ctx.h, C.byref(self._kv), pages.data_ptr(), pages.shape[0], self._types[dtype], k.data_ptr(), v.data_ptr(), self._stream())
        if rc:
            self.ctx.check(rc)
        return k, v
