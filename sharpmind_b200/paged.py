"""A paged key/value cache in 8 bits on the device, beside `ops.KVCache`: sequences of their own lengths whose tokens live in
pages, e4m3 codes with a power-of-two scale for each page and head (the format is described with `smc_paged_kv` in the C
header).  The reference's caches are contiguous (SharpMind.Model/IKVCache.cs); this one has no counterpart there.

The memory is three tensors of the caller's (`PagedKVCache.create` makes them), and which page belongs to which
sequence is the caller's too: every call takes the page table, the lengths (new tokens included) and, where sequences have
other than one row each, the rows' starts, all int32 tensors on the device.  A sequence of length 0 is an empty slot: `Update` writes
nothing for its rows and passes their queries on as they are, `attention` gives them zeros.  No call waits for the device, and a captured
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


def _require(ok: bool, text: str, error=ops.ArgumentException):
    if not ok:
        raise error(text)


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
        self._kv_ref, self._index = C.byref(self._kv), ctx.device
        self._types = {torch.float32: 0, torch.bfloat16: 30}

    @classmethod
    def create(cls, ctx: "ops.CudaContext", pages: int, kv_heads: int, head_dim: int, page: int = 64) -> "PagedKVCache":
        import torch

        dev = torch.device("cuda", ctx.device)
        k = torch.zeros((pages, kv_heads, page, head_dim), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        v = torch.zeros((pages, kv_heads, head_dim, page), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        return cls(ctx, k, v, torch.zeros((pages, kv_heads, 2), dtype=torch.float32, device=dev))

    # A call of few rows is bound by the host, so each method looks at its arguments in one expression of attribute reads; the text of what
    # is wrong with them is found afterwards.
    def _stream(self):
        return self.torch._C._cuda_getCurrentRawStream(self.ctx.device)

    def _rows_ok(self, x, heads, rows, dtype):
        return (x.dtype is dtype and x.shape == (rows, heads, self.head_dim) and x.get_device() == self._index
                and (x.is_contiguous() or (x.stride(2) == 1 and x.stride(1) == self.head_dim)))

    def _refuse_rows(self, x, heads, rows, dtype, name):
        _require(x.dtype in self._types, f"activations of {x.dtype} (float32 and bfloat16 are served)", ops.NotSupportedException)
        _require(x.dim() == 3 and x.shape[2] == self.head_dim and x.shape[1] == heads, f"{name} is [rows, {heads}, {self.head_dim}]")
        _require(x.get_device() == self._index and x.dtype is dtype and x.shape[0] == rows, f"{name} is of another device, type or number of rows")
        _require(self._rows_ok(x, heads, rows, dtype), f"the heads of a row of {name} are contiguous")

    def _seqs(self, table, lengths, row_start, rows):
        i32, index = self.torch.int32, self._index
        if not (table.dtype is i32 and table.dim() == 2 and table.is_contiguous() and table.get_device() == index):
            raise ops.ArgumentException("table is a contiguous int32 [batch, width] on the cache's device")
        batch, width = table.shape
        if not (lengths.dtype is i32 and lengths.shape == (batch,) and lengths.is_contiguous() and lengths.get_device() == index):
            raise ops.ArgumentException("lengths is an int32 [batch] on the cache's device")
        if row_start is None:
            if rows != batch:
                raise ops.ArgumentException(f"{rows} rows for {batch} sequences of one row")
            return _Seqs(table.data_ptr(), lengths.data_ptr(), None, batch, width, rows)
        if not (row_start.dtype is i32 and row_start.shape == (batch + 1,) and row_start.is_contiguous() and row_start.get_device() == index):
            raise ops.ArgumentException("row_start is an int32 [batch + 1] on the cache's device")
        return _Seqs(table.data_ptr(), lengths.data_ptr(), row_start.data_ptr(), batch, width, rows)

    def _out(self, out, q, name):
        """Where the rows of q go: contiguous, as q otherwise."""
        if out is None:
            return self.torch.empty_like(q, memory_format=self.torch.contiguous_format)
        if not (out.shape == q.shape and out.dtype is q.dtype and out.get_device() == self._index and out.is_contiguous()):
            raise ops.ArgumentException(f"{name} is contiguous and of q's shape and type")
        return out

    def Update(self, k, v, table, lengths, row_start=None, cos=None, sin=None, neox: bool = True, q=None, q_out=None):
        """Appends k, v [rows, kv_heads, head_dim], the last rows of every sequence.  With cos, sin [positions, rope_dim / 2] the keys are rotated to
        their positions on the way, and so are the queries q [rows, heads, head_dim]: returned in `q_out` (a new tensor without one)."""
        rows, dtype = k.shape[0], k.dtype
        for x, name in ((k, "k"), (v, "v")):
            if dtype not in self._types or not self._rows_ok(x, self.kv_heads, rows, dtype):
                self._refuse_rows(x, self.kv_heads, rows, dtype, name)
        seqs = self._seqs(table, lengths, row_start, rows)
        c = s = to = src = None
        half = positions = heads = stride = 0
        if cos is not None or sin is not None:
            _require(cos is not None and sin is not None, "cos and sin come together")
            f32, index = self.torch.float32, self._index
            if not (cos.dtype is f32 and sin.dtype is f32 and cos.dim() == 2 and cos.shape == sin.shape and cos.is_contiguous() and sin.is_contiguous()
                    and cos.get_device() == index and sin.get_device() == index):
                raise ops.ArgumentException("cos and sin are contiguous float32 [positions, rope_dim / 2] on the cache's device")
            positions, half = cos.shape
            if not (0 < half <= self.head_dim // 2 and half % 4 == 0 and positions > 0):
                raise ops.ArgumentException(f"rotation of {2 * half} of {self.head_dim} dimensions: a multiple of 8 is served")
            c, s = cos.data_ptr(), sin.data_ptr()
        if q is not None:
            heads = q.shape[1] if q.dim() == 3 else 0
            if not self._rows_ok(q, heads, rows, dtype):
                self._refuse_rows(q, heads, rows, dtype, "q")
            q_out = self._out(q_out, q, "q_out")
            src, to, stride = q.data_ptr(), q_out.data_ptr(), q.stride(0)
            if src == to and not q.is_contiguous():
                raise ops.ArgumentException("queries in place are contiguous rows")
        if rows == 0:
            return q_out
        wide = self.kv_heads * self.head_dim
        rc = self.ctx.lib.smc_paged_update_dev(self.ctx.h, self._kv_ref, C.byref(seqs), self._types[dtype], k.data_ptr(), k.stride(0) if rows > 1 else wide, v.data_ptr(),
                                               v.stride(0) if rows > 1 else wide, src, stride if rows > 1 else heads * self.head_dim, to, heads, c, s, 2 * half, positions,
                                               1 if neox else 0, self._stream())
        if rc:
            self.ctx.check(rc)
        return q_out

    def attention(self, q, table, lengths, scale: float, row_start=None, max_rows: int | None = None, max_len: int | None = None, window: int = 0, out=None):
        """Causal attention of q [rows, heads, head_dim], the last rows of every sequence, over the sequences' pages; the same shape and type.
        window > 0: a position sees itself and the window - 1 before it.  max_rows, max_len: the most rows and tokens that a sequence
        has (all rows, and what the table holds, where they are not given)."""
        rows, dtype = q.shape[0], q.dtype
        heads = q.shape[1] if q.dim() == 3 else 0
        if dtype not in self._types or not self._rows_ok(q, heads, rows, dtype):
            self._refuse_rows(q, heads, rows, dtype, "q")
        if heads == 0 or heads % self.kv_heads:
            raise ops.ArgumentException(f"{heads} query heads on {self.kv_heads} key/value heads")
        seqs = self._seqs(table, lengths, row_start, rows)
        out = self._out(out, q, "out")
        if rows == 0:
            return out
        most = 1 if row_start is None else rows if max_rows is None else max_rows
        long = seqs.width * self.page if max_len is None else max_len
        lib, h, kv = self.ctx.lib, self.ctx.h, self._kv_ref
        n = lib.smc_paged_attention_work(h, kv, seqs.batch, rows, heads, most, long)
        if n < 0:
            raise ops.ArgumentException(f"max_rows {most} and max_len {long} do not describe a call")
        # (of the caching allocator: a call's own until it has completed, on any stream and in any captured graph)
        work = self.torch.empty(n, dtype=self.torch.uint8, device=self.device) if n else None
        rc = lib.smc_paged_attention_dev(h, kv, C.byref(seqs), self._types[dtype], q.data_ptr(), q.stride(0) if rows > 1 else heads * self.head_dim, out.data_ptr(), heads,
                                         scale, window, most, long, work.data_ptr() if n else None, n, self._stream())
        if rc:
            self.ctx.check(rc)
        return out

    def read(self, pages, dtype=None):
        """(keys, values) of the listed pages (int32), [n, page, kv_heads, head_dim] float32 or bfloat16."""
        t = self.torch
        dtype = dtype or t.float32
        if not (pages.dtype is t.int32 and pages.dim() == 1 and pages.is_contiguous() and pages.get_device() == self._index):
            raise ops.ArgumentException("pages is an int32 [n] on the cache's device")
        if dtype not in self._types:
            raise ops.NotSupportedException(f"values as {dtype} (float32 and bfloat16 are served)")
        n = pages.shape[0]
        k = t.empty((n, self.page, self.kv_heads, self.head_dim), dtype=dtype, device=self.device)
        v = t.empty_like(k)
        rc = self.ctx.lib.smc_paged_read_dev(self.ctx.h, self._kv_ref, pages.data_ptr(), n, self._types[dtype], k.data_ptr(), v.data_ptr(), self._stream())
        if rc:
            self.ctx.check(rc)
        return k, v
