"""Attention over a paged key-value cache.

`PagedAttention` is the paged counterpart of `CUDAAttention`: the same options,
but the keys and values of all sequences live in one pool of fixed-size pages
that the caller allocates and hands out. A step is `append` (rotation and
append, returns the rotated queries) and `decode`; a long context may be read
sparsely with `select` between the two:

    layer = PagedAttention(hidden, heads, max_tokens, key_pages, value_pages, options, key_bounds=bounds)
    layer.append(prompt_qkv, starts, table, row_offsets=offsets)     # prompts, any lengths
    q = layer.append(qkv, positions, table)                          # one new token each
    out = layer.decode(q, positions, table)
    out = layer.decode(q, positions, table, pages=layer.select(q, positions, table, 64))
"""
import ctypes

import numpy as np
import torch

from . import _abi
from ._abi import check, lib
from .attention import Context, _ptr, attn_config

_IO_FLAGS = {torch.float16: 0, torch.bfloat16: _abi.FLAG_IO_BF16, torch.float32: _abi.FLAG_IO_FP32}
_PAGE_FLAGS = {torch.float16: 0, torch.bfloat16: _abi.FLAG_CACHE_BF16, torch.float32: _abi.FLAG_CACHE_FP32}


class PagedAttention:
    """One attention layer over a page pool.

    key_pages, value_pages: CUDA tensors of equal shape and strides,
    [pages, kvHeadCount, pageSize, headDim], or with the option `pageLayout`
    "NHD" [pages, pageSize, kvHeadCount, headDim]; float16, bfloat16 or
    float32, the last dimension dense. pageSize is a power of two up to 1024.
    key_bounds: None or a contiguous [pages, kvHeadCount, 2, headDim] tensor of
    the pages' type; `append` keeps each page's smallest and largest keys in
    it, and `select` needs it.
    options: the AttentionKernelOptions keys as for CUDAAttention (no gateNode,
    positionNode or sharedAttention), `dtype` (qkv, query, gate and out: the
    pages' type, or float32; default the pages' type), `maxBatch` (default
    1024) and `pageLayout` ("HND" or "NHD").

    The tensors stay the caller's; the layer holds references to them. Calls
    allocate only their outputs and a workspace, on the stream they run on.
    Page table, position and page-list conventions: include/tla_api.h.
    """

    def __init__(self, hidden_size, head_count, max_tokens, key_pages, value_pages, options=None, key_bounds=None,
                 context=None):
        o = dict(options or {})
        self.handle = None
        self.hiddenSize = hidden_size
        self.headCount = head_count
        self.headDim = o.get("headDim") or hidden_size // head_count
        self.kvHeadCount = o.get("kvHeadCount") or head_count
        self.maxTokens = max_tokens
        self.maxBatch = int(o.get("maxBatch", 1024))
        self.qSize = self.headCount * self.headDim
        self.rowSize = (self.headCount + 2 * self.kvHeadCount) * self.headDim
        self.pageLayout = o.get("pageLayout", "HND")
        if self.pageLayout not in ("HND", "NHD"):
            raise ValueError(f"pageLayout must be 'HND' or 'NHD', not {self.pageLayout!r}")
        k, v = key_pages, value_pages
        if k.dtype not in _PAGE_FLAGS or v.dtype != k.dtype:
            raise TypeError("key_pages and value_pages must both be float16, bfloat16 or float32")
        if not k.is_cuda or v.device != k.device:
            raise TypeError("key_pages and value_pages must be CUDA tensors on one device")
        if k.dim() != 4 or v.shape != k.shape or v.stride() != k.stride():
            raise ValueError("key_pages and value_pages must be 4-dimensional with equal shapes and strides")
        head_at, slot_at = (1, 2) if self.pageLayout == "HND" else (2, 1)
        if k.shape[head_at] != self.kvHeadCount or k.shape[3] != self.headDim:
            raise ValueError(f"pages {tuple(k.shape)} are not {self.kvHeadCount} kv heads of {self.headDim} "
                             f"({self.pageLayout})")
        if k.stride(3) != 1 and k.shape[3] != 1:
            raise ValueError("the last dimension of the pages must be dense")
        self.dtype = o.get("dtype") or k.dtype
        if self.dtype not in _IO_FLAGS:
            raise TypeError("dtype must be float16, bfloat16 or float32")
        self.pageSize = k.shape[slot_at]
        self.device = k.device
        if key_bounds is not None:
            if key_bounds.dtype != k.dtype or key_bounds.device != k.device or not key_bounds.is_contiguous():
                raise TypeError("key_bounds must be a contiguous tensor of the pages' type and device")
            if tuple(key_bounds.shape) != (k.shape[0], self.kvHeadCount, 2, self.headDim):
                raise ValueError("key_bounds must be [pages, kvHeadCount, 2, headDim]")
        self.keyPages, self.valuePages, self.keyBounds = k, v, key_bounds
        self.context = context or Context.default(self.device.index or 0)
        if self.context.device != (self.device.index or 0):
            raise ValueError("the context and the pages are on different devices")
        cfg = attn_config(o, self.headCount, self.kvHeadCount, self.headDim, max_tokens, self.maxBatch)
        cfg.flags |= _IO_FLAGS[self.dtype] | _PAGE_FLAGS[k.dtype]
        pool = _abi.PagePool()
        pool.key, pool.value = k.data_ptr(), v.data_ptr()
        pool.bounds = None if key_bounds is None else key_bounds.data_ptr()
        pool.page_stride, pool.head_stride, pool.slot_stride = k.stride(0), k.stride(head_at), k.stride(slot_at)
        pool.page_count, pool.page_size = k.shape[0], self.pageSize
        norms = []
        for key in ("qNormWeight", "kNormWeight"):
            w = None if o.get(key) is None else np.ascontiguousarray(o[key], np.float32)
            if w is not None and w.shape != (self.headDim,):
                raise ValueError(f"{key} must have headDim values")
            norms.append(w)
        self.qNormAttribute, self.kNormAttribute = norms
        h = ctypes.c_void_p()
        check(lib().tla_paged_create(self.context.handle, ctypes.byref(cfg), ctypes.byref(pool),
                                     *(None if w is None else w.ctypes.data_as(ctypes.c_void_p) for w in norms),
                                     ctypes.byref(h)), "PagedAttention constructor")
        self.handle = h
        self._workspace_bytes = {}

    # ---- argument checks
    def _rows(self, t, name, rows, width):
        if t.dtype != self.dtype or t.device != self.device or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous {self.dtype} tensor on {self.device}")
        if t.numel() != rows * width:
            raise ValueError(f"{name} must hold {rows} rows of {width} values, not shape {tuple(t.shape)}")

    def _ints(self, t, name, shape):
        if t.dtype != torch.int32 or t.device != self.device or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous int32 tensor on {self.device}")
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")

    def _sequences(self, positions, page_table):
        """(batch, table width) of a call."""
        if positions.dim() != 1 or page_table.dim() != 2:
            raise ValueError("positions must be [batch] and page_table [batch, width]")
        batch, width = positions.shape[0], page_table.shape[1]
        self._ints(positions, "positions", (batch,))
        self._ints(page_table, "page_table", (batch, width))
        return batch, width

    def _on(self, stream):
        """The stream of a call, and the context that makes tensors on it."""
        if stream is None:
            return torch.cuda.current_stream(self.device)
        if stream.device != self.device:
            raise ValueError("the stream and the pages are on different devices")
        return stream

    def _new(self, shape, dtype, stream):
        if stream == torch.cuda.current_stream(self.device):
            return torch.empty(shape, dtype=dtype, device=self.device)
        with torch.cuda.stream(stream):
            return torch.empty(shape, dtype=dtype, device=self.device)

    def _workspace(self, batch, width, stream):
        n = self._workspace_bytes.get((batch, width))
        if n is None:
            size = ctypes.c_size_t()
            check(lib().tla_paged_workspace(self.handle, batch, width, ctypes.byref(size)), "workspace")
            n = self._workspace_bytes[batch, width] = size.value
        return self._new((n,), torch.uint8, stream)

    # ---- the operators
    def append(self, qkv, positions, page_table, row_offsets=None, query=None, stream=None):
        """Append rows of packed [Q | K | V]; returns the rotated queries [rows, headCount * headDim].

        qkv [rows, (headCount + 2*kvHeadCount) * headDim]. Without row_offsets, row b is
        sequence b's new token at positions[b]. With it (int32 [batch + 1]), rows
        row_offsets[b] .. row_offsets[b+1]-1 are sequence b's tokens from positions[b] on."""
        s = self._on(stream)
        batch, width = self._sequences(positions, page_table)
        rows = qkv.shape[0]
        self._rows(qkv, "qkv", rows, self.rowSize)
        if row_offsets is None:
            if rows != batch:
                raise ValueError(f"{rows} rows for {batch} sequences need row_offsets")
        else:
            self._ints(row_offsets, "row_offsets", (batch + 1,))
        if query is None:
            query = self._new((rows, self.qSize), self.dtype, s)
        else:
            self._rows(query, "query", rows, self.qSize)
        check(lib().tla_paged_append(self.handle, _ptr(qkv), _ptr(positions), _ptr(row_offsets), _ptr(page_table),
                                     width, batch, rows, _ptr(query), ctypes.c_void_p(s.cuda_stream)), "append")
        return query

    def decode(self, query, positions, page_table, pages=None, gate=None, out=None, stream=None):
        """Attention of one new token per sequence: query [batch, headCount * headDim] as append
        returned it; pages None, or int32 [batch, kvHeadCount, count] as select returned them."""
        s = self._on(stream)
        batch, width = self._sequences(positions, page_table)
        self._rows(query, "query", batch, self.qSize)
        count = 0
        if pages is not None:
            count = pages.shape[-1]
            if count == 0:  # (an empty tensor's null address would read as no list)
                raise _abi.TlaError(-1, "decode: pages lists nothing")
            self._ints(pages, "pages", (batch, self.kvHeadCount, count))
        if gate is not None:
            self._rows(gate, "gate", batch, self.qSize)
        if out is None:
            out = self._new((batch, self.qSize), self.dtype, s)
        else:
            self._rows(out, "out", batch, self.qSize)
        work = self._workspace(batch, width, s)
        check(lib().tla_paged_decode(self.handle, _ptr(query), _ptr(positions), _ptr(page_table), width, _ptr(pages),
                                     count, _ptr(gate), _ptr(out), batch, _ptr(work), work.numel(),
                                     ctypes.c_void_p(s.cuda_stream)), "decode")
        return out

    def select(self, query, positions, page_table, count, first=1, last=1, pages=None, stream=None):
        """The `count` pages per sequence and kv head that decode should read: the first `first`,
        the last `last` and the best scored of the others; int32 [batch, kvHeadCount, count]."""
        s = self._on(stream)
        batch, width = self._sequences(positions, page_table)
        self._rows(query, "query", batch, self.qSize)
        count = int(count)
        if pages is None:
            pages = self._new((batch, self.kvHeadCount, max(count, 0)), torch.int32, s)
        else:
            self._ints(pages, "pages", (batch, self.kvHeadCount, count))
        work = self._workspace(batch, width, s)
        check(lib().tla_paged_select(self.handle, _ptr(query), _ptr(positions), _ptr(page_table), width, int(first),
                                     int(last), _ptr(pages), count, batch, _ptr(work), work.numel(),
                                     ctypes.c_void_p(s.cuda_stream)), "select")
        return pages

    def close(self):
        if self.handle:
            lib().tla_paged_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
