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
from .attention import Context, attn_config

_IO_FLAGS = {torch.float16: 0, torch.bfloat16: _abi.FLAG_IO_BF16, torch.float32: _abi.FLAG_IO_FP32}
_PAGE_FLAGS = {torch.float16: 0, torch.bfloat16: _abi.FLAG_CACHE_BF16, torch.float32: _abi.FLAG_CACHE_FP32}


def _current_raw_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


# the same handle without a Stream object around it, where this PyTorch offers it
_current_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_raw_stream)


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
        self._index = self.device.index
        self._lib = lib()
        self.context = context or Context.default(self._index)
        if self.context.device != self._index:
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
        check(self._lib.tla_paged_create(self.context.handle, ctypes.byref(cfg), ctypes.byref(pool),
                                     *(None if w is None else w.ctypes.data_as(ctypes.c_void_p) for w in norms),
                                     ctypes.byref(h)), "PagedAttention constructor")
        self.handle = h
        self._workspace_bytes = {}

    # ---- argument checks (a step makes several calls per layer: each check is a few attribute reads)
    def _rows(self, t, name, rows, width):
        if t.dtype is not self.dtype or t.get_device() != self._index or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous {self.dtype} tensor on {self.device}")
        if t.numel() != rows * width:
            raise ValueError(f"{name} must hold {rows} rows of {width} values, not shape {tuple(t.shape)}")

    def _ints(self, t, name, shape):
        if t.dtype is not torch.int32 or t.get_device() != self._index or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous int32 tensor on {self.device}")
        if t.shape != shape:
            raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")

    def _sequences(self, positions, page_table):
        """(batch, table width) of a call."""
        try:
            (batch,), (rows, width) = positions.shape, page_table.shape
        except ValueError:
            raise ValueError("positions must be [batch] and page_table [batch, width]") from None
        if (positions.dtype is not torch.int32 or page_table.dtype is not torch.int32
                or positions.get_device() != self._index or page_table.get_device() != self._index
                or not positions.is_contiguous() or not page_table.is_contiguous() or rows != batch):
            self._ints(positions, "positions", (batch,))
            self._ints(page_table, "page_table", (batch, width))
        return batch, width

    def _on(self, stream):
        """The raw stream of a call: the current one of the pages' device, or the given one."""
        if stream is None:
            return _current_raw_stream(self._index)
        if stream.device != self.device:
            raise ValueError("the stream and the pages are on different devices")
        return stream.cuda_stream

    @staticmethod
    def _new(like, shape, stream, dtype=None):
        """A dense tensor on `like`'s device that belongs to the call's stream."""
        if stream is None:
            return like.new_empty(shape) if dtype is None else like.new_empty(shape, dtype=dtype)
        with torch.cuda.stream(stream):
            return like.new_empty(shape, dtype=dtype or like.dtype)

    def _workspace(self, like, batch, width, count, which, stream):
        """(the tensor that keeps it, its address, its size) of a call's workspace; which: 0 decode, 1 select."""
        sizes = self._workspace_bytes.get((batch, width, count))
        if sizes is None:
            d, s = ctypes.c_size_t(), ctypes.c_size_t()
            check(self._lib.tla_paged_workspace(self.handle, batch, width, count, ctypes.byref(d), ctypes.byref(s)),
                  "workspace")
            if len(self._workspace_bytes) >= 4096:
                self._workspace_bytes.clear()
            sizes = self._workspace_bytes[batch, width, count] = (d.value, s.value)
        size = sizes[which]
        if size == 0:
            return None, None, 0
        work = self._new(like, size, stream, torch.uint8)
        return work, work.data_ptr(), size

    # ---- the operators
    def append(self, qkv, positions, page_table, row_offsets=None, query=None, stream=None):
        """Append rows of packed [Q | K | V]; returns the rotated queries [rows, headCount * headDim].

        qkv [rows, (headCount + 2*kvHeadCount) * headDim]. Without row_offsets, row b is
        sequence b's new token at positions[b]. With it (int32 [batch + 1]), rows
        row_offsets[b] .. row_offsets[b+1]-1 are sequence b's tokens from positions[b] on."""
        on = self._on(stream)
        batch, width = self._sequences(positions, page_table)
        rows = qkv.shape[0]
        self._rows(qkv, "qkv", rows, self.rowSize)
        offsets = None
        if row_offsets is not None:
            self._ints(row_offsets, "row_offsets", (batch + 1,))
            offsets = row_offsets.data_ptr()
        elif rows != batch:
            raise ValueError(f"{rows} rows for {batch} sequences need row_offsets")
        if query is None:
            n = self.qSize  # (the strides given: a quicker call)
            query = qkv.new_empty_strided((rows, n), (n, 1)) if stream is None else self._new(qkv, (rows, n), stream)
        else:
            self._rows(query, "query", rows, self.qSize)
        rc = self._lib.tla_paged_append(self.handle, qkv.data_ptr(), positions.data_ptr(), offsets,
                                        page_table.data_ptr(), width, batch, rows, query.data_ptr(), on)
        if rc:
            check(rc, "append")
        return query

    def decode(self, query, positions, page_table, pages=None, gate=None, out=None, stream=None):
        """Attention of one new token per sequence: query [batch, headCount * headDim] as append
        returned it; pages None, or int32 [batch, kvHeadCount, count] as select returned them.
        The output has the query's shape."""
        on = self._on(stream)
        batch, width = self._sequences(positions, page_table)
        self._rows(query, "query", batch, self.qSize)
        listed, count = None, 0
        if pages is not None:
            count = pages.shape[-1]
            if count == 0:  # (an empty tensor's null address would read as no list)
                raise _abi.TlaError(-1, "decode: pages lists nothing")
            self._ints(pages, "pages", (batch, self.kvHeadCount, count))
            listed = pages.data_ptr()
        if gate is not None:
            self._rows(gate, "gate", batch, self.qSize)
            gate = gate.data_ptr()
        if out is None:
            out = torch.empty_like(query) if stream is None else self._new(query, query.shape, stream)
        else:
            self._rows(out, "out", batch, self.qSize)
        work, at, size = self._workspace(query, batch, width, count, 0, stream)
        rc = self._lib.tla_paged_decode(self.handle, query.data_ptr(), positions.data_ptr(), page_table.data_ptr(),
                                        width, listed, count, gate, out.data_ptr(), batch, at, size, on)
        if rc:
            check(rc, "decode")
        return out

    def select(self, query, positions, page_table, count, first=1, last=1, pages=None, stream=None):
        """The `count` pages per sequence and kv head that decode should read: the first `first`,
        the last `last` and the best scored of the others; int32 [batch, kvHeadCount, count]."""
        on = self._on(stream)
        batch, width = self._sequences(positions, page_table)
        self._rows(query, "query", batch, self.qSize)
        count = int(count)
        if pages is None:
            h, n = self.kvHeadCount, max(count, 0)
            pages = (query.new_empty_strided((batch, h, n), (h * n, n, 1), dtype=torch.int32) if stream is None
                     else self._new(query, (batch, h, n), stream, torch.int32))
        else:
            self._ints(pages, "pages", (batch, self.kvHeadCount, count))
        work, at, size = self._workspace(query, batch, width, 0, 1, stream)
        rc = self._lib.tla_paged_select(self.handle, query.data_ptr(), positions.data_ptr(), page_table.data_ptr(),
                                        width, int(first), int(last), pages.data_ptr(), count, batch, at, size, on)
        if rc:
            check(rc, "select")
        return pages

    def close(self):
        if self.handle:
            self._lib.tla_paged_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
