"""The paged key/value cache as a program holds it: torch tensors, described once to the library.

``KvCache`` is one layer's pool of pages and ``KvBatch`` the sequences of a step
(hc_kv_cache and hc_kv_batch of include/hayai_cuda.h); ``CudaEngine.kv_append_dev``,
``kv_read_dev`` and ``attn_paged_dev`` take both.  They keep references to their tensors and
no copies: a step that changes page numbers, lengths or offsets in place needs no new batch.
The reference keeps a sink-and-window INT8 cache of one sequence on the host
(crates/hayai-cpu/src/kv_cache.rs).
"""
from __future__ import annotations

import ctypes

F32, F16, I8, BF16 = 0, 1, 24, 30  # GgmlType ids
_ROW_TYPES, _CACHE_TYPES = {}, {}  # by torch's types: the package imports without torch, descriptions need it


def _torch():
    import torch

    if not _ROW_TYPES:
        _ROW_TYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
        _CACHE_TYPES.update({torch.float16: F16, torch.bfloat16: BF16, torch.int8: I8})
    return torch


class _Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("type", "n_pages", "n_heads", "page_size", "head_dim")] + \
               [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + \
               [(n, ctypes.c_size_t) for n in ("page_stride", "head_stride", "row_stride", "scale_page_stride")]


class _Batch(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("n_seq", "n_tok", "max_new", "max_pages")] + \
               [("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_size_t), ("q_start", ctypes.c_void_p),
                ("kv_len", ctypes.c_void_p)]


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class KvCache:
    """One layer's pages: k and v [n_pages][n_heads][page_size][head_dim] of float16, bfloat16, or
    int8 codes with float32 scales [n_pages][n_heads][page_size] (value = code * scale).  The page,
    head and row axes may be strided (views of a larger pool, or another order), by whole 64 bytes;
    of the scales only the page axis."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        torch = _torch()
        _need(k.is_cuda and v.is_cuda and k.device == v.device, "k and v must be CUDA tensors of one device")
        _need(k.dtype in _CACHE_TYPES and v.dtype == k.dtype, "k and v must both be float16, bfloat16 or int8")
        _need(k.dim() == 4 and v.shape == k.shape, "k and v must be [n_pages][n_heads][page_size][head_dim]")
        _need(k.stride(3) == 1 and v.stride() == k.stride(), "k and v need equal strides, 1 along head_dim")
        n_pages, n_heads, page_size, head_dim = k.shape
        if k.dtype == torch.int8:
            for s in (k_scale, v_scale):
                _need(s is not None and s.dtype == torch.float32 and s.device == k.device and s.shape == k.shape[:3],
                      "int8 pages need float32 scales [n_pages][n_heads][page_size]")
                _need((page_size == 1 or s.stride(2) == 1) and (n_heads == 1 or s.stride(1) == page_size)
                      and s.stride(0) == k_scale.stride(0), "scales may be strided along pages only, both alike")
        else:
            _need(k_scale is None and v_scale is None, "scales belong to int8 pages")
        # the stride of an axis of one page, head or row is not used: any whole stride will do
        strides = [s if n > 1 else max(64, head_dim) for s, n in zip(k.stride(), k.shape)]
        _need(all(s >= 0 for s in strides), "negative strides")
        self._keep = (k, v, k_scale, v_scale)
        self.index, self.n_heads, self.head_dim = k.get_device(), n_heads, head_dim
        self.default_scale = float(head_dim) ** -0.5 if head_dim else 0.0
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.struct = _Cache(_CACHE_TYPES[k.dtype], n_pages, n_heads, page_size, head_dim, ptr(k), ptr(v), ptr(k_scale),
                             ptr(v_scale), *strides[:3],
                             0 if k_scale is None else max(k_scale.stride(0), n_heads * page_size if n_pages == 1 else 0))
        self.ref = ctypes.addressof(self.struct)

    def rows(self, batch, x, heads: int, what: str):
        """(type id, leading dimension) of packed rows x [n_tok][heads][head_dim]."""
        t = _ROW_TYPES.get(x.dtype)
        if t is None or x.shape != (batch.n_tok, heads, self.head_dim) or x.get_device() != self.index:
            raise ValueError(f"{what} must be float32, float16 or bfloat16 [n_tok={batch.n_tok}][heads={heads}]"
                             f"[head_dim={self.head_dim}] on the cache's device")
        ld, head, one = x.stride()
        if one != 1 or (head != self.head_dim and heads > 1):
            raise ValueError(f"{what} must have contiguous rows (only the token axis may be strided)")
        return t, ld if batch.n_tok > 1 else heads * self.head_dim

    def pair(self, batch, k, v):
        """Arguments (type, k, ldk, v, ldv) of the new tokens' key and value rows."""
        t, ldk = self.rows(batch, k, self.n_heads, "k")
        tv, ldv = self.rows(batch, v, self.n_heads, "v")
        if tv != t:
            raise ValueError("k and v need one type")
        return t, k.data_ptr(), ldk, v.data_ptr(), ldv

    def lse_ptr(self, lse, q):
        if lse is None:
            return None
        if _ROW_TYPES.get(lse.dtype) != F32 or lse.shape != q.shape[:2] or not lse.is_contiguous() or lse.get_device() != self.index:
            raise ValueError("lse must be a contiguous float32 tensor [n_tok][n_heads] on q's device")
        return lse.data_ptr()


class KvBatch:
    """The sequences of a step: page_table int32 [n_seq][max_pages], q_start int32 [n_seq + 1]
    (sequence s has rows q_start[s] to q_start[s + 1] of the n_tok packed rows), kv_len int32
    [n_seq] (its tokens in the cache, the new ones included).  max_new: a bound on any sequence's
    new tokens, where the program knows one (1 when decoding)."""

    def __init__(self, page_table, q_start, kv_len, n_tok: int, max_new: int = 0):
        torch = _torch()
        for t, d in ((page_table, 2), (q_start, 1), (kv_len, 1)):
            _need(t.is_cuda and t.dtype == torch.int32 and t.dim() == d and t.device == page_table.device,
                  "page_table, q_start and kv_len must be int32 CUDA tensors of one device, of 2, 1 and 1 axes")
            _need(t.shape[-1] <= 1 or t.stride(-1) == 1, "page_table rows, q_start and kv_len must be contiguous")
        n_seq, max_pages = page_table.shape
        _need(kv_len.shape[0] == n_seq and q_start.shape[0] == n_seq + 1, "kv_len must hold n_seq and q_start n_seq + 1")
        _need(n_tok >= 0 and max_new >= 0, "n_tok and max_new must not be negative")
        self._keep = (page_table, q_start, kv_len)
        self.n_tok, self.index = int(n_tok), page_table.get_device()
        stride = page_table.stride(0) if n_seq > 1 else max_pages
        _need(stride >= max_pages, "page_table rows overlap")
        self.struct = _Batch(n_seq, n_tok, max_new, max_pages, page_table.data_ptr(), stride, q_start.data_ptr(),
                             kv_len.data_ptr())
        self.ref = ctypes.addressof(self.struct)
