"""The paged key/value cache as a program holds it: torch tensors, described once to the library.

``KvCache`` is one layer's pool of pages and ``KvBatch`` the sequences of a step
(hc_kv_cache and hc_kv_batch of include/hayai_cuda.h); ``CudaEngine.kv_append_dev``,
``kv_read_dev`` and ``attn_paged_dev`` take both.  ``KvShared`` names the sequences of a batch that
share their first tokens, for ``attn_shared_dev``; ``KvPages`` is the bookkeeping of all layers' pools,
which ``kv_fork_dev``, ``kv_resize_dev`` and ``kv_compact_dev`` change; ``Rope`` says how queries and keys
are turned by their positions (``rope_dev``, ``kv_append_rope_dev``).  They keep references to their
tensors and no copies: a step that changes page numbers, lengths or offsets in place needs no new batch.
The reference keeps a sink-and-window INT8 cache of one sequence on the host
(crates/hayai-cpu/src/kv_cache.rs).
"""
from __future__ import annotations

import ctypes
import math

from . import _lib

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


class _Shared(ctypes.Structure):
    _fields_ = [("n_groups", ctypes.c_int), ("max_new", ctypes.c_int), ("least", ctypes.c_int64),
                ("seq_start", ctypes.c_void_p), ("length", ctypes.c_void_p)]


class _Pages(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("n_slots", "max_pages", "n_layers")] + \
               [("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_size_t)] + \
               [(n, ctypes.c_void_p) for n in ("kv_len", "refs", "scratch", "layers")]


class _Rope(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("layout", "head_dim", "rot_dim")] + \
               [("amplitude", ctypes.c_float), ("turns", ctypes.c_uint64 * 128)]


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


class KvShared:
    """Groups of a batch's sequences that share their first tokens: group g is the sequences
    seq_start[g] to seq_start[g + 1] (int32 [n_groups + 1]), whose first length[g] positions (int32
    [n_groups]) are the same, and are read by the pages of the first one that has new tokens.  max_new: a bound
    on any group's new tokens, where the program knows one.  least: how many tokens of reading the sharing has
    to save, over all groups, to be made (0: by the library's rule, which leaves it where it would be slower)."""

    def __init__(self, seq_start, length, max_new: int = 0, least: int = 0):
        torch = _torch()
        for t in (seq_start, length):
            _need(t.is_cuda and t.dtype == torch.int32 and t.dim() == 1 and t.device == seq_start.device,
                  "seq_start and length must be int32 CUDA tensors of one device and one axis")
            _need(t.shape[0] <= 1 or t.stride(0) == 1, "seq_start and length must be contiguous")
        _need(seq_start.shape[0] == length.shape[0] + 1, "length must hold n_groups and seq_start n_groups + 1")
        _need(max_new >= 0 and least >= 0, "max_new and least must not be negative")
        self._keep = (seq_start, length)
        self.index = seq_start.get_device()
        self.struct = _Shared(length.shape[0], min(max_new, 2**31 - 1), min(least, 2**62), seq_start.data_ptr(), length.data_ptr())
        self.ref = ctypes.addressof(self.struct)


class KvPages:
    """The bookkeeping of a pool that sequences share in every layer: caches, a KvCache for each layer, all
    of one shape; page_table int32 [n_slots][max_pages], kv_len int32 [n_slots] (the tokens that a slot
    holds, 0 for an unused one) and refs int32 [n_pages] (how many table entries in use name a page, 0
    for a free one).  The calls change the three in place; page_table and kv_len serve as a KvBatch's."""

    def __init__(self, caches, page_table, kv_len, refs):
        torch = _torch()
        caches = list(caches)
        _need(len(caches) > 0, "caches must hold at least one KvCache")
        for t, d in ((page_table, 2), (kv_len, 1), (refs, 1)):
            _need(t.is_cuda and t.dtype == torch.int32 and t.dim() == d and t.device == page_table.device,
                  "page_table, kv_len and refs must be int32 CUDA tensors of one device, of 2, 1 and 1 axes")
            _need(t.shape[-1] <= 1 or t.stride(-1) == 1, "page_table rows, kv_len and refs must be contiguous")
        n_slots, max_pages = page_table.shape
        self.index, self.n_pages, self.int32 = page_table.get_device(), caches[0].struct.n_pages, torch.int32
        _need(all(c.index == self.index for c in caches), "the caches must be on page_table's device")
        _need(kv_len.shape[0] == n_slots and refs.shape[0] == self.n_pages, "kv_len must hold n_slots and refs n_pages")
        stride = page_table.stride(0) if n_slots > 1 else max_pages
        _need(stride >= max_pages, "page_table rows overlap")
        size = ctypes.c_size_t()
        rc = _lib.lib().hc_kv_pages_scratch(self.n_pages, ctypes.byref(size))
        _need(rc == 0, "the caches hold no pages")
        scratch = torch.empty(size.value, dtype=torch.int32, device=page_table.device)
        layers = (_Cache * len(caches))(*[c.struct for c in caches])
        self._keep = (caches, page_table, kv_len, refs, scratch, layers)
        self.struct = _Pages(n_slots, max_pages, len(caches), page_table.data_ptr(), stride, kv_len.data_ptr(),
                             refs.data_ptr(), scratch.data_ptr(), ctypes.addressof(layers))
        self.ref = ctypes.addressof(self.struct)

    def items(self, a, b, what: str):
        """(n, pointers) of a call's two int32 arrays."""
        n = a.numel()
        for t in (a, b):
            if t.dtype is not self.int32 or t.dim() != 1 or t.numel() != n or t.get_device() != self.index or not t.is_contiguous():
                raise ValueError(f"{what} must be contiguous int32 tensors of one length on the pages' device")
        return n, a.data_ptr(), b.data_ptr()


class Rope:
    """Rotary positions: how the first rot_dim values of a head (0: all) are turned, in pairs (i, i + rot_dim / 2)
    (layout "half") or (2 i, 2 i + 1) ("pairs"), by the angles position * base^(-2 i / rot_dim) / factors[i].

    Longer contexts: ``factor`` alone divides every frequency (linear scaling).  With ``original``, the
    context that the model was trained with, a frequency that made r turns there is divided by bands: wholly
    where r <= low, not at all where r >= high, and in proportion between.  ``amplitude`` multiplies the
    turned values (0.1 ln factor + 1 with bands: YaRN).  factors: a sequence of rot_dim / 2 positive numbers,
    as a GGUF file's rope_freqs."""

    LAYOUTS = {"half": 0, "pairs": 1}

    def __init__(self, head_dim: int, rot_dim: int = 0, base: float = 10000.0, layout: str = "half", factor: float = 1.0,
                 original: float = 0, low: float = 0.0, high: float = 0.0, factors=None, amplitude: float = 1.0):
        _need(layout in self.LAYOUTS, f"layout must be one of {sorted(self.LAYOUTS)}")
        _need(math.isfinite(amplitude), "amplitude must be finite")
        rot_dim = rot_dim or head_dim
        given = None
        if factors is not None:
            factors = [float(f) for f in factors]
            _need(len(factors) == rot_dim // 2, "factors must hold rot_dim / 2 numbers")
            given = (ctypes.c_float * len(factors))(*factors)
        self.struct = _Rope()
        rc = _lib.lib().hc_rope_init(ctypes.addressof(self.struct), self.LAYOUTS[layout], head_dim, rot_dim, base, factor,
                                     original, low, high, given, amplitude)
        _need(rc == 0, _lib.lib().hc_last_error().decode(errors="replace"))
        self.ref = ctypes.addressof(self.struct)
        self.head_dim, self.rot_dim = head_dim, rot_dim

    def count(self, positions) -> int:
        """How many positions there are."""
        if positions.dtype is not _torch().int32 or positions.dim() != 1 or not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int32 tensor [n_tok]")
        return positions.numel()

    def rows(self, x, what: str, n: int, like=None):
        """(type id, heads, leading dimension) of packed rows x [n_tok][heads][head_dim]."""
        if not _ROW_TYPES:
            _torch()
        t = _ROW_TYPES.get(x.dtype)
        if t is None or not x.is_cuda or x.dim() != 3 or x.shape[0] != n or x.shape[2] != self.head_dim or \
                (like is not None and (x.shape != like.shape or x.dtype != like.dtype)):
            raise ValueError(f"{what} must be float32, float16 or bfloat16 [n_tok={n}][heads][head_dim={self.head_dim}] on the "
                             "engine's device, and rows that go together of one shape and type")
        ld, head, one = x.stride()
        heads = x.shape[1]
        if x.numel() and (one != 1 or (head != self.head_dim and heads > 1)):
            raise ValueError(f"{what} must have contiguous rows (only the token axis may be strided)")
        return t, heads, ld if n > 1 else heads * self.head_dim
