"""The paged key/value cache of a decoder layer's attention half, over the C ABI.

The reference keeps one contiguous cache per sequence and computes a layer's attention from it
(engine/src/model.rs:900-1116; on Metal ``attn_prep``, ``attn_split_*`` and ``attn_flash*``,
engine/src/metal/kernels.metal:959-1573).  Here the tokens of all requests share pages, and three
calls stand beside ``Moe`` so that a layer's rows stay on the device:

``extend``  pages, slots and positions for a step's new tokens, from the requests' lengths
``store``   rotary positions on q and k; k and v into their pages
``attend``  attention of each request's new tokens over its pages

Pools, tables and lengths are torch tensors of the caller on the cache's device; every call runs on
the current torch stream, waits for nothing and can be captured into a graph.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import NamedTuple, Optional, Sequence

import torch

from . import capi

# bivmoe_extend_args, bivmoe_store_args and bivmoe_attend_args field by field (native order, C's alignment)
_ROWS, _POOL = "Pqqii", "Pqqqq"
_EXTEND = struct.Struct("6Pq4i6P").pack_into
_STORE = struct.Struct(_ROWS * 4 + _POOL * 2 + "2Pq2i").pack_into
_ATTEND = struct.Struct(_ROWS * 2 + _POOL * 2 + "Pq4i2Pf3i").pack_into
_GGML = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


class Rope:
    """Rotary positions: the head's first ``n_rot`` values turn by position * base^(-2i / n_rot), the
    pairs shared out over one to four axes of positions.  ``sections``: pairs of each axis (default:
    one axis with all); ``interleaved``: pair i belongs to axis i % axes as long as that axis has pairs
    left, instead of the axes' pairs following one another; ``adjacent``: a pair is neighbours,
    instead of half of ``n_rot`` apart."""

    def __init__(self, n_rot: int, base: float = 10000.0, sections: Optional[Sequence[int]] = None,
                 interleaved: bool = False, adjacent: bool = False):
        self.n_rot, self.base, self.interleaved, self.adjacent = n_rot, float(base), interleaved, adjacent
        self.sections = list(sections) if sections is not None else [n_rot // 2]
        if not 1 <= len(self.sections) <= 4:
            raise ValueError("one to four axes")


class Step(NamedTuple):
    """What ``PagedCache.extend`` leaves for the calls of a step (device tensors)."""
    length: torch.Tensor      # [n_seq] int32: past + added
    first: torch.Tensor       # [n_seq + 1] int32: first row of each request, and their number
    slots: torch.Tensor       # [n_tokens] int64: page * page_size + place, -1 without a page
    positions: torch.Tensor   # [n_tokens] int32
    left: torch.Tensor        # [2] int32: free pages that remain, pages that were missing
    held: torch.Tensor        # [n_seq] int32: pages of each request


class PagedCache:
    """Geometry and workspace of the calls.  Pools are [pages, page_size, n_head_kv, head_dim] tensors
    of ``dtype`` (views with other orders of the first three in memory too)."""

    def __init__(self, n_head: int, n_head_kv: int, head_dim: int, page_size: int, max_seqs: int, max_tokens: int,
                 dtype: torch.dtype = torch.bfloat16, rope: Optional[Rope] = None, device: int = 0):
        self._h = None
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("a cache is float16 or bfloat16")
        d = capi.CacheDesc()
        d.ggml_type, d.n_head, d.n_head_kv, d.head_dim = _GGML[dtype], n_head, n_head_kv, head_dim
        d.page_size, d.max_seqs, d.max_tokens, d.device = page_size, max_seqs, max_tokens, device
        if rope is not None:
            d.n_rot, d.rope_axes, d.rope_base = rope.n_rot, len(rope.sections), rope.base
            d.rope_interleaved, d.rope_adjacent = int(rope.interleaved), int(rope.adjacent)
            for i, s in enumerate(rope.sections):
                d.rope_sections[i] = s
        h = C.c_void_p()
        capi.check(capi.lib().bivmoe_cache_create(C.byref(d), C.byref(h)))
        self._h = h
        self.n_head, self.n_head_kv, self.head_dim, self.page_size = n_head, n_head_kv, head_dim, page_size
        self.max_seqs, self.max_tokens, self.dtype, self.rope, self.device = max_seqs, max_tokens, dtype, rope, device
        self._set_up(torch.device("cuda", device))

    def _set_up(self, dev):
        self._dev = dev
        L = capi.lib()
        self._calls = L.bivmoe_cache_extend, L.bivmoe_cache_store, L.bivmoe_cache_attend
        self._scale = 1.0 / math.sqrt(self.head_dim)
        # A call's arguments are packed anew for every launch, into a buffer of the struct's size; a step
        # of small kernels is bound by the host, so one pack and few attribute look-ups.
        self._bufs = [C.create_string_buffer(C.sizeof(t)) for t in (capi.ExtendArgs, capi.StoreArgs, capi.AttendArgs)]
        self._refs = [C.cast(b, C.POINTER(t)) for b, t in zip(self._bufs, (capi.ExtendArgs, capi.StoreArgs, capi.AttendArgs))]
        self._ggml = _GGML[self.dtype]
        self._pool_shape = (self.page_size, self.n_head_kv, self.head_dim)
        self._axes = len(self.rope.sections) if self.rope is not None else 0

    def close(self):
        if self._h is not None:
            capi.lib().bivmoe_cache_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _call(self, i, pack, *values):
        pack(self._bufs[i], 0, *values)
        code = self._calls[i](self._h, self._refs[i], torch.cuda.current_stream(self._dev).cuda_stream)
        if code:
            capi.check(code)

    def _ints(self, t, what, n, dtype=torch.int32):
        if t.dtype is not dtype or t.device != self._dev or not t.is_contiguous() or t.numel() < n:
            raise ValueError(f"{what}: {n} contiguous {dtype} on {self._dev} are wanted")
        return t.data_ptr()

    def pools(self, n_pages: int):
        """A layer's k and v pools."""
        shape = (n_pages, self.page_size, self.n_head_kv, self.head_dim)
        return tuple(torch.empty(shape, dtype=self.dtype, device=self._dev) for _ in range(2))

    def _table(self, t, n_seq):
        """address, stride, width"""
        if t.dtype is not torch.int32 or t.device != self._dev or t.dim() != 2:
            raise ValueError("table: [n_seq, pages] int32 is wanted")
        rows, width = t.shape
        stride, one = t.stride()
        if rows < n_seq or (width > 1 and one != 1):
            raise ValueError("table: [n_seq, pages] with neighbouring pages is wanted")
        return t.data_ptr(), stride, width

    def _pool(self, t, name):
        """address, strides of a page, a token and a head, pages: a ``bivmoe_pool``"""
        shape, stride = t.shape, t.stride()
        if t.dtype is not self.dtype or t.device != self._dev or shape[1:] != self._pool_shape or stride[3] != 1:
            raise ValueError(f"{name}: [pages, {self.page_size}, {self.n_head_kv}, {self.head_dim}] of {self.dtype} is wanted")
        return t.data_ptr(), stride[0], stride[1], stride[2], shape[0]

    def _rows(self, t, what, heads, n):
        """address, strides of a token and a head"""
        stride = t.stride()
        if t.shape != (n, heads, self.head_dim) or stride[2] != 1 or t.device != self._dev:
            raise ValueError(f"{what}: [tokens, {heads}, {self.head_dim}] rows on {self._dev} are wanted")
        return t.data_ptr(), stride[0], stride[1]

    def _out(self, out, q):
        if out is None:
            return torch.empty_like(q, dtype=self.dtype)
        if out.dtype is not self.dtype:
            raise ValueError(f"out: {self.dtype} is wanted")
        return out

    def extend(self, past, added, free_pages, free_count, table, n_tokens: int, held=None, out: Optional[Step] = None) -> Step:
        """Pages for ``added[b]`` new tokens of each request b, which has ``past[b]`` (int32 device
        tensors).  Takes them from the end of the free list (``free_pages[:free_count]``), writes the
        new entries of ``table`` [n_seq, pages], and returns the step.  ``n_tokens`` rows are laid out:
        more than the requests add (a padded batch) have slot -1.  ``held``: pages each request holds
        already, where that is not what ``past`` needs (drafted tokens that were taken back); ``out``:
        a step to write into."""
        n_seq = past.numel()
        if out is None:
            room = torch.empty(3 * n_seq + 3 + n_tokens, dtype=torch.int32, device=self._dev)
            length, first, left, kept, positions = room.split((n_seq, n_seq + 1, 2, n_seq, n_tokens))
            out = Step(length, first, torch.empty(n_tokens, dtype=torch.int64, device=self._dev), positions, left, kept)
            wrote = [t.data_ptr() for t in (length, first, positions, left, kept, out.slots)]
        else:
            wrote = [self._ints(out.length, "length", n_seq), self._ints(out.first, "first", n_seq + 1),
                     self._ints(out.positions, "positions", n_tokens), self._ints(out.left, "left", 2),
                     self._ints(out.held, "held", n_seq), self._ints(out.slots, "slots", n_tokens, torch.int64)]
        self._call(0, _EXTEND, self._ints(past, "past", n_seq), self._ints(added, "added", n_seq),
                   0 if held is None else self._ints(held, "held", n_seq), self._ints(free_pages, "free_pages", 0),
                   self._ints(free_count, "free_count", 1), *self._table(table, n_seq), free_pages.numel(), n_seq, n_tokens, *wrote)
        return out

    def store(self, q, k, v, k_pool, v_pool, slots, positions=None, out=None):
        """q and k [n, heads, head_dim] (float32, float16 or bfloat16; any strides of the first two)
        turned by ``positions`` ([n], or [axes, n]), k and v into the pages at ``slots``; returns the
        turned q in the cache's type."""
        n, ty = q.shape[0], _GGML.get(q.dtype)
        if ty is None or k.dtype is not q.dtype or v.dtype is not q.dtype:
            raise ValueError("q, k and v: rows of one type, float32, float16 or bfloat16, are wanted")
        out = self._out(out, q)
        where, stride = 0, 0
        if self._axes:
            if positions is None or positions.dtype is not torch.int32 or positions.device != self._dev or \
                    positions.numel() != self._axes * n or (n > 1 and positions.stride(-1) != 1):
                raise ValueError(f"positions: [{self._axes}, n] int32 are wanted" if self._axes > 1 else "positions: [n] int32 are wanted")
            where, stride = positions.data_ptr(), positions.stride(0) if positions.dim() > 1 else n
        kv = self.n_head_kv
        self._call(1, _STORE, *self._rows(q, "q", self.n_head, n), ty, 0, *self._rows(k, "k", kv, n), ty, 0,
                   *self._rows(v, "v", kv, n), ty, 0, *self._rows(out, "out", self.n_head, n), self._ggml, 0,
                   *self._pool(k_pool, "k_pool"), *self._pool(v_pool, "v_pool"),
                   self._ints(slots, "slots", n, torch.int64), where, stride, n, 0)
        return out

    def attend(self, q, k_pool, v_pool, table, first, length, max_new: int = 0, scale: Optional[float] = None,
               window: int = 0, sinks: int = 0, out=None):
        """Attention of the rows q [n, n_head, head_dim], request b's from first[b] to first[b + 1] - 1,
        the last tokens of its length[b] tokens.  A token at position p sees p and what is before it;
        with ``window`` the last ``window`` positions up to its own and the first ``sinks``.  ``max_new``:
        the most new rows of a request, where the caller knows it."""
        n, n_seq = q.shape[0], length.numel()
        if q.dtype is not self.dtype:
            raise ValueError(f"q: {self.dtype} is wanted")
        out = self._out(out, q)
        self._call(2, _ATTEND, *self._rows(q, "q", self.n_head, n), self._ggml, 0, *self._rows(out, "out", self.n_head, n), self._ggml, 0,
                   *self._pool(k_pool, "k_pool"), *self._pool(v_pool, "v_pool"), *self._table(table, n_seq), n_seq, n, max_new,
                   self._ints(first, "first", n_seq + 1), self._ints(length, "length", n_seq),
                   self._scale if scale is None else scale, window, sinks, 0)
        return out

    def status(self):
        """Waits for the current stream and raises if a kernel of this cache gave up on a bounded wait
        since the last report."""
        capi.check(capi.lib().bivmoe_cache_status(self._h, torch.cuda.current_stream(self._dev).cuda_stream))
