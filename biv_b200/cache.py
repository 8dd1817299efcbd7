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
from typing import NamedTuple, Optional, Sequence

import torch

from . import capi

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
        self._dev = torch.device("cuda", device)
        self._scale = 1.0 / math.sqrt(head_dim)
        # the structs of a call, filled in anew each time: what does not change is set here
        self._e, self._s, self._a = capi.ExtendArgs(), capi.StoreArgs(), capi.AttendArgs()
        self._s.q_out_type = self._a.q_type = self._a.out_type = _GGML[dtype]
        self._refs = C.byref(self._e), C.byref(self._s), C.byref(self._a)

    def close(self):
        if self._h is not None:
            capi.lib().bivmoe_cache_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _stream(self):
        return torch.cuda.current_stream(self._dev).cuda_stream

    def _ints(self, t, what, n, dtype=torch.int32):
        if t.dtype != dtype or t.device != self._dev or not t.is_contiguous() or t.numel() < n:
            raise ValueError(f"{what}: {n} contiguous {dtype} on {self._dev} are wanted")
        return t.data_ptr()

    def pools(self, n_pages: int):
        """A layer's k and v pools."""
        shape = (n_pages, self.page_size, self.n_head_kv, self.head_dim)
        return tuple(torch.empty(shape, dtype=self.dtype, device=self._dev) for _ in range(2))

    def _table(self, a, table, n_seq):
        if table.dtype != torch.int32 or table.device != self._dev or table.dim() != 2 or table.shape[0] < n_seq or \
                (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError("table: [n_seq, pages] int32 with neighbouring pages is wanted")
        a.table, a.table_stride, a.table_width, a.n_seq = table.data_ptr(), table.stride(0), table.shape[1], n_seq

    def _pool(self, a, name, t):
        shape = t.shape
        if t.dtype != self.dtype or t.device != self._dev or len(shape) != 4 or shape[1] != self.page_size or \
                shape[2] != self.n_head_kv or shape[3] != self.head_dim or t.stride(3) != 1:
            raise ValueError(f"{name}: [pages, {self.page_size}, {self.n_head_kv}, {self.head_dim}] of {self.dtype} is wanted")
        p, k, h, _ = t.stride()
        if name == "k_pool":
            a.k_pool, a.k_pool_stride_page, a.k_pool_stride_token, a.k_pool_stride_head, a.k_pool_n_pages = t.data_ptr(), p, k, h, shape[0]
        else:
            a.v_pool, a.v_pool_stride_page, a.v_pool_stride_token, a.v_pool_stride_head, a.v_pool_n_pages = t.data_ptr(), p, k, h, shape[0]

    def _rows(self, t, what, heads, n=None):
        shape = t.shape
        if t.device != self._dev or len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim or t.stride(2) != 1 or \
                (n is not None and shape[0] != n):
            raise ValueError(f"{what}: [tokens, {heads}, {self.head_dim}] rows on {self._dev} are wanted")
        return t.data_ptr(), t.stride(0), t.stride(1)

    def extend(self, past, added, free_pages, free_count, table, n_tokens: int, held=None, out: Optional[Step] = None) -> Step:
        """Pages for ``added[b]`` new tokens of each request b, which has ``past[b]`` (int32 device
        tensors).  Takes them from the end of the free list (``free_pages[:free_count]``), writes the
        new entries of ``table`` [n_seq, pages], and returns the step.  ``n_tokens`` rows are laid out:
        more than the requests add (a padded batch) have slot -1.  ``held``: pages each request holds
        already, where that is not what ``past`` needs (drafted tokens that were taken back); ``out``:
        a step to write into."""
        n_seq, a = past.numel(), self._e
        if out is None:
            i32 = dict(dtype=torch.int32, device=self._dev)
            room = torch.empty(3 * n_seq + 3 + n_tokens, **i32)
            length, first, left, kept, positions = room.split([n_seq, n_seq + 1, 2, n_seq, n_tokens])
            out = Step(length, first, torch.empty(n_tokens, dtype=torch.int64, device=self._dev), positions, left, kept)
        a.past, a.added = self._ints(past, "past", n_seq), self._ints(added, "added", n_seq)
        a.held = None if held is None else self._ints(held, "held", n_seq)
        a.free_pages, a.n_free = self._ints(free_pages, "free_pages", 0), free_pages.numel()
        a.free_count = self._ints(free_count, "free_count", 1)
        self._table(a, table, n_seq)
        a.n_tokens = n_tokens
        a.length, a.first = self._ints(out.length, "length", n_seq), self._ints(out.first, "first", n_seq + 1)
        a.slots = self._ints(out.slots, "slots", n_tokens, torch.int64)
        a.positions, a.left = self._ints(out.positions, "positions", n_tokens), self._ints(out.left, "left", 2)
        a.held_out = self._ints(out.held, "held", n_seq)
        capi.check(capi.lib().bivmoe_cache_extend(self._h, self._refs[0], self._stream()))
        return out

    def store(self, q, k, v, k_pool, v_pool, slots, positions=None, out=None):
        """q and k [n, heads, head_dim] (float32, float16 or bfloat16; any strides of the first two)
        turned by ``positions`` ([n], or [axes, n]), k and v into the pages at ``slots``; returns the
        turned q in the cache's type."""
        n, a = q.shape[0], self._s
        a.q, a.q_stride_token, a.q_stride_head = self._rows(q, "q", self.n_head)
        a.k, a.k_stride_token, a.k_stride_head = self._rows(k, "k", self.n_head_kv, n)
        a.v, a.v_stride_token, a.v_stride_head = self._rows(v, "v", self.n_head_kv, n)
        if q.dtype not in _GGML or k.dtype != q.dtype or v.dtype != q.dtype:
            raise ValueError("q, k and v: rows of one type, float32, float16 or bfloat16, are wanted")
        a.q_type = a.k_type = a.v_type = _GGML[q.dtype]
        if out is None:
            out = torch.empty((n, self.n_head, self.head_dim), dtype=self.dtype, device=self._dev)
        elif out.dtype != self.dtype:
            raise ValueError(f"out: {self.dtype} is wanted")
        a.q_out, a.q_out_stride_token, a.q_out_stride_head = self._rows(out, "out", self.n_head, n)
        self._pool(a, "k_pool", k_pool)
        self._pool(a, "v_pool", v_pool)
        a.slots, a.n_tokens = self._ints(slots, "slots", n, torch.int64), n
        a.positions, a.positions_stride = None, 0
        if self.rope is not None:
            axes = len(self.rope.sections)
            if positions is None or positions.dtype != torch.int32 or positions.device != self._dev or \
                    positions.numel() != axes * n or (n > 1 and positions.stride(-1) != 1):
                raise ValueError(f"positions: [{axes}, n] int32 are wanted" if axes > 1 else "positions: [n] int32 are wanted")
            a.positions, a.positions_stride = positions.data_ptr(), positions.stride(0) if positions.dim() > 1 else n
        capi.check(capi.lib().bivmoe_cache_store(self._h, self._refs[1], self._stream()))
        return out

    def attend(self, q, k_pool, v_pool, table, first, length, max_new: int = 0, scale: Optional[float] = None,
               window: int = 0, sinks: int = 0, out=None):
        """Attention of the rows q [n, n_head, head_dim], request b's from first[b] to first[b + 1] - 1,
        the last tokens of its length[b] tokens.  A token at position p sees p and what is before it;
        with ``window`` the last ``window`` positions up to its own and the first ``sinks``.  ``max_new``:
        the most new rows of a request, where the caller knows it."""
        n_seq, a = length.numel(), self._a
        if q.dtype != self.dtype:
            raise ValueError(f"q: {self.dtype} is wanted")
        a.q, a.q_stride_token, a.q_stride_head = self._rows(q, "q", self.n_head)
        n = q.shape[0]
        if out is None:
            out = torch.empty((n, self.n_head, self.head_dim), dtype=self.dtype, device=self._dev)
        elif out.dtype != self.dtype:
            raise ValueError(f"out: {self.dtype} is wanted")
        a.out, a.out_stride_token, a.out_stride_head = self._rows(out, "out", self.n_head, n)
        self._pool(a, "k_pool", k_pool)
        self._pool(a, "v_pool", v_pool)
        self._table(a, table, n_seq)
        a.first, a.length = self._ints(first, "first", n_seq + 1), self._ints(length, "length", n_seq)
        a.n_tokens, a.max_new = n, max_new
        a.scale, a.window, a.sinks = self._scale if scale is None else scale, window, sinks
        capi.check(capi.lib().bivmoe_cache_attend(self._h, self._refs[2], self._stream()))
        return out

    def status(self):
        """Waits for the current stream and raises if a kernel of this cache gave up on a bounded wait
        since the last report."""
        capi.check(capi.lib().bivmoe_cache_status(self._h, self._stream()))
