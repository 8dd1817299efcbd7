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
from typing import NamedTuple, Optional, Sequence

import torch

from . import capi

try:
    from . import _cache_calls
except ImportError as e:
    raise ImportError("biv_b200/_cache_calls.so is missing or was built for another torch: build it with `python -c "
                      "'import __graft_entry__ as g; g.build()'` (or `make -C biv_b200/csrc all`); there is no fallback") from e

_GGML = {torch.float16: 1, torch.bfloat16: 30}


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
    held: torch.Tensor        # [n_seq] int32: pages that each request's tokens take, missing ones among them


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
        # the calls go through a small extension module (checks, outputs, argument structs), by these addresses
        L = capi.lib()
        at = [C.cast(f, C.c_void_p).value for f in (L.bivmoe_cache_extend, L.bivmoe_cache_store, L.bivmoe_cache_attend)]
        self._geometry = _cache_calls.make(h.value, *at, device, n_head, n_head_kv, head_dim, page_size, _GGML[dtype],
                                           len(rope.sections) if rope is not None else 0)

    def close(self):
        if self._h is not None:
            capi.lib().bivmoe_cache_destroy(self._h)
            self._h = self._geometry = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def pools(self, n_pages: int):
        """A layer's k and v pools."""
        shape = (n_pages, self.page_size, self.n_head_kv, self.head_dim)
        return tuple(torch.empty(shape, dtype=self.dtype, device=f"cuda:{self.device}") for _ in range(2))

    def extend(self, past, added, free_pages, free_count, table, n_tokens: int, held=None, out: Optional[Step] = None) -> Step:
        """Pages for ``added[b]`` new tokens of each request b, which has ``past[b]`` (int32 device
        tensors).  Takes them from the end of the free list (``free_pages[:free_count]``), writes the
        new entries of ``table`` [n_seq, pages], and returns the step.  ``n_tokens`` rows are laid out:
        more than the requests add (a padded batch) have slot -1.  ``held``: pages each request holds
        already, where that is not what ``past`` needs (drafted tokens that were taken back); ``out``:
        a step to write into.  Tokens that got no slot (``unstored``) are not stored and not seen later: such a
        step is made again, from the same lists with more free pages at their end or a wider table, before its
        lengths are used."""
        r = _cache_calls.extend(self._geometry, past, added, held, free_pages, free_count, table, n_tokens, out)
        if r.__class__ is int:
            capi.check(r)
        return r if out is not None else Step._make(r)

    def store(self, q, k, v, k_pool, v_pool, slots, positions=None, out=None):
        """q and k [n, heads, head_dim] (float32, float16 or bfloat16; any strides of the first two)
        turned by ``positions`` ([n], or [axes, n], which may be one row expanded), k and v into the pages at ``slots``; returns the
        turned q in the cache's type."""
        r = _cache_calls.store(self._geometry, q, k, v, k_pool, v_pool, slots, positions, out)
        if r.__class__ is int:
            capi.check(r)
        return r

    def attend(self, q, k_pool, v_pool, table, first, length, max_new: int = 0, scale: Optional[float] = None,
               window: int = 0, sinks: int = 0, out=None):
        """Attention of the rows q [n, n_head, head_dim], request b's from first[b] to first[b + 1] - 1,
        the last tokens of its length[b] tokens.  A token at position p sees p and what is before it;
        with ``window`` the last ``window`` positions up to its own and the first ``sinks``.  ``max_new``:
        the most new rows of a request; pass it where it is known: it decides the kernel, and a decode step without it
        may take twice as long."""
        r = _cache_calls.attend(self._geometry, q, k_pool, v_pool, table, first, length, max_new, scale, window, sinks, out)
        if r.__class__ is int:
            capi.check(r)
        return r

    def status(self):
        """Waits for the current stream and raises if a kernel of this cache gave up on a bounded wait
        since the last report."""
        capi.check(capi.lib().bivmoe_cache_status(self._h, torch.cuda.current_stream(self.device).cuda_stream))

    def unstored(self) -> int:
        """Waits for the current stream; how many new tokens of ``extend`` calls got no slot since the last
        report: for want of a free page, in this call or in an earlier one, or of a place in the table."""
        n = C.c_uint64()
        capi.check(capi.lib().bivmoe_cache_unstored(self._h, C.byref(n), torch.cuda.current_stream(self.device).cuda_stream))
        return n.value
