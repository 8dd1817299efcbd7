"""Linear attention with a decay for each head, over the C ABI: the other kind of a decoder layer's attention half.

The reference's recurrent layers keep, instead of keys and values, one state of dim_v x dim_k for each head, to which every token
adds (engine/src/model.rs:900-1116; on Metal ``gdn_128``, engine/src/metal/kernels.metal:959-1573).  ``LinearAttention`` stands
beside ``PagedCache`` for such layers: the states of all requests lie in slots, a call takes each request's new tokens, from one to
a whole prompt, and every call runs on the current torch stream, waits for nothing and can be captured into a graph.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import capi

try:
    from . import _step_calls
except ImportError as e:
    raise ImportError("biv_b200/_step_calls.so is missing or was built for another torch: build it with `python -c "
                      "'import __graft_entry__ as g; g.build()'` (or `make -C biv_b200/csrc all`); there is no fallback") from e

_GGML = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


class LinearAttention:
    """Geometry of the calls: ``n_head`` heads of v, outputs, decays and states, which share ``n_head_qk`` heads of q and k; dims
    of 64, 128 or 256; rows of ``dtype`` (bfloat16, float16 or float32).  States are float32 whatever the rows' type."""

    def __init__(self, n_head: int, n_head_qk: int, dim_k: int, dim_v: int, max_seqs: int, dtype: torch.dtype = torch.bfloat16,
                 device: int = 0):
        self._h = None
        if dtype not in _GGML:
            raise ValueError("rows are float32, float16 or bfloat16")
        d = capi.LinearDesc(_GGML[dtype], n_head, n_head_qk, dim_k, dim_v, max_seqs, device, 0)
        h = C.c_void_p()
        L = capi.lib()
        capi.check(L.bivmoe_linear_create(C.byref(d), C.byref(h)))
        self._h = h
        self.n_head, self.n_head_qk, self.dim_k, self.dim_v = n_head, n_head_qk, dim_k, dim_v
        self.max_seqs, self.dtype, self.device = max_seqs, dtype, device
        self._geometry = _step_calls.make(h.value, C.cast(L.bivmoe_linear_attend, C.c_void_p).value, device, n_head, n_head_qk,
                                          dim_k, dim_v, _GGML[dtype])

    def close(self):
        if self._h is not None:
            capi.lib().bivmoe_linear_destroy(self._h)
            self._h = self._geometry = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def states(self, n_slots: int):
        """A layer's states, cleared."""
        return torch.zeros((n_slots, self.n_head, self.dim_v, self.dim_k), device=f"cuda:{self.device}")

    def attend(self, q, k, v, decay, states, slots, first, beta=None, past=None, keep=None, max_new: int = 0,
               scale: Optional[float] = None, out=None):
        """For each request b, in the order of its rows first[b] to first[b + 1] - 1, on its state S in ``states[slots[b]]``:
        ``S = exp(decay) S + v k^T`` or, with ``beta`` (the delta rule), ``S = exp(decay) S + beta (v - exp(decay) S k) k^T``; and
        ``out = scale S q`` (scale: dim_k^-0.5).  q and k are [n, n_head_qk, dim_k], v and out [n, n_head, dim_v] (any strides of
        the first two that are multiples of 16 bytes), decay (logarithms, at most zero) and beta [n, n_head] float32.  A request
        with ``past[b]`` 0 starts from zeros whatever its slot holds.  ``keep[b]``: the state is kept as it is after that many
        of the call's tokens, with 0 left as it was: drafted tokens are computed with 0, and ``advance`` takes the accepted ones.
        Slots below zero, past the states, or that an earlier request has already: from zeros, and not kept.  ``max_new``: the
        most new tokens of a request; it decides the kernel for all of them, and so the speed: single tokens are best not given in one call
        with prompts.  ``out`` may be v itself."""
        r = _step_calls.attend(self._geometry, q, k, v, decay, states, slots, first, beta, past, keep, max_new, scale, out)
        if r.__class__ is int:
            capi.check(r)
        return r

    def advance(self, k, v, decay, states, slots, first, beta=None, past=None, keep=None, max_new: int = 0):
        """``attend`` without its outputs: the states alone."""
        r = _step_calls.attend(self._geometry, None, k, v, decay, states, slots, first, beta, past, keep, max_new, None, None)
        if r.__class__ is int:
            capi.check(r)

    def status(self):
        """Waits for the current stream and raises if a kernel of this layer gave up on a bounded wait since the last report."""
        capi.check(capi.lib().bivmoe_linear_status(self._h, torch.cuda.current_stream(self.device).cuda_stream))
