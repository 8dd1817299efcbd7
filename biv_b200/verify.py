"""Drafted tokens against the target's probabilities, over the C ABI.

The reference drafts tokens, lets the model see them in one pass and keeps those that it agrees with (``Session::{draft, verify,
keep}``, chat.rs:632-678).  ``verify`` makes the choice on the device, from given random numbers, so that the tokens that come out
are distributed as the target's own, and leaves the lengths that the next ``PagedCache.extend`` starts from.  It runs on the current
torch stream, waits for nothing and can be captured into a graph.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import capi
from .linear import _step_calls

_call = None


class Verified(NamedTuple):
    """What ``verify`` leaves (device tensors, int32)."""
    accepted: torch.Tensor            # [n_seq]: how many of its drafts
    token: torch.Tensor               # [n_seq]: the token after them; -1 where p holds nothing positive
    kept: Optional[torch.Tensor]      # [n_seq]: length less the drafts that were not accepted


def verify(p, tokens, uniform, sample, first, q=None, length=None) -> Verified:
    """Rows first[b] to first[b + 1] - 1 of p [n, vocabulary] (float32, float16 or bfloat16) are request b's: ``tokens`` [n] int32
    holds its current token and then its drafts, and p[r] is the target's distribution of the token after row r's.  ``q`` [n,
    vocabulary]: the one that the draft after row r was drawn from; without it the drafts are certain (looked up, or a greedy
    choice).  Draft d after row r is accepted while ``uniform[r] * q[r, d] < p[r, d]``; then a token is drawn by ``sample[b]`` from
    max(p - q, 0) of the first row whose draft failed, or from p of the request's last row.  ``length`` [n_seq]: the requests' tokens
    with all of the rows (``Step.length``); ``kept`` is then the next step's ``past``.  Random numbers are float32 in [0, 1).  A draft
    whose q or p is NaN is not accepted, a weight that is NaN counts as zero, and of infinite weights the last positive one is drawn."""
    global _call
    if _call is None:
        _call = C.cast(capi.lib().bivmoe_verify, C.c_void_p).value
    r = _step_calls.verify(_call, p, q, tokens, uniform, sample, first, length)
    if r.__class__ is int:
        capi.check(r)
    return Verified._make(r)
