"""Beam search: which continuations live on, and the states that follow them.

A request keeps ``beams`` hypotheses, one row of the decode batch each. After a step, :func:`beam_select` scores every continuation of every beam,
``scores[b, w] + log softmax(logits[b, w])[v]``, and returns the best ones with the beam they go on from. :func:`beam_reorder` then gives every beam
its parent's past: the recurrent states, and of the paged cache the rows of the page that is still being filled. Full pages are not copied, the
beams share them by reference (``engine.beams``).
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import ops
from . import ref

MAX_BEAMS = 32
MAX_CANDIDATES = 64


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, mask: Optional[torch.Tensor] = None, softcap: float = 0.0, inv_scale: float = 1.0):
    """The ``k`` best continuations of every request: ``(values [B, k] fp32, parents [B, k], tokens [B, k])``, best first, equal values in the order of
    beam and token. ``logits [B * W, V]`` (fp32 or bf16, post-processed like :func:`ops.logits_post`: ``softcap(logits * inv_scale)``, tokens outside the int32
    allow-bitmask ``mask`` left out), ``scores [B, W]`` fp32, the beams' sums so far; -inf for a beam that is not in use. A candidate's value is finite in fp32: a logit of
    -inf is a masked token, a row with a NaN (or +inf, without a softcap) and a beam whose score is not finite give none. Places that no candidate is left for have value
    -inf, parent and token -1. On the GPU a beam's log-sum-exp is off by 4e-6 at most (32-bit exponentials), the same for all of its tokens: candidates of different beams that are closer than twice that
    may come in either order, candidates of one beam come in the order of their logits."""
    if logits.is_cuda:  # (the extension checks)
        ops._count(2)
        return ops.require_ext().beam_select(logits, scores, k, mask, softcap, inv_scale)
    if scores.dim() != 2 or logits.dim() != 2 or logits.shape[0] != scores.numel():
        raise ValueError("logits must be [requests * beams, V], scores [requests, beams]")
    if not 1 <= scores.shape[1] <= MAX_BEAMS or not 1 <= k <= min(MAX_CANDIDATES, scores.shape[1] * logits.shape[1]):
        raise ValueError(f"1 to {MAX_BEAMS} beams, 1 to {MAX_CANDIDATES} candidates, no more than there are")
    if not inv_scale > 0 or not softcap >= 0:
        raise ValueError("inv_scale must be positive, softcap not negative")
    return ref.beam_select(logits, scores, k, None if mask is None else ops.unpack_mask(mask, logits.shape[1]), softcap, inv_scale)


def beam_reorder(parents: torch.Tensor, states=(), slots: Optional[torch.Tensor] = None, caches=(), pages: Optional[torch.Tensor] = None,
                 rows: Optional[torch.Tensor] = None) -> None:
    """Every beam takes over its parent's state, in place: ``t[slots[b, j]] = t[slots[b, parents[b, j]]]`` (as they were before the call) for the tensors ``states``
    (``[slots, ...]``), and the first ``rows[b]`` rows of all heads of page ``pages[b, parents[b, j]]`` go to page ``pages[b, j]`` for the page pools ``caches``
    (``[pages, KV, page, D]``; ``rows`` None: whole pages). ``parents``, ``slots`` and ``pages`` are int64 ``[B, W]``, ``rows`` int32 ``[B]``. A parent outside
    ``0 .. W - 1`` leaves its beam as it is. All slots (pages) of a call are different ones; one outside the tensors is left out and reported by
    :func:`ops.check_status` (on the CPU: raised)."""
    if parents.is_cuda:  # (the extension checks: a loop over the layers here takes longer than the kernel)
        e = ops.require_ext()
        if len(states):
            ops._count(e.beam_move(states, slots, parents))
        if len(caches):
            ops._count(e.beam_move(caches, pages, parents, rows, True))
        return
    for group, index, name in ((states, slots, "slots"), (caches, pages, "pages")):
        if group and (index is None or index.shape != parents.shape or index.dim() != 2 or index.shape[1] > MAX_BEAMS or index.dtype != torch.int64 or parents.dtype != torch.int64):
            raise ValueError(f"{name} and parents must be int64 [requests, beams] with at most {MAX_BEAMS} beams")
    if any(c is not None and c.dim() != 4 for c in caches):
        raise ValueError("page pools are [pages, KV, page, D]")
    if rows is not None and (rows.shape != parents.shape[:1] or rows.dtype != torch.int32):
        raise ValueError("rows must be int32 [requests]")
    for t in _distinct(states):
        ref.beam_move(t, slots, parents, None)
    for t in _distinct(caches):
        ref.beam_move(t, pages, parents, rows if rows is not None else torch.full((parents.shape[0],), t.shape[2], dtype=torch.int32))


def _distinct(tensors) -> list:
    """Layers that share a cache name it twice; it moves once."""
    return list({t.data_ptr(): t for t in tensors if t is not None}.values())
