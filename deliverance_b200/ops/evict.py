"""A cache of bounded length: the attention weights that every cached key has received are added up, and from time to time the keys that received
the least are dropped.

Every sequence has a row ``weights[slot]`` per layer, fp32 ``[KV, capacity]``: entry i is the sum, over the decode steps since the key came into row i and
over the query heads that share the KV head, of the probabilities it had. :func:`decode_attention_weighted` is decode attention that also adds a step's
probabilities. :func:`evict_keys` keeps, per layer, sequence and KV head, the newest rows and the heaviest of the others, in their order, in the first rows of
the sequence's pages. KV heads keep different keys, but all of them equally many, so that block tables and lengths stay what they are for the rest of
the framework. Keys carry their rotary positions with them; what changes is the row that they lie in.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import ops
from . import ref


def by_length(splits: int, B: int, H: int, KV: int, D: int) -> bool:
    """Whether weighted attention of ``B`` sequences of unlike lengths is launched otherwise than of like ones, ``splits`` being what the caller allows (us per layer, launched as of like
    lengths / as of their own, plan shared by four layers, heads of 128 on 8 KV heads: 8 sequences of 1,000 to 32,000 keys 86.0 / 73.2, 16 of 500 to 16,000 90.6 / 70.1, 64 of 100 to 2,176 52.2 / 47.1;
    heads of 64 on 4: 16 of 500 to 16,000 41.0 / 31.2; 2 of 200 to 2,000, with room for 74, the same)."""
    room = ops.decode_room(B, H, KV, D)
    return splits > room or room <= 32


def score_room(B: int, H: int, rows: int, capacity: int) -> int:
    """Scores that weighted attention of ``B`` sequences keeps for a while, with block tables of ``rows`` rows and weights of ``capacity``."""
    return B * H * max(16, (min(rows, capacity) + 15) // 16 * 16)


def decode_attention_weighted(q, k_cache, v_cache, block_tables, ctx_lens, H, scale, weights, slots, softcap=0.0, window=0, splits=1, even=False, plan=None, scores=None):
    """:func:`ops.decode_attention`, which also adds every key's probabilities to ``weights[slots[b], kv head, row]`` (fp32 ``[slots, KV, capacity]``, in place;
    ``slots`` int64 ``[B]``). Rows of a sequence at or behind the capacity are attended to and not counted. Slot 0 is the scratch slot: a sequence with slot 0 adds nothing. The other
    slots of a call are different ones; a second sequence on a slot, or a slot outside ``weights``, adds nothing and is reported by :func:`ops.check_status` (on the CPU:
    raised). ``scores``: fp32 workspace of :func:`score_room` numbers, for calls that follow one another on a stream (captured ones would else keep one each); default: the call's own."""
    if q.is_cuda:  # (the extension checks)
        B, (_, KV, page, D) = q.shape[0], k_cache.shape
        if even:
            # Of heads of 64 four CTAs are resident per SM, and parts are longer here (us, as many as the engine asks for / this: 6 sequences of 23,000 keys 48.7 / 38.6; 2 of 8,000 18.0 / 16.0;
            # 1 of 60,000 28.7 / 19.5; 4 of 4,000 13.3 / 13.0). Of heads of 128 two are: 1 of 4,000 9.9 / 11.4, 3 of 20,000 49.3 / 49.5.
            if D <= 64 and splits > 1:
                splits = max(splits, min(ops.decode_room(B, H, KV, D), 128, block_tables.shape[1] * page // 128))
        elif splits <= 32 and (plan is not None or block_tables.shape[1] * page >= 4096):
            # Splits by length pay here where splits by number do not, because every part's tail is longer: twice as many as the batch has use for, given to the long sequences
            # (us, as many as the engine asks for / this, plan kept by the caller: 16 sequences of 500 to 16,000 keys, heads of 64, 47.3 / 41.3; 24 of 100 to 6,000 25.6 / 19.1; 8 of 1,000 to 32,000, heads of
            # 128, 69.7 / 66.8; 12 of 50 to 500 11.8 / 11.9, and 13.3 with a plan of its own; 3 sequences, with room for 98, 19.1 / 22.8).
            room = ops.decode_room(B, H, KV, D)
            if splits <= room <= 32:
                splits = 2 * room
        splits, used = ops.decode_launch(splits, even, plan, ctx_lens, B, H, KV, D, int(window))
        out, launches = ops.require_ext().decode_attention_weighted(q, k_cache, v_cache, block_tables, ctx_lens, H, scale, softcap, window, splits, weights, slots, used, scores)
        ops._count(launches)
        return out
    if weights.dim() != 3 or weights.dtype != torch.float32 or weights.shape[1] != k_cache.shape[1]:
        raise ValueError("weights must be fp32 [slots, KV, capacity]")
    if slots.dim() != 1 or slots.shape[0] != q.shape[0] or slots.dtype != torch.int64:
        raise ValueError("slots must be int64, one per query row")
    return ref.decode_attention_weighted(q, k_cache, v_cache, block_tables, ctx_lens, H, scale, weights, slots, softcap, window)


def evict_keys(k_caches, v_caches, weights, block_tables, ctx_lens, slots, keep: int, recent: int, out_tables: Optional[torch.Tensor] = None):
    """Shorten sequences of more than ``keep`` rows to ``keep``: the last ``recent`` rows and, of the others, those with the largest weights (equal weights, and NaN
    as the smallest: the earliest; rows at or behind the capacity count as weight 0). What is kept moves, in order, to the first rows of ``out_tables[b]`` (default: of ``block_tables[b]``) in all layers, its weights to the first entries of
    ``weights[layer][slots[b]]``; the weights behind them, up to the old length, become zero. Sequences that are short enough keep everything, and with ``out_tables`` move too.

    ``k_caches`` / ``v_caches``: per layer ``[pages, KV, page, D]`` (widths may differ); ``weights``: per layer fp32 ``[slots, KV, capacity]``; ``block_tables`` / ``out_tables`` int32 ``[B, pages]``,
    ``ctx_lens`` int32 ``[B]``, ``slots`` int64 ``[B]``, all different (0, the scratch slot: only for sequences of length 0). An entry of ``out_tables`` is either the page that ``block_tables`` has in the same place, if no other sequence has it, or a page that no sequence of the
    call reads: what sequences share (a cached prefix, beams) is replaced, not changed. A sequence on a slot that another one has, or outside the weights, is left as it is; that, pages
    outside the caches and lengths beyond the table are reported by :func:`ops.check_status` (on the CPU: raised).
    Returns the rows that were kept, int32 ``[layers, B, KV, keep]`` (-1 behind a sequence's end), and the new lengths, int32 ``[B]``."""
    if ctx_lens.is_cuda:  # (the extension checks: a loop over the layers here takes longer than the kernels)
        kept, lens, launches = ops.require_ext().evict_keys(k_caches, v_caches, weights, block_tables, ctx_lens, slots, keep, recent, block_tables if out_tables is None else out_tables)
        ops._count(launches)
        return kept, lens
    k_caches, v_caches, weights = list(k_caches), list(v_caches), list(weights)
    if not k_caches or not len(k_caches) == len(v_caches) == len(weights):
        raise ValueError("one key cache, value cache and weight tensor per layer")
    if not 0 <= recent <= keep or keep < 1:
        raise ValueError("0 <= recent <= keep, 1 <= keep")
    first = k_caches[0]
    for k, v, w in zip(k_caches, v_caches, weights):
        if k.dim() != 4 or v.dim() != 4 or k.shape[:3] != first.shape[:3] or v.shape[:3] != first.shape[:3]:
            raise ValueError("caches must be [pages, KV, page, D], with the same pages and KV heads in all layers")
        if w.dim() != 3 or w.dtype != torch.float32 or w.shape != weights[0].shape or w.shape[1] != k.shape[1]:
            raise ValueError("weights must be fp32 [slots, KV, capacity], the same in all layers")
    if len({t.data_ptr() for t in k_caches + v_caches}) < 2 * len(k_caches):
        raise ValueError("a cache that several layers share cannot be shortened for one of them")
    B = ctx_lens.shape[0]
    out = block_tables if out_tables is None else out_tables
    if block_tables.dim() != 2 or block_tables.shape[0] != B or slots.shape != (B,) or slots.dtype != torch.int64 or block_tables.dtype != torch.int32 or ctx_lens.dtype != torch.int32:
        raise ValueError("block_tables int32 [B, pages], ctx_lens int32 [B], slots int64 [B]")
    if out.dim() != 2 or out.shape[0] != B or out.dtype != torch.int32 or out.shape[1] * first.shape[2] < min(keep, block_tables.shape[1] * first.shape[2]):
        raise ValueError("out_tables must be int32 [B, pages] with room for the kept rows")
    return ref.evict_keys(k_caches, v_caches, weights, block_tables, ctx_lens, slots, keep, recent, out)
