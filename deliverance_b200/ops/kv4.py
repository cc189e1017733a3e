"""A paged KV cache in 4 bits: 3.2 times as many tokens per byte as bf16, and as much less to read in every decode step.

Caches are uint8 ``[pages, KV, page, row bytes]``. A row of ``D`` numbers (one token, one KV head) is ``D / 2`` bytes of codes, byte i with element 2 i in its low half and 2 i + 1 in the high
one, and then per block of 32 elements two fp16 numbers, the block's step s and its minimum m: 5 bits a number. ``value = code * s + m``. Rows stand by themselves, so that
pages can be shared, copied and moved as bytes.

Quantising a block: ``m = fp16(min)``, ``s = (max - m) / 15`` rounded up to 7 significant bits (below 2^-14 to multiples of 2^-20), ``code = rint((x - m) / s)``; the divisions are
products with the fp32 reciprocals. What comes back is off by ``s / 2 + |min| 2^-11`` at most. Magnitudes above 472 are held as 472, a NaN makes its block NaN.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import ops
from . import ref


def row_bytes(D: int) -> int:
    """Bytes of a cached row of ``D`` numbers."""
    if D % 32:
        raise ValueError("rows of 4-bit caches are multiples of 32 numbers")
    return D // 2 + D // 8


def _check_caches(k, v, D: int) -> None:
    if D not in (64, 128, 256):
        raise ValueError("heads of 64, 128 or 256")
    for t in (k, v):
        if t.dtype != torch.uint8 or t.dim() != 4 or t.shape[3] != row_bytes(D) or t.shape != k.shape or not t.is_contiguous():
            raise ValueError(f"caches must be contiguous uint8 [pages, KV, page, {row_bytes(D)}]")
    if k.shape[2] % 32 or k.shape[2] < 32:
        raise ValueError("pages must have a multiple of 32 rows")


def rope_kv4(qkv, positions, slots, q_norm_w, k_norm_w, cos, sin, k_cache, v_cache, H: int, KV: int, D: int, eps: float, norm_offset: float = 0.0, rotate: str = "halves"):
    """:func:`ops.rope_kv` for 4-bit caches: head norms (both weights or None), rotation and cache write of ``qkv [T, (H + 2 KV) * D]``; returns the queries ``[T, H * D]``, ``qkv`` stays as it is.
    ``cos`` / ``sin`` fp32 ``[positions, half]`` (or None) rotate the first ``2 * half`` columns of a head: ``rotate`` ``"halves"`` column i with i + half, ``"pairs"`` 2 i with 2 i + 1. Positions
    outside the tables take their first or last row. A row with a negative slot is not written; the other slots of a call are different ones (but for rows of padding in the scratch page).
    Slots behind the caches are reported by :func:`ops.check_status` (on the CPU: an IndexError). On GPUs qkv and norms are bf16."""
    if rotate not in ("halves", "pairs"):
        raise ValueError("rotate must be 'halves' or 'pairs'")
    if qkv.is_cuda:
        ops._count()
        return ops.require_ext().kv4_write(qkv, positions, slots, q_norm_w, k_norm_w, cos, sin, k_cache, v_cache, H, KV, D, eps, norm_offset, rotate == "pairs")
    _check_caches(k_cache, v_cache, D)
    T = qkv.shape[0]
    if qkv.dim() != 2 or qkv.shape[1] != (H + 2 * KV) * D or k_cache.shape[1] != KV or positions.shape != (T,) or slots.shape != (T,) or slots.dtype != torch.int64:
        raise ValueError("qkv [T, (H + 2 KV) * D], positions [T], slots int64 [T] and caches do not fit")
    if (q_norm_w is None) != (k_norm_w is None) or (cos is None) != (sin is None):
        raise ValueError("both norms or none, both rotary tables or none")
    if cos is not None and (cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > D or cos.shape[0] < 1):
        raise ValueError("cos / sin must be [positions, half], with 2 * half columns of the head at most")
    return ref.rope_kv4(qkv, positions, slots, q_norm_w, k_norm_w, cos, sin, k_cache, v_cache, H, KV, D, eps, norm_offset, rotate == "pairs")


def expand4(k_cache, v_cache, pages, dtype: torch.dtype = torch.bfloat16):
    """The values of some pages (int32 ``[n]``, any order, repeats allowed) as ``[n, KV, page, D]`` keys and values in bf16 or fp32, each rounded once. Pages outside the caches are
    reported by :func:`ops.check_status` (on the CPU: an IndexError)."""
    D = k_cache.shape[3] * 8 // 5
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("values come in bf16 or fp32")
    if k_cache.is_cuda:
        ops._count()
        return ops.require_ext().kv4_expand(k_cache, v_cache, pages, D, dtype == torch.float32)
    _check_caches(k_cache, v_cache, D)
    if bool((pages < 0).any()):
        raise IndexError("pages must lie in the caches")
    return ref.kv4_unpack(k_cache[pages.long()], dtype), ref.kv4_unpack(v_cache[pages.long()], dtype)


def decode_attention4(q, k_cache, v_cache, block_tables, ctx_lens, H: int, scale: float, softcap: float = 0.0, window: int = 0):
    """:func:`ops.decode_attention` for 4-bit caches: one query row per sequence, ``q [B, H * D]`` -> ``[B, H * D]``, heads of 64, 128 or 256, up to 16 query heads per KV head. A sequence without keys gets
    zeros; what pages hold behind a sequence's end or in front of its window does not matter. Pages outside the caches and lengths beyond the table are reported by :func:`ops.check_status`
    (on the CPU: raised)."""
    if q.is_cuda:
        out, launches = ops.require_ext().kv4_decode(q, k_cache, v_cache, block_tables, ctx_lens, H, scale, softcap, window)
        ops._count(launches)
        return out
    B, D = q.shape[0], q.shape[1] // H
    _check_caches(k_cache, v_cache, D)
    if H % k_cache.shape[1] or H // k_cache.shape[1] > 16 or window < 0 or softcap < 0:
        raise ValueError("up to 16 query heads per KV head, window and softcap not negative")
    if block_tables.dim() != 2 or block_tables.shape[0] != B or ctx_lens.shape != (B,) or block_tables.dtype != torch.int32 or ctx_lens.dtype != torch.int32:
        raise ValueError("block_tables int32 [B, pages], ctx_lens int32 [B]")
    if bool((ctx_lens < 0).any()) or (int(ctx_lens.max()) if B else 0) > block_tables.shape[1] * k_cache.shape[2]:
        raise ValueError("lengths beyond the block table")
    return _plain(q, k_cache, v_cache, block_tables, torch.arange(B), torch.ones(B, dtype=torch.long), ctx_lens, H, scale, softcap, window, True)


def _plain(q, k_cache, v_cache, block_tables, q_start, q_len, ctx_lens, H, scale, softcap, window, causal):
    """CPU statement: the pages in use as fp32, one after another, then attention over them. (Rows behind a sequence's end are left out there, keys in front of a window have weight zero and
    finite values.)"""
    page = k_cache.shape[2]
    counts = [(int(n) + page - 1) // page for n in ctx_lens]
    table, used = torch.zeros(len(counts), max(counts + [1]), dtype=torch.int32), []
    for i, n in enumerate(counts):
        table[i, :n] = torch.arange(len(used), len(used) + n)
        used += [int(p) for p in block_tables[i, :n]]
    k, v = expand4(k_cache, v_cache, torch.tensor(used or [0], dtype=torch.int32), torch.float32)
    for i, n in enumerate(ctx_lens):
        first = max(0, int(n) - int(q_len[i]) + 1 - window) if window else 0
        if first:
            dead = table[i, : first // page].long()
            k[dead] = v[dead] = 0.0
            if first % page:
                k[table[i, first // page].long(), :, : first % page] = v[table[i, first // page].long(), :, : first % page] = 0.0
    T, D = q.shape[0], q.shape[1] // H
    live = [i for i in range(len(counts)) if int(ctx_lens[i]) > 0]
    o = ref.paged_attention(q.float().reshape(T, H, D), k, v, table[live], q_start[live], q_len[live], ctx_lens[live], scale, softcap, window, causal)
    return o.to(q.dtype).reshape(T, H * D)


EXPAND_PAGES_BYTES = 512 << 20  # fp16 pages that a call of prefill_attention4 makes at one time (at least one sequence's)


def prefill_attention4(q, k_cache, v_cache, block_tables, q_start, q_len, ctx_lens, H: int, scale: float, softcap: float = 0.0, window: int = 0, causal: bool = True,
                       q_len_host: Optional[list] = None, ctx_len_host: Optional[list] = None, tiles_for=None):
    """:func:`ops.prefill_attention` for 4-bit caches: packed query rows of sequences of different lengths (``q_start`` adds ``q_len`` up), which are the last rows of their ``ctx_lens`` cached ones. On
    GPUs the pages in use are unpacked to fp16 next to one another, :data:`EXPAND_PAGES_BYTES` of them at a time, and attended to there. ``q_len_host`` / ``ctx_len_host``: the same lengths on the
    host (else they are read back); ``tiles_for`` as there. What pages hold behind a sequence's end or in front of all its rows' windows does not matter. Pages outside the caches, cached lengths that are not the host's, and more query rows than
    there are or than cached ones, are reported by :func:`ops.check_status` (on the CPU: raised)."""
    T, D = q.shape[0], q.shape[1] // H
    if H % k_cache.shape[1] or window < 0 or softcap < 0 or not scale > 0:
        raise ValueError("KV heads must divide the query heads, scale must be positive, window and softcap not negative")
    news = q_len_host if q_len_host is not None and q.is_cuda else q_len.tolist()
    lens = ctx_len_host if ctx_len_host is not None and q.is_cuda else ctx_lens.tolist()
    S, KV, page = len(news), k_cache.shape[1], k_cache.shape[2]
    if sum(news) != T or len(lens) != S or any(not 0 <= n <= m for n, m in zip(news, lens)) or max(lens, default=0) > block_tables.shape[1] * page:
        raise ValueError("the query rows must be those of the sequences, no more than their cached rows, and these no more than the block table has")
    if not q.is_cuda:
        _check_caches(k_cache, v_cache, D)
        if block_tables.dim() != 2 or block_tables.shape[0] != S or any(t.dtype != torch.int32 for t in (block_tables, q_start, q_len, ctx_lens)) or q_start.tolist() != [sum(news[:i]) for i in range(S)]:
            raise ValueError("block_tables int32 [S, pages]; q_start, q_len, ctx_lens int32 [S], q_start the sums of q_len")
        if (q_len_host is not None and list(q_len_host) != news) or (ctx_len_host is not None and list(ctx_len_host) != lens):
            raise ValueError("the lengths on the host are other ones")
        return _plain(q, k_cache, v_cache, block_tables, q_start, q_len, ctx_lens, H, scale, softcap, window, causal)
    ext = ops.require_ext()
    if q.stride(1) != 1 or q.stride(0) % 8 or q.stride(0) < q.shape[1] or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)  # (``contiguous`` leaves a single row its stride)
    rows = ext.prefill_tc_tile_rows(D)
    # A CTA takes a tile of query rows of one head. Tiles of half the height where all of them run at one time on the 148 SMs: the softmax of a key tile has half the rows to wait for (heads of 128, us:
    # 700 rows of 16 heads 23.2 for 26.4, 2,048 of 8 heads 45.3 for 53.4, 200 rows behind 9,000 of 32 heads 193 for 221). Beyond that the second wave costs more (1,024 rows of 32 heads 45.7 for 35.7).
    if sum(-(-n // 128) for n in news) * H <= 148:
        rows = 128
    pages = [-(-n // page) for n in lens]
    tile_seq, tile_q0 = tiles_for(rows) if tiles_for is not None else _tiles(news, rows, q.device)
    if sum(pages) * KV * page * D * 4 <= EXPAND_PAGES_BYTES or S == 1:
        parts = _parts(news, lens, rows, H, window)
        ops._count(2 + (parts > 1))
        return ext.kv4_prefill(q, k_cache, v_cache, block_tables, q_start, q_len, ctx_lens, tile_seq, tile_q0, H, scale, softcap, window, causal, sum(pages), max(pages, default=0), rows, parts)
    outs, i, row, tile = [], 0, 0, 0  # (nothing comes from the host here: the portions' tables are cut out of the call's)
    while i < S:
        j, n_pages = i, 0
        while j < S and (j == i or (n_pages + pages[j]) * KV * page * D * 4 <= EXPAND_PAGES_BYTES):
            n_pages += pages[j]
            j += 1
        part, n, n_tiles = slice(i, j), sum(news[i:j]), sum(-(-m // rows) for m in news[i:j])
        parts = _parts(news[part], lens[part], rows, H, window)
        ops._count(2 + (parts > 1))
        outs.append(ext.kv4_prefill(q[row : row + n], k_cache, v_cache, block_tables[part], q_start[part] - row, q_len[part], ctx_lens[part], tile_seq[tile : tile + n_tiles] - i,
                                    tile_q0[tile : tile + n_tiles], H, scale, softcap, window, causal, n_pages, max(pages[part]), rows, parts))
        i, row, tile = j, row + n, tile + n_tiles
    return torch.cat(outs)


def _parts(news, lens, rows: int, H: int, window: int) -> int:
    """In how many parts, a CTA each, a call cuts the keys of its query tiles: as many as the 148 SMs hold at one time, of 128 keys or more. A part costs its CTA's start and a pass over its accumulator, so
    that a second wave loses (100 rows behind 9,000 of 32 heads of 128, us: 192 whole, 109 in 2 parts, 67 in 4, 74 in 8; 300 behind 30,000 of 8 heads 616, 144 in 6, 150 in 12; 20 behind 400 of 32 heads
    17.4, 14.5 in 4, 20.6 in 8)."""
    tiles = sum(-(-n // 128) for n in news) * H
    if rows != 128 or tiles * 2 > 148 or tiles == 0:
        return 1
    keys = max(min(m, window + 128) if window else m for m in lens)  # (of any tile, at most)
    return max(1, min(148 // tiles, keys // 128, 32))


def _tiles(news, rows: int, device):
    return tuple(torch.tensor(t, dtype=torch.int32, device=device) for t in ops.prefill_tiles(news, rows))
