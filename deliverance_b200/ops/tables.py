"""Tables of a step built where they are used: the host sends the requests' lengths and page lists, one kernel writes what the layers read."""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import ops
from . import ref


class StepTables(NamedTuple):
    positions: torch.Tensor  # [T] int32
    slots: torch.Tensor  # [T] int64 flat cache rows (page * page_size + offset)
    q_start: torch.Tensor  # [S] int32
    ctx_len: torch.Tensor  # [S] int32 cached rows after the step
    block_tables: torch.Tensor  # [S, width] int32, zeros behind a sequence's pages
    logits_rows: torch.Tensor  # [S] int64 row of each sequence's last token
    tile_seq: torch.Tensor  # [tiles] int32
    tile_q0: torch.Tensor  # [tiles] int32


def step_tables(pages, page_start, cached, start, new, tokens: int, width: int, page_size: int, tile: int = 64, tiles: int = 0) -> StepTables:
    """Tables of a step of ``S`` sequences, ``new[i]`` tokens each. ``pages [n]``: the sequences' pages one after another, those of sequence i from ``page_start[i]`` to ``page_start[i + 1]``;
    ``cached[i]``: the cache row of its first new token, ``start[i]``: that token's position. All int32 on one device. Known to the host: ``tokens``, the sum of ``new``; ``width``, the columns of
    the block tables; ``tiles``, the number of query tiles of ``tile`` rows (0: none are made). At most 8,192 sequences.
    Lengths that do not add up, rows without a page and tables that are too narrow are reported by :func:`ops.check_status` (on the CPU: raised); such rows get slot -1."""
    if new.is_cuda:
        ops._count()
        return StepTables(*ops.require_ext().step_tables(pages, page_start, cached, start, new, tokens, width, page_size, tile, tiles))
    S = new.shape[0]
    if any(t.dtype != torch.int32 or t.dim() != 1 for t in (pages, page_start, cached, start, new)) or page_start.shape[0] != S + 1 or cached.shape[0] != S or start.shape[0] != S:
        raise ValueError("pages [n], page_start [S + 1], cached, start and new [S] must be int32")
    if S > 8192 or page_size < 1 or tile < 1 or tokens < 0 or width < 0 or not 0 <= tiles <= tokens:
        raise ValueError("sizes out of range")
    return StepTables(*ref.step_tables(pages, page_start, cached, start, new, tokens, width, page_size, tile, tiles))
