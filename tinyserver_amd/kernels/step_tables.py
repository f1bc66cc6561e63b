"""A step's block tables, positions and slots, built on the GPU.

What the reference does on the host for every step: BlockManager's pages for the
new tokens (server/model/block_manager.py:102-134) and the patch's padded tables
and mapping loop (server/model/patches/qwen3.py:296-318, 388-397). Here the tables
and the free list live on the GPU, and a step gives the requests' lengths.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib


class StepTables(NamedTuple):
    """What the store and the attention of a step take, all int32 on the GPU."""

    block_tables: torch.Tensor   # (B, width), 0 behind a request's pages
    cu_seqlens: torch.Tensor     # (B + 1,)
    seq_lens: torch.Tensor       # (B,) cached and new tokens
    positions: torch.Tensor      # (num_tokens,)
    block_mapping: torch.Tensor  # (num_tokens,) page of each new token
    slot_mapping: torch.Tensor   # (num_tokens,) its slot there
    free_left: torch.Tensor | None  # (1,) entries of the free list that are left


def _ints(name: str, t: torch.Tensor, dims: int = 1) -> torch.Tensor:
    if t.dim() != dims:
        raise ValueError(f"{name} must be a {dims}D tensor, but got shape {tuple(t.shape)}")
    return t if t.dtype == torch.int32 else t.to(torch.int32)


def step_tables(
    tables: torch.Tensor,
    context_lens: torch.Tensor,
    query_lens: torch.Tensor,
    block_size: int,
    num_tokens: int,
    *,
    rows: torch.Tensor | None = None,
    width: int | None = None,
    free_blocks: torch.Tensor | None = None,
    num_free: torch.Tensor | None = None,
) -> StepTables:
    """The tables of a step in which request s, with ``context_lens[s]`` tokens in
    the cache, brings ``query_lens[s]`` new ones.

    tables (R, W) int32: the block tables of all requests; request s's is row
    ``rows[s]`` (by default s). With ``free_blocks`` the pages that the new tokens
    need beyond ``ceil(context_lens[s] / block_size)`` are taken off that list in
    batch order, entry ``num_free - 1`` first (num_free (1,) int32 on the GPU; by
    default all entries), and written to ``tables``; ``free_left`` says how many
    entries are left, which the next step takes as its num_free. If the list is too
    short free_left is negative, and the requests it does not reach have -1 in their
    tables, which every kernel skips. Without ``free_blocks`` the tables hold the
    new tokens' pages already.

    num_tokens: rows of the token outputs, at least the sum of query_lens; those
    past the sum (a step padded for a captured graph) have position 0, and block
    and slot -1, which the stores skip. width: columns of ``block_tables``, at least
    the pages of the longest request (by default W). Pages past W are not given.
    Lengths are taken within [0, 2^30); a row outside ``tables`` takes no page and
    has -1 throughout. A row may stand once in ``rows``, and a page once in the
    list.
    """
    if tables.dim() != 2 or tables.dtype != torch.int32:
        raise ValueError(f"tables must be a 2D int32 tensor, but got {tables.dtype} of shape {tuple(tables.shape)}")
    context_lens, query_lens = _ints("context_lens", context_lens), _ints("query_lens", query_lens)
    if rows is not None:
        rows = _ints("rows", rows)
    if free_blocks is not None:
        free_blocks = _ints("free_blocks", free_blocks)
    elif num_free is not None:
        raise ValueError("num_free goes with free_blocks")
    if num_free is not None:
        num_free = _ints("num_free", num_free)
    num_tokens, block_size = int(num_tokens), int(block_size)
    width = tables.shape[1] if width is None else int(width)
    if num_tokens < 0 or width < 0:
        raise ValueError(f"num_tokens and width must be non-negative, but got {num_tokens} and {width}")
    dev = _lib.require_device(tables, context_lens, query_lens, rows, free_blocks, num_free)
    b = context_lens.shape[0]
    sizes = (b * width, b + 1, b, num_tokens, num_tokens, num_tokens, 1)
    parts = torch.empty(sum(sizes), dtype=torch.int32, device=dev).split_with_sizes(sizes)  # (one allocation)
    left = parts[6] if free_blocks is not None else None
    block_tables = parts[0].view(b, width)
    _lib.launch("tsa_step_tables", "step_tables", dev, block_tables, *parts[1:6], left, tables, rows, context_lens,
                query_lens, free_blocks, num_free, block_size)
    return StepTables(block_tables, *parts[1:6], left)
