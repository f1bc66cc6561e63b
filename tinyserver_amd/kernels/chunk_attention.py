"""Attention of a chunk of new tokens over the paged cache.

Beside ``paged_attention_forward`` (server/model/kernels/paged_attention.py:
124-192, one new token a sequence) and ``flash_attn_varlen_func``
(varlen_attention.py:145-218, whole prompts from position 0): a prompt brought in
pieces, a prompt whose first part is in the cache already, or a step that decodes
some sequences and brings pieces of others. The new tokens' keys and values go
into the cache first, at the positions behind the context
(``store_kv_cache_paged`` or ``qk_norm_rope_store`` with those positions).
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from .window_attention import _check_cache

_WS_BYTES: dict[tuple, int] = {}


def _workspace(dev: torch.device, *shape) -> torch.Tensor | None:
    """The workspace of a call of this shape (tsa_paged_chunk_workspace_bytes; None where it needs none). Allocated
    for the call: the caching allocator orders its reuse on the stream, and a captured graph keeps its own."""
    key = (dev.index, *shape)
    n = _WS_BYTES.get(key)
    if n is None:
        if len(_WS_BYTES) >= 4096:
            _WS_BYTES.clear()
        with torch.cuda.device(dev):  # (the workgroups are those of the device's CUs)
            n = _WS_BYTES[key] = int(_lib.load().tsa_paged_chunk_workspace_bytes(*shape))
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def paged_attention_chunk(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    block_size: int,
    context_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    max_seqlen: int | None = None,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """out[t] = softmax(query[t] K^T * scale) V over its sequence's tokens up to its own.

    query: (T, Hq, D), the new tokens of all sequences packed, sequence s's at rows
    ``cu_seqlens[s]:cu_seqlens[s+1]``; caches (NB, Hkv, BS, D) of its dtype;
    block_tables (B, max_blocks) int32; context_lens (B,) int32, the tokens that
    each sequence has in the cache before the new ones; cu_seqlens (B + 1,) int32.
    Row i of a sequence stands at position ``context_lens[s] + i`` and sees the
    positions up to that one. A sequence may have one new token (a decode step's),
    many, or none. Tokens whose page id is outside the pool are not seen; a row that
    sees nothing gives 0.

    ``max_seqlen``: at least the largest number of new tokens a sequence has; by
    default T. Give it where it is known: the kernel is chosen by it. Rows past
    max_seqlen in their sequence, and rows outside ``cu_seqlens[0]:cu_seqlens[B]``,
    are left as they were in ``out``.
    """
    _check_cache(query, k_cache, v_cache, block_tables, block_size)
    dev = _lib.require_device(query, k_cache, v_cache, block_tables, context_lens, cu_seqlens, out)
    if block_tables.dtype != torch.int32:
        block_tables = block_tables.to(torch.int32)
    if context_lens.dtype != torch.int32:
        context_lens = context_lens.to(torch.int32)
    if cu_seqlens.dtype != torch.int32:
        cu_seqlens = cu_seqlens.to(torch.int32)
    num_tokens, num_heads, head_dim = query.shape
    max_seqlen = num_tokens if max_seqlen is None else min(int(max_seqlen), num_tokens)
    if max_seqlen < 0:
        raise ValueError(f"max_seqlen must be non-negative, but got {max_seqlen}")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    ws = _workspace(dev, block_tables.shape[0], num_tokens, max_seqlen, num_heads, k_cache.shape[1], head_dim,
                    block_tables.shape[1], k_cache.shape[2])
    _lib.launch("tsa_paged_chunk", "paged_attention_chunk", dev, out, query, k_cache, v_cache, block_tables,
                context_lens, cu_seqlens, max_seqlen,
                1.0 / math.sqrt(max(head_dim, 1)) if softmax_scale is None else float(softmax_scale),
                ws.data_ptr() if ws is not None else 0, ws.numel() if ws is not None else 0)
    return out
