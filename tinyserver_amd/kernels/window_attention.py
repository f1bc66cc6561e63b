"""Attention with a sliding window and a few first tokens that stay visible.

Beside ``paged_attention_forward`` and ``flash_attn_varlen_func`` (server/model/
kernels/paged_attention.py:124-192, varlen_attention.py:145-218): a query at
position i sees the keys j <= i with ``j > i - window`` or ``j < sinks``. Keys
outside that are not read. A query that sees nothing gives 0.
"""

from __future__ import annotations

import math

import torch

from .. import _lib

_WS_BYTES: dict[tuple, int] = {}


def _workspace(dev: torch.device, *shape) -> torch.Tensor | None:
    """The workspace of a call of this shape (tsa_paged_rows_workspace_bytes; None where it needs none). Allocated for
    the call: the caching allocator orders its reuse on the stream, and a captured graph keeps its own."""
    key = (dev.index, *shape)
    n = _WS_BYTES.get(key)
    if n is None:
        if len(_WS_BYTES) >= 4096:
            _WS_BYTES.clear()
        with torch.cuda.device(dev):  # (the stream's waves are those of the device's CUs)
            n = _WS_BYTES[key] = int(_lib.load().tsa_paged_rows_workspace_bytes(*shape))
    return torch.empty(n, dtype=torch.uint8, device=dev) if n else None


def _check_cache(query, k_cache, v_cache, block_tables, block_size):
    if query.dim() != 3:
        raise ValueError(f"query must be a 3D tensor, but got shape {query.shape}")
    if k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("k_cache and v_cache must be 4D tensors (num_blocks, num_kv_heads, block_size, head_dim)")
    if block_tables.dim() != 2:
        raise ValueError(f"block_tables must be a 2D tensor, but got shape {block_tables.shape}")
    if int(block_size) != k_cache.shape[2]:
        raise ValueError(f"block_size {block_size} does not match the cache's {k_cache.shape[2]}")


def _decode(what, query, k_cache, v_cache, k_scale, v_scale, block_tables, block_size, seq_lens, window, sinks,
            softmax_scale, out):
    _check_cache(query, k_cache, v_cache, block_tables, block_size)
    window, sinks = int(window), int(sinks)
    if window < 0 or sinks < 0:
        raise ValueError(f"window and sinks must be non-negative, but got {window} and {sinks}")
    dev = _lib.require_device(query, k_cache, v_cache, k_scale, v_scale, block_tables, seq_lens, out)
    if block_tables.dtype != torch.int32:
        block_tables = block_tables.to(torch.int32)
    if seq_lens.dtype != torch.int32:
        seq_lens = seq_lens.to(torch.int32)
    num_seqs, num_heads, head_dim = query.shape
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    ws = _workspace(dev, num_seqs, 1, num_heads, k_cache.shape[1], head_dim, block_tables.shape[1], k_cache.shape[2],
                    window, sinks)
    _lib.launch("tsa_paged_decode_window", what, dev, out, query, k_cache, v_cache, k_scale, v_scale, block_tables,
                seq_lens, window, sinks,
                1.0 / math.sqrt(max(head_dim, 1)) if softmax_scale is None else float(softmax_scale),
                ws.data_ptr() if ws is not None else 0, ws.numel() if ws is not None else 0)
    return out


def paged_attention_window(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    block_size: int,
    seq_lens: torch.Tensor,
    window: int,
    sinks: int = 0,
    *,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``paged_attention_forward`` over the last ``window`` tokens of each
    sequence (the new one included) and its first ``sinks``. query: (B, Hq, D);
    caches (NB, Hkv, BS, D) of its dtype; block_tables (B, max_blocks) int32;
    seq_lens (B,) int32. Only the pages of visible tokens are read, so a
    sequence's other pages may be given back (their table entries may hold
    anything). A sequence of length 0 gives 0."""
    if int(window) < 1:
        raise ValueError(f"window must be positive, but got {window}")
    return _decode("paged_attention_window", query, k_cache, v_cache, None, None, block_tables, block_size, seq_lens,
                   window, sinks, softmax_scale, out)


def flash_attn_varlen_window(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int,
    max_seqlen_k: int,
    window: int,
    sinks: int = 0,
    softmax_scale: float | None = None,
    *,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``flash_attn_varlen_func`` (causal) over part of the keys: query i of a
    sequence sees the keys j <= i (positions within the sequence, top-left
    aligned) with ``j > i - window`` or ``j < sinks``. Key blocks that no query
    of a block sees are not visited."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k, v must be 3D tensors")
    _, num_heads_q, head_dim = q.shape
    if k.shape[1] == 0 or num_heads_q % k.shape[1] != 0:
        raise ValueError("num_heads_q must be divisible by num_heads_k for GQA")
    window, sinks = int(window), int(sinks)
    if window < 1:
        raise ValueError(f"window must be positive, but got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must be non-negative, but got {sinks}")
    dev = _lib.require_device(q, k, v, cu_seqlens_q, cu_seqlens_k, out)
    if cu_seqlens_q.dtype != torch.int32:
        cu_seqlens_q = cu_seqlens_q.to(torch.int32)
    if cu_seqlens_k.dtype != torch.int32:
        cu_seqlens_k = cu_seqlens_k.to(torch.int32)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    _lib.launch("tsa_varlen_prefill_window", "flash_attn_varlen_window", dev, out, q, k, v, cu_seqlens_q, cu_seqlens_k,
                int(max_seqlen_q), int(max_seqlen_k), window, sinks,
                1.0 / math.sqrt(max(head_dim, 1)) if softmax_scale is None else float(softmax_scale))
    return out
