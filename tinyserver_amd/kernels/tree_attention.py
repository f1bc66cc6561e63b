"""Attention of a tree of drafted tokens over the paged cache.

The verification step of speculative decoding, beside ``paged_attention_forward``
(server/model/kernels/paged_attention.py:124-192): a sequence's drafted tokens
are nodes of a tree that hangs from its context, each attending to the context,
its ancestors and itself. The nodes' keys and values go into the cache first, at
the positions behind the context (``store_kv_cache_paged`` or
``qk_norm_rope_store`` with those positions; the rotary tables they are given
are those of the nodes' depths).
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from .window_attention import _check_cache, _workspace


def paged_attention_tree(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    block_size: int,
    context_lens: torch.Tensor,
    cu_nodes: torch.Tensor,
    tree_mask: torch.Tensor,
    *,
    max_nodes: int | None = None,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """out[n] = softmax(query[n] K^T * scale) V over what node n sees.

    query: (N, Hq, D), the nodes of all sequences packed, sequence s's at rows
    ``cu_nodes[s]:cu_nodes[s+1]``; caches (NB, Hkv, BS, D) of its dtype;
    block_tables (B, max_blocks) int32; context_lens (B,) int32, the cache's
    tokens before the drafted ones; cu_nodes (B + 1,) int32. Node i of a
    sequence has its key and value at cache position ``context_lens[s] + i``
    and sees the context and the nodes j whose bit is set in its mask:
    tree_mask (N, words) int64 (or (N,), one word), bit ``j % 64`` of word
    ``j // 64``. A node sees itself only by its own bit; one that sees nothing
    gives 0.

    ``max_nodes``: at least the largest number of nodes a sequence has; by
    default the most that the mask's width and N allow. Give it where it is
    known: the kernel, the splits and the workspace go by it, and small trees
    of a large batch would be taken for ones of 64 nodes. Rows past max_nodes or
    the mask's width in their sequence, and rows outside
    ``cu_nodes[0]:cu_nodes[B]``, are left as they were in ``out``.
    """
    _check_cache(query, k_cache, v_cache, block_tables, block_size)
    if tree_mask.dim() == 1:
        tree_mask = tree_mask.unsqueeze(1)
    if tree_mask.dim() != 2 or tree_mask.dtype != torch.int64:
        raise ValueError(f"tree_mask must be an int64 tensor (num_nodes, words), but got {tree_mask.dtype} of shape "
                         f"{tuple(tree_mask.shape)}")
    dev = _lib.require_device(query, k_cache, v_cache, block_tables, context_lens, cu_nodes, tree_mask, out)
    if block_tables.dtype != torch.int32:
        block_tables = block_tables.to(torch.int32)
    if context_lens.dtype != torch.int32:
        context_lens = context_lens.to(torch.int32)
    if cu_nodes.dtype != torch.int32:
        cu_nodes = cu_nodes.to(torch.int32)
    num_nodes, num_heads, head_dim = query.shape
    most = min(num_nodes, 64 * tree_mask.shape[1])
    max_nodes = most if max_nodes is None else min(int(max_nodes), most)
    if max_nodes < 0:
        raise ValueError(f"max_nodes must be non-negative, but got {max_nodes}")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    ws = _workspace(dev, block_tables.shape[0], max_nodes, num_heads, k_cache.shape[1], head_dim,
                    block_tables.shape[1], k_cache.shape[2], 0, 0)
    _lib.launch("tsa_paged_tree", "paged_attention_tree", dev, out, query, k_cache, v_cache, block_tables, context_lens,
                cu_nodes, tree_mask, max_nodes,
                1.0 / math.sqrt(max(head_dim, 1)) if softmax_scale is None else float(softmax_scale),
                ws.data_ptr() if ws is not None else 0, ws.numel() if ws is not None else 0)
    return out
