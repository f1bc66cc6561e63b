"""The paged K/V cache in 8 bits: written, read back, and attended to.

The pools (NB, Hkv, BS, D) are ``torch.float8_e4m3fn`` or ``torch.int8`` and
each row (token and kv head) has one float32 scale in (NB, Hkv, BS) tensors; a
row's values are ``code * scale``. Block tables, lengths and addressing are
those of the 16-bit cache (server/model/kernels/kv_cache.py:122-251,
paged_attention.py:124-192); a page takes ``D + 4`` bytes a row where bf16
takes ``2 D``.
"""

from __future__ import annotations

import torch

from .. import _lib
from .window_attention import _decode


def store_kv_cache_quantized(
    k_src: torch.Tensor,
    v_src: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    cu_seqlens: torch.Tensor,
    positions: torch.Tensor | None = None,
) -> None:
    """``store_kv_cache_paged`` into an 8-bit cache.

    k_src, v_src: (Hkv, T, D) bf16, f16 or f32, any strides (the (T, Hkv, D)
    projection output is passed as ``k.transpose(0, 1)`` without a copy).
    Tokens of sequence s are ``cu_seqlens[s]:cu_seqlens[s+1]``; token t sits at
    ``positions[t]`` or, with positions None, at ``t - cu_seqlens[s]``. A row's
    scale is its largest magnitude over 448 (e4m3) or 127 (int8); its codes are
    the quotients by it, rounded to nearest, ties to even. A row of zeros has
    scale 0; a row holding a NaN or an infinity has scale NaN and reads back as
    NaN. Tokens whose page is past the table or outside the pool are skipped,
    and no other row of the cache is touched. Give each slot once per call.
    """
    if k_src.dim() != 3 or v_src.dim() != 3:
        raise ValueError(f"k_src and v_src must be 3D tensors, but got shapes {k_src.shape} and {v_src.shape}")
    if k_src.shape != v_src.shape:
        raise ValueError(f"k_src and v_src must have the same shape, but got {k_src.shape} and {v_src.shape}")
    dev = _lib.require_device(k_src, v_src, k_cache, v_cache, k_scale, v_scale, block_tables, cu_seqlens, positions)
    _lib.launch("tsa_store_kv_quantized", "store_kv_cache_quantized", dev, k_src, v_src, k_cache, v_cache, k_scale,
                v_scale, block_tables, cu_seqlens, positions)


def load_kv_cache_quantized(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    cu_seqlens: torch.Tensor,
    num_tokens: int,
    positions: torch.Tensor | None = None,
    *,
    dtype: torch.dtype = torch.bfloat16,
    k_out: torch.Tensor | None = None,
    v_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of an 8-bit cache as packed (num_tokens, Hkv, D) keys and values of ``dtype``.

    Addressing as ``store_kv_cache_quantized``'s: what it wrote for a packed
    batch, this reads for the same cu_seqlens and positions: a sequence on its
    way to a 16-bit pool (``store_kv_cache_paged``) or out of the cache. (The
    varlen functions place a sequence's queries at its start, so a chunk's
    queries behind rows read here are not theirs to attend from.) Each value
    is ``code * scale`` in float32, rounded to ``dtype``. A token that no
    sequence holds, or whose page is past the table or outside the pool, reads
    as 0. k_out and v_out, if given, set the dtype.
    """
    if k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("k_cache and v_cache must be 4D tensors (num_blocks, num_kv_heads, block_size, head_dim)")
    dev = _lib.require_device(k_cache, v_cache, k_scale, v_scale, block_tables, cu_seqlens, positions, k_out, v_out)
    shape = (int(num_tokens), k_cache.shape[1], k_cache.shape[3])
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None and tuple(t.shape) != shape:
            raise ValueError(f"{name} must be {shape}, but got {tuple(t.shape)}")
    like = k_out if k_out is not None else v_out
    if like is not None:
        dtype = like.dtype
    k_out = torch.empty(shape, dtype=dtype, device=dev) if k_out is None else k_out
    v_out = torch.empty(shape, dtype=dtype, device=dev) if v_out is None else v_out
    _lib.launch("tsa_load_kv_quantized", "load_kv_cache_quantized", dev, k_out, v_out, k_cache, v_cache, k_scale,
                v_scale, block_tables, cu_seqlens, positions)
    return k_out, v_out


def paged_attention_quantized(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    block_size: int,
    seq_lens: torch.Tensor,
    *,
    window: int = 0,
    sinks: int = 0,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``paged_attention_forward`` over an 8-bit cache, without a 16-bit copy of it.

    The codes are widened exactly, the scales multiply the fp32 scores and
    weights: the result is that of attention over the values the cache holds.
    With ``window`` (0: none) and ``sinks``, over the last and first tokens
    only, as ``paged_attention_window``. A sequence of length 0 gives 0.
    """
    return _decode("paged_attention_quantized", query, k_cache, v_cache, k_scale, v_scale, block_tables, block_size,
                   seq_lens, window, sinks, softmax_scale, out)
