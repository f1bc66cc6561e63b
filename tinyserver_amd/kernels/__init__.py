"""Drop-in replacements for tinyserver's Triton kernel modules.

Same module names, function names, signatures and ValueError guards as
server/model/kernels/{kv_cache,paged_attention,varlen_attention}.py, backed by
the gfx950 HIP library; plus the fused QK RMSNorm + RoPE the reference runs as
eager PyTorch, the batched sampler of server/model/sampling.py, and a
continuous-batching step's prefill and decode attention in one launch; the
paged cache in 8 bits, attention with a sliding window and first tokens, and
attention of drafted tokens' trees; a step's block tables and slots built on the
GPU, attention of a chunk of new tokens over the paged cache, and log
probabilities of given tokens.
"""

from .chunk_attention import paged_attention_chunk
from .kv_cache import store_kv_cache, store_kv_cache_batched, store_kv_cache_paged
from .kv_cache_quantized import load_kv_cache_quantized, paged_attention_quantized, store_kv_cache_quantized
from .logprobs import TokenLogprobs, token_logprobs
from .mixed_attention import mixed_attention
from .paged_attention import paged_attention_forward, paged_decode_step
from .qk_norm_rope import qk_norm_rope, qk_norm_rope_store
from .sampling import sample_tokens
from .step_tables import StepTables, step_tables
from .tree_attention import paged_attention_tree
from .varlen_attention import flash_attn_varlen_func
from .window_attention import flash_attn_varlen_window, paged_attention_window

__all__ = [
    "store_kv_cache",
    "store_kv_cache_batched",
    "store_kv_cache_paged",
    "paged_attention_forward",
    "paged_decode_step",
    "flash_attn_varlen_func",
    "qk_norm_rope",
    "qk_norm_rope_store",
    "sample_tokens",
    "mixed_attention",
    "store_kv_cache_quantized",
    "load_kv_cache_quantized",
    "paged_attention_quantized",
    "paged_attention_window",
    "flash_attn_varlen_window",
    "paged_attention_tree",
    "paged_attention_chunk",
    "StepTables",
    "step_tables",
    "TokenLogprobs",
    "token_logprobs",
]
