"""Log probabilities of given tokens, beside ``sample_tokens`` (server/model/
sampling.py:119-194): those of a step's sampled tokens, or of a prompt's.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # (N,) float32: of the given tokens
    entropy: torch.Tensor       # (N,) float32: of each row's distribution, in nats
    top_logprobs: torch.Tensor  # (N, num_top) float32: of the most likely tokens, falling
    top_tokens: torch.Tensor    # (N, num_top) int64


_WS_BYTES: dict[tuple, int] = {}


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, num_top: int = 0) -> TokenLogprobs:
    """log softmax(logits)[n, tokens[n]], the entropy of softmax(logits[n]), and
    the ``num_top`` (up to 64) most likely tokens of each row with their log
    probabilities, the lowest index first where logits tie.

    logits (N, V) bf16, f16 or f32; tokens (N,) int32 or int64. All is computed in
    float32. A logit of -inf has probability 0 and adds nothing to the entropy; a
    token outside the vocabulary has log probability -inf. A row that holds a NaN
    or +inf, or nothing but -inf, has no distribution: its log probabilities and
    entropy are NaN (its top tokens are still its largest logits; NaN ranks below
    every number).
    """
    if logits.dim() != 2:
        raise ValueError(f"Expected logits shape [N, vocab_size], got {logits.dim()}D")
    if tokens.shape != logits.shape[:1]:
        raise ValueError(f"Expected tokens shape [{logits.shape[0]}], got {tuple(tokens.shape)}")
    num_top = int(num_top)
    if num_top < 0:
        raise ValueError(f"num_top must be non-negative, but got {num_top}")
    dev = _lib.require_device(logits, tokens)
    n, vocab = logits.shape
    scalars = torch.empty(2, n, dtype=torch.float32, device=dev)
    top_logprobs = torch.empty(n, num_top, dtype=torch.float32, device=dev)
    top_tokens = torch.empty(n, num_top, dtype=torch.int64, device=dev)
    logprobs, entropy = scalars.unbind()
    key = (n, vocab, num_top)
    nbytes = _WS_BYTES.get(key)
    if nbytes is None:
        if len(_WS_BYTES) >= 4096:
            _WS_BYTES.clear()
        nbytes = _WS_BYTES[key] = int(_lib.load().tsa_token_logprobs_workspace_bytes(*key))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _lib.launch("tsa_token_logprobs", "token_logprobs", dev, logprobs, entropy, top_logprobs, top_tokens, logits, tokens,
                ws.data_ptr() if ws is not None else 0, nbytes)
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_tokens)
