"""Log probabilities of given tokens, with entropies, ranks and alternatives.

What a user of a decoder asks for beside the token that ``sample_tokens`` gives,
and what the score of a text is made of.  The reference decodes with HF
``generate`` (examples/run_atlas_inference.py:244-264), where it takes a
log_softmax of the whole row, a gather and a top-k; ``token_logprobs`` reads the
logits once (``aq_token_logprobs``).  ``GraphDecoder(logprobs=n)`` uses it for
each token it chooses, ``GraphDecoder.score`` for given texts.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from .sampling import MAX_VOCAB, _DTYPES

MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # f32 [B], of the given tokens
    entropies: torch.Tensor     # f32 [B], of the rows, in nats
    ranks: torch.Tensor         # int64 [B]: tokens that stand before the given one
    top_logprobs: torch.Tensor  # f32 [B, top], falling
    top_tokens: torch.Tensor    # int64 [B, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Of every row of ``logits`` (fp16, bf16 or fp32 [B, V], on a HIP device, rows
    contiguous) the log probability and rank of ``tokens[b]`` (int64 [B]), the
    entropy, and the ``top`` most likely tokens (0 .. 64) with theirs, in the order of
    falling logit, equal ones by index.  NaN logits count as -inf; a row without a
    logit above -inf has NaN; a token outside the row has NaN and rank -1.  Records no
    gradients."""
    if logits.dim() != 2 or logits.device.type != "cuda" or logits.dtype not in _DTYPES:
        raise ValueError(f"token_logprobs: logits must be fp16, bf16 or fp32 [B, V] on a HIP device, got "
                         f"{logits.dtype} {tuple(logits.shape)} on {logits.device}")
    B, V = logits.shape
    dev = logits.device
    if not 0 < V <= MAX_VOCAB or B > 65535:
        raise ValueError(f"token_logprobs: {B} rows (up to 65535) of {V} logits (1 .. {MAX_VOCAB})")
    if tokens.dtype != torch.int64 or tokens.shape != (B,) or tokens.device != dev or not tokens.is_contiguous():
        raise ValueError(f"token_logprobs: tokens must be contiguous int64 [{B}] on {dev}")
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"token_logprobs: {top} alternatives (0 .. {MAX_TOP}, at most a row's {V})")
    if torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("token_logprobs records no gradients: call it under torch.no_grad()")
    # (allocations are most of a small call: those of known shape and type are the cheapest)
    logprobs, top_logprobs = torch.empty(B, dtype=torch.float32, device=dev), torch.empty(B, top, dtype=torch.float32, device=dev)
    out = TokenLogprobs(logprobs, torch.empty_like(logprobs), torch.empty_like(tokens), top_logprobs,
                        torch.empty(B, top, dtype=torch.int64, device=dev))
    if B == 0:
        return out
    if (logits.stride(1) != 1 and V > 1) or (logits.stride(0) < V and B > 1):
        logits = logits.contiguous()
    L, dtype = _lib.load(), _DTYPES[logits.dtype]
    size = L.aq_token_logprobs_workspace(B, V, dtype, top)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
    with _lib.on_device(dev):
        _lib.check(L.aq_token_logprobs(logits.data_ptr(), dtype, B, V, max(logits.stride(0), V), tokens.data_ptr(), top,
                                       *[_lib.ptr(t) for t in out], _lib.ptr(ws), size, _lib.stream_of(dev)),
                   "aq_token_logprobs")
    return out
