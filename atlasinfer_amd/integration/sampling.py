"""Sampling of the next token: temperature, top-k, top-p and min-p.

The reference decodes with HF ``generate`` (examples/run_atlas_inference.py
:244-264), whose sampling is a chain of logits processors, a sort of the
vocabulary and torch's multinomial.  ``sample_tokens`` does it in the library
(``aq_sample``) from one given random number per sequence, so a step can be
captured in a HIP graph and the same numbers give the same tokens;
``GraphDecoder(..., sampling=True)`` uses it, with generate's ``temperature``,
``top_k``, ``top_p`` and ``min_p``.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _lib

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # AQ_F16, AQ_BF16, AQ_F32
MAX_VOCAB = 1 << 18
Setting = Union[float, int, torch.Tensor]


def _setting(name: str, x: Setting, dtype: torch.dtype, B: int, dev):
    """(device address or None, the value for all rows, the tensor kept)."""
    if isinstance(x, torch.Tensor):
        if x.dtype != dtype or x.shape != (B,) or x.device != dev or not x.is_contiguous():
            raise ValueError(f"sample_tokens: {name} must be a number or a contiguous {dtype} [{B}] on {dev}")
        return x.data_ptr(), 0
    return None, x


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The next token of every row of ``logits`` (fp16, bf16 or fp32 [B, V], on a
    HIP device, rows contiguous), int64 [B].

    With w_i = exp((x_i - max) / temperature) and the tokens in the order of
    falling logit (equal ones by index), those are kept that are among the first
    ``top_k`` (0: all), before which less than ``top_p`` of the mass of these lies
    (1: all), and whose w is at least ``min_p`` (0: all) -- the largest always.
    The token is the first kept one, by index, at which the running mass exceeds
    ``u[b]`` (float32 [B], uniform in [0, 1)) times the whole kept mass.
    ``temperature`` 0: the largest logit, the lowest index of equal ones.  NaN
    logits count as -inf.  Each setting is a number or one per row (float32 [B],
    ``top_k`` int32 [B])."""
    if logits.dim() != 2 or logits.device.type != "cuda" or logits.dtype not in _DTYPES:
        raise ValueError(f"sample_tokens: logits must be fp16, bf16 or fp32 [B, V] on a HIP device, got "
                         f"{logits.dtype} {tuple(logits.shape)} on {logits.device}")
    B, V = logits.shape
    dev = logits.device
    if not 0 < V <= MAX_VOCAB:
        raise ValueError(f"sample_tokens: {V} logits a row (1 .. {MAX_VOCAB})")
    if u.dtype != torch.float32 or u.shape != (B,) or u.device != dev or not u.is_contiguous():
        raise ValueError(f"sample_tokens: u must be contiguous float32 [{B}] on {dev}")
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    elif out.dtype != torch.int64 or out.shape != (B,) or out.device != dev or not out.is_contiguous():
        raise ValueError(f"sample_tokens: out must be contiguous int64 [{B}] on {dev}")
    tp, t0 = _setting("temperature", temperature, torch.float32, B, dev)
    kp, k0 = _setting("top_k", top_k, torch.int32, B, dev)
    pp, p0 = _setting("top_p", top_p, torch.float32, B, dev)
    mp, m0 = _setting("min_p", min_p, torch.float32, B, dev)
    if B == 0:
        return out
    if (logits.stride(1) != 1 and V > 1) or (logits.stride(0) < V and B > 1):
        logits = logits.contiguous()
    stride = max(logits.stride(0), V)
    L, dtype = _lib.load(), _DTYPES[logits.dtype]
    k0 = min(max(int(k0), 0), V)
    size = L.aq_sample_workspace(B, V, dtype, k0)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
    with _lib.on_device(dev):
        _lib.check(L.aq_sample(logits.data_ptr(), dtype, B, V, stride, u.data_ptr(), tp, kp, pp, mp, t0, k0, p0, m0,
                               out.data_ptr(), _lib.ptr(ws), size, _lib.stream_of(dev)), "aq_sample")
    return out
