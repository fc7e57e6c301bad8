"""Attention of a prompt through a sliding window with sinks.

``window_attention`` is the kernel's call (``aq_window_attention``);
``window_prompts`` makes an HF OPT / Llama / Mistral model's own forward use it
for a while, which ``GraphDecoder(window=...)`` does for its prompts.  No counterpart
in the reference, whose attention (integration/atlas_wrappers.py:161-262) sees
every position through torch's SDPA and a dense mask.
"""
from __future__ import annotations

import contextlib
import ctypes
import threading
from typing import Optional

import torch

from .. import _lib


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                     scale: Optional[float] = None, starts: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v in fp16 for the last M of N positions.

    q [B, H, M, D], k and v [B, Hkv, N, D] (fp16 on a HIP device, any strides, H a
    multiple of Hkv, D 64 or 128, M <= N); returns [B, M, H, D].  Query i stands
    at position N - M + i and sees the keys j at or before it that are less than
    ``window`` positions back (None: all) or among the first ``sinks``.
    ``starts`` (int32 [B]): sequence b begins at that position (left padding):
    earlier keys are not seen, and sinks count from there.  A query that sees
    nothing gets zeros."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"window_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    B, H, M, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    dev = q.device
    if k.shape[0] != B or k.shape[3] != D or D not in (64, 128) or Hkv == 0 or H % Hkv or M > N:
        raise ValueError(f"window_attention: q {tuple(q.shape)}, k {tuple(k.shape)} (D 64 or 128, H a multiple of "
                         "Hkv, no more queries than keys)")
    for t in (q, k, v):
        if t.dtype != torch.float16 or t.device.type != "cuda" or t.device != dev:
            raise ValueError("window_attention: q, k and v must be fp16 on one HIP device")
    window = N if window is None else int(window)
    if window < 1 or sinks < 0:
        raise ValueError(f"window_attention: window {window}, {sinks} sinks")
    if starts is not None and (starts.dtype != torch.int32 or starts.shape != (B,) or starts.device != dev
                               or not starts.is_contiguous()):
        raise ValueError(f"window_attention: starts must be contiguous int32 [{B}] on {dev}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        raise RuntimeError("window_attention records no gradients: call it under torch.no_grad()")
    out = torch.empty(B, M, H, D, dtype=torch.float16, device=dev)
    if out.numel() == 0:
        return out
    q, k, v = (_lib.strided_rows(t) for t in (q, k, v))
    arr = [_lib.ptr_array(t.stride()[:3], ctypes.c_int64) for t in (q, k, v)]
    with _lib.on_device(dev):
        _lib.check(_lib.load().aq_window_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), B, H, Hkv, M, N, D, *arr,
                                                   window, int(sinks), D ** -0.5 if scale is None else scale,
                                                   _lib.ptr(starts), out.data_ptr(), _lib.stream_of(dev)),
                   "aq_window_attention")
    return out


_NAME = "atlas_window"  # this attention's name among HF's
_local = threading.local()  # .open: the thread's open contexts, the innermost last
_switch = threading.Lock()  # held while a model's attention is changed


class _Context:
    def __init__(self, config, window, sinks, before):
        self.config, self.window, self.sinks, self.before = config, window, sinks, before


def _open():
    if not hasattr(_local, "open"):
        _local.open = []
    return _local.open


def _attention(module, query, key, value, attention_mask, scaling=None, dropout=0.0, **kwargs):
    """HF's attention interface: [B, H, M, D] and [B, Hkv, N, D] to [B, M, H, D]."""
    for c in reversed(_open()):
        if c.config is module.config:
            return window_attention(query, key, value, window=c.window, sinks=c.sinks, scale=scaling), None
    raise RuntimeError("window_prompts: the model runs in a thread that has not entered the context it is in")


@contextlib.contextmanager
def window_prompts(model, window: Optional[int], sinks: int = 0):
    """Within the context ``model``'s forward (HF OPT, Llama or Mistral, fp16 on a
    HIP device) attends through a sliding window with sinks, whatever its
    configuration says; prompts without padding (the attention mask is not
    looked at).  Contexts of a model nest, the innermost counts.  A model's
    attention is its threads' in common, so while one thread is in a context of it
    another can neither enter one nor run it (RuntimeError)."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface
    AttentionInterface.register(_NAME, _attention)
    AttentionMaskInterface.register(_NAME, lambda *args, **kwargs: None)  # no dense mask is made
    mine, config = _open(), model.config
    with _switch:
        outer = next((c for c in mine if c.config is config), None)
        before = outer.before if outer is not None else config._attn_implementation
        if outer is None and before == _NAME:
            raise RuntimeError("window_prompts: the model is in another thread's context")
        model.set_attn_implementation(_NAME)
        context = _Context(config, window, sinks, before)
        mine.append(context)
    try:
        yield model
    finally:
        with _switch:
            mine.remove(context)
            if all(c.config is not config for c in mine):
                model.set_attn_implementation(before)
