"""A paged key/value cache for sequences of any lengths, and attention over it.

The cache of a layer is two buffers of pages (``paged_buffers``); a table says
which pages hold a sequence's positions, so sequences grow page by page and may
share pages.  New tokens come packed: ``PagedBatch`` says which rows are whose.
``paged_store`` puts their keys and values in, turned to their positions
(``Rotary``), and turns their queries; ``paged_attention`` lets them attend:
whole prompts, chunks of prompts, single tokens and mixtures of these in one
call.  ``GraphDecoder(page_size=...)`` decodes prompts of different lengths with
them.  The reference keeps a tensor per layer that grows by concatenation
(atlasinfer_core/memory/unified_memory_manager.py:111-563).

What describes a batch is device memory, read when a kernel runs, so a captured
HIP graph replays with new lengths and pages; only its shapes and the bounds
``max_new`` and ``max_length`` are the host's.  Nothing here records gradients.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from .. import _lib

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}  # AQ_F16, AQ_BF16
_INT_MAX = (1 << 31) - 1


def _refuse(what: str):
    raise ValueError(what)


class PagedBatch:
    """The new tokens of S sequences as packed rows, and where their pages are.

    ``starts`` int32 [S + 1]: sequence s has rows starts[s] .. starts[s + 1] - 1;
    ``lengths`` int32 [S]: its positions after them; ``table`` int32 [S, W]: its
    pages in order; all contiguous on one HIP device.  ``max_new`` and
    ``max_length``: host bounds on a sequence's new rows and length.  A sequence
    that passes them, or has more new rows than positions, is left out."""

    __slots__ = ("starts", "lengths", "table", "max_new", "max_length", "device", "sequences", "width", "_args")

    def __init__(self, starts: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, max_new: int, max_length: int):
        dev = table.device
        if table.dim() != 2 or lengths.dim() != 1 or starts.dim() != 1:
            _refuse(f"PagedBatch: starts {tuple(starts.shape)}, lengths {tuple(lengths.shape)}, table {tuple(table.shape)}")
        S, W = table.shape
        if not (0 < S <= 65535 and W > 0 and lengths.shape[0] == S and starts.shape[0] == S + 1):
            _refuse(f"PagedBatch: starts {tuple(starts.shape)}, lengths {tuple(lengths.shape)}, table {tuple(table.shape)} "
                    "(S + 1, S and S rows, S from 1 to 65535)")
        for t in (starts, lengths, table):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != dev or dev.type != "cuda":
                _refuse("PagedBatch: starts, lengths and table must be contiguous int32 on one HIP device")
        max_new, max_length = int(max_new), int(max_length)
        if max_new < 1 or max_length < 1:
            _refuse(f"PagedBatch: at most {max_new} new tokens, {max_length} positions")
        args = (starts.data_ptr(), lengths.data_ptr(), S, table.data_ptr(), W, max_new, max_length)
        for name, x in zip(self.__slots__, (starts, lengths, table, max_new, max_length, dev, S, W, args)):
            object.__setattr__(self, name, x)

    def __setattr__(self, name, value):
        raise AttributeError("PagedBatch: change what the tensors hold, or make another one")


class Rotary(NamedTuple):
    """Rotary positions: ``frequencies`` f32 [rotary / 2] on the device (the angle
    of pair i per position); ``interleaved``: pairs are neighbours instead of
    halves apart; ``factor`` multiplies the turned elements."""
    frequencies: torch.Tensor
    interleaved: bool = False
    factor: float = 1.0


def rotary_frequencies(rotary: int, base: float = 10000.0, scaling: Optional[dict] = None, device=None
                       ) -> Tuple[torch.Tensor, float]:
    """(frequencies f32 [rotary / 2], factor) of rotary positions over ``rotary``
    elements of the head: base^(-2 i / rotary), for long contexts changed as
    ``scaling`` says (the ``rope_scaling`` of a model's configuration):

    * ``linear``: all divided by ``factor``;
    * ``llama3``: those whose wavelength passes ``original_max_position_embeddings /
      low_freq_factor`` divided by ``factor``, those below ``/ high_freq_factor`` as
      they are, blended in between;
    * ``yarn``: divided by ``factor`` below ``beta_slow`` turns over the original
      length, as they are above ``beta_fast``, blended by index in between; the
      factor of the turned elements is 0.1 ln(factor) + 1, or where both ``mscale`` = a
      and ``mscale_all_dim`` = b are given (and not 0) (0.1 a ln(factor) + 1) / (0.1 b
      ln(factor) + 1), unless ``attention_factor`` gives it.
    """
    if rotary <= 0 or rotary % 2:
        _refuse(f"rotary_frequencies: {rotary} elements")
    f = float(base) ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    m = 1.0
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))

    def given(key):
        x = scaling.get(key)
        if x is None:
            _refuse(f"rotary_frequencies: rope type {kind!r} without {key}")
        return x

    if kind == "linear":
        f = f / given("factor")
    elif kind == "llama3":
        s, low, high = given("factor"), given("low_freq_factor"), given("high_freq_factor")
        turns = given("original_max_position_embeddings") * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)  # 0: divided, 1: as they are
        f = f * keep + f / s * (1 - keep)
    elif kind == "yarn":
        s, n = given("factor"), given("original_max_position_embeddings")
        fast, slow = scaling.get("beta_fast") or 32, scaling.get("beta_slow") or 1

        def index(turns):  # the pair that makes so many turns over n positions
            return rotary * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = index(fast), index(slow)
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary - 1)
        ramp = ((torch.arange(rotary // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / s * ramp + f * (1 - ramp)
        m = scaling.get("attention_factor")
        if m is None:
            a, b = scaling.get("mscale"), scaling.get("mscale_all_dim")

            def size(weight):
                return 0.1 * weight * math.log(s) + 1.0 if s > 1 else 1.0

            m = size(a) / size(b) if a and b else size(1.0)
    elif kind != "default":
        raise NotImplementedError(f"rotary_frequencies: rope type {kind!r} (default, linear, llama3, yarn supported)")
    return f.float().to(device), float(m)


def paged_buffers(pages: int, kv_heads: int, page_size: int, head_dim: int, dtype=torch.float16, device="cuda"
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Empty keys and values of a paged cache, [pages, kv_heads, page_size, head_dim] each."""
    if head_dim not in (64, 128) or dtype not in _DTYPES:
        _refuse(f"paged cache: head size {head_dim} (64 and 128 supported), {dtype} (fp16 and bf16 supported)")
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1) or pages <= 0 or kv_heads <= 0:
        _refuse(f"paged cache: {pages} pages of {page_size} slots (a power of two from 16 to 1024), {kv_heads} heads")
    shape = (pages, kv_heads, page_size, head_dim)
    return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)


# The checks below run in every layer of a step: no message is put together
# unless it is raised.


def _cache(what, cache, batch):
    """(keys, values, Hkv, page size, D) of a cache, which is checked."""
    k, v = cache
    if not (k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.dtype in _DTYPES and k.is_contiguous()
            and v.is_contiguous() and k.device == v.device):
        _refuse(f"{what}: the cache must be two contiguous fp16 or bf16 buffers [pages, heads, page size, head size] on one device")
    if k.device != batch.device:
        _refuse(f"{what}: the cache is on {k.device}, the batch on {batch.device}")
    _, Hkv, P, D = k.shape
    if D not in (64, 128) or P < 16 or P > 1024 or P & (P - 1):
        _refuse(f"{what}: cache {tuple(k.shape)} (head sizes 64 and 128, pages of a power of two from 16 to 1024 supported)")
    if batch.max_length > batch.width * P:
        _refuse(f"{what}: {batch.max_length} positions in {batch.width} pages of {P}")
    return k, v, Hkv, P, D


def _no_gradients(what):
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} records no gradients: call it under torch.no_grad()")


def paged_store(k: torch.Tensor, v: torch.Tensor, cache: Sequence[torch.Tensor], batch: PagedBatch, *,
                q: Optional[torch.Tensor] = None, rope: Optional[Rotary] = None,
                q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write the packed rows' keys and values (k, v [T, Hkv, D], the cache's type,
    any strides) to their places in the cache.  ``rope``: keys are turned to their
    positions, over the first ``2 len(frequencies)`` elements (a multiple of 16).
    ``q`` [T, H, D] is turned likewise and returned as [T, H, D] (in ``q_out`` if
    given, which must overlap neither the inputs nor the cache; rows that belong to no
    sequence are not written)."""
    what = "paged_store"
    kc, vc, Hkv, P, D = _cache(what, cache, batch)
    dev, dtype = kc.device, kc.dtype
    T = k.shape[0] if k.dim() == 3 else -1
    if k.shape != (T, Hkv, D) or v.shape != k.shape or k.dtype != dtype or v.dtype != dtype or k.device != dev or v.device != dev:
        _refuse(f"{what}: k {tuple(k.shape)}, v {tuple(v.shape)} must be {dtype} [T, {Hkv}, {D}] on {dev}")
    H = 0
    if q is not None:
        H = q.shape[1] if q.dim() == 3 else -1
        if q.shape != (T, H, D) or q.dtype != dtype or q.device != dev or not 0 < H <= 1024:
            _refuse(f"{what}: q {tuple(q.shape)} must be {dtype} [{T}, H, {D}] on {dev}")
        if q_out is None:
            q_out = torch.empty(T, H, D, dtype=dtype, device=dev)
        elif not (q_out.shape == q.shape and q_out.dtype == dtype and q_out.device == dev and q_out.is_contiguous()
                  and q_out.data_ptr() % 16 == 0):
            _refuse(f"{what}: q_out must be contiguous {dtype} {tuple(q.shape)} on {dev}")
    elif q_out is not None:
        _refuse(f"{what}: q_out without q")
    freq, R, inter, factor = None, 0, False, 1.0
    if rope is not None:
        freq, inter, factor = rope
        R = 2 * freq.numel()
        if freq.dtype != torch.float32 or freq.dim() != 1 or not freq.is_contiguous() or freq.device != dev or R % 16 or not 0 < R <= D:
            _refuse(f"{what}: frequencies must be contiguous float32 [n] on {dev}, n a multiple of 8 up to {D // 2}")
    if k.requires_grad or v.requires_grad or (q is not None and q.requires_grad):
        _no_gradients(what)
    if T == 0:
        return q_out
    if q is not None:
        q = _lib.strided_rows(q)
        if q_out.data_ptr() == q.data_ptr():
            _refuse(f"{what}: q_out must not be q")
    k, v = _lib.strided_rows(k), _lib.strided_rows(v)
    starts, lengths, S, table, W, max_new, max_length = batch._args
    with _lib.on_device(dev):
        _lib.check(_lib.load().aq_paged_store(
            _lib.ptr(q), k.data_ptr(), v.data_ptr(), _DTYPES[dtype], T, H, Hkv, D, *(q.stride()[:2] if H else (0, 0)),
            *k.stride()[:2], *v.stride()[:2], starts, lengths, S, table, W, max_new, max_length, _lib.ptr(freq), R, int(inter),
            factor, _lib.ptr(q_out), kc.data_ptr(), vc.data_ptr(), kc.shape[0], P, _lib.stream_of(dev)), "aq_paged_store")
    return q_out


def paged_attention_workspace(rows: int, heads: int, kv_heads: int, head_dim: int, batch: PagedBatch) -> int:
    """Bytes of workspace of ``paged_attention`` for these sizes (calls that
    follow each other can share one)."""
    return int(_lib.load().aq_paged_attention_workspace(rows, batch.sequences, heads, kv_heads, head_dim, batch.max_new,
                                                        batch.max_length))


def paged_attention(q: torch.Tensor, cache: Sequence[torch.Tensor], batch: PagedBatch, *, scale: float,
                    window: Optional[int] = None, sinks: int = 0, workspace: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of the packed rows q [T, H, D] (the cache's type, any
    strides, H a multiple of Hkv) over their sequences' keys and values, their own
    positions' (``paged_store``) included; [T, H, D].  A row at position p sees the
    keys at or before it that are less than ``window`` positions back (None: all) or
    among the first ``sinks``.  ``workspace`` (uint8, paged_attention_workspace
    bytes) and ``out`` (which must overlap neither q nor the cache): given, or allocated;
    rows that belong to no sequence are not written."""
    what = "paged_attention"
    kc, vc, Hkv, P, D = _cache(what, cache, batch)
    dev, dtype = kc.device, kc.dtype
    T, H = q.shape[:2] if q.dim() == 3 else (-1, 0)
    if q.shape != (T, H, D) or H == 0 or H > 1024 or H % Hkv or q.dtype != dtype or q.device != dev:
        _refuse(f"{what}: q {tuple(q.shape)} must be {dtype} [T, H, {D}] on {dev}, H a multiple of {Hkv}")
    if window is None:
        window = batch.max_length
    if window < 1 or sinks < 0:
        _refuse(f"{what}: window {window}, {sinks} sinks")
    if out is None:
        out = torch.empty(T, H, D, dtype=dtype, device=dev)
    elif not (out.shape == q.shape and out.dtype == dtype and out.device == dev and out.is_contiguous()
              and out.data_ptr() % 16 == 0):
        _refuse(f"{what}: out must be contiguous {dtype} {tuple(q.shape)} on {dev}")
    if workspace is not None and not (workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.device == dev):
        _refuse(f"{what}: the workspace must be contiguous uint8 on {dev}")
    if q.requires_grad or kc.requires_grad or vc.requires_grad:
        _no_gradients(what)
    if T == 0:
        return out
    row, head, last = q.stride()
    if last != 1 or (row | head) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        row, head, _ = q.stride()
    if out.data_ptr() == q.data_ptr():
        _refuse(f"{what}: out must not be q")
    starts, lengths, S, table, W, max_new, max_length = batch._args
    L = _lib.load()
    if workspace is None:
        size = L.aq_paged_attention_workspace(T, S, H, Hkv, D, max_new, max_length)
        workspace = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
    ws, size = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
    with _lib.on_device(dev):
        _lib.check(L.aq_paged_attention(q.data_ptr(), _DTYPES[dtype], T, H, Hkv, D, row, head,
                                        kc.data_ptr(), vc.data_ptr(), kc.shape[0], P, starts, lengths, S, table, W, max_new, max_length,
                                        min(window, _INT_MAX), min(sinks, _INT_MAX), scale, ws, size, out.data_ptr(),
                                        _lib.stream_of(dev)), "aq_paged_attention")
    return out
