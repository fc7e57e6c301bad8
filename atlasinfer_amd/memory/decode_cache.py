"""Static key/value caches of a decoding loop, and a step's attention over them.

Two kinds beside the plain static cache of ``aq_decode_attention``, which the
reference's cache (atlasinfer_core/memory/unified_memory_manager.py, every
position in fp16) has no counterpart of:

* a window: the cache's slots hold the first ``sinks`` positions and the last
  ``slots - sinks``; position p is in slot p while p < slots, then in slot
  ``sinks + (p - sinks) % (slots - sinks)``.  Memory and time per token stop
  growing there.
* 4 bits: groups of 32 elements of a key or value share a scale and a minimum,
  5 bits an element in all, so a cache of the same memory holds 3.2 times the
  positions (``kv4_buffers`` has the layout).

Both can be had together.  ``DecodeCache`` keeps a layer's buffers;
``GraphDecoder`` uses it for ``window=`` and ``kv_bits=4``.  The functions
below are the same on buffers of the caller's own.  Positions are device
memory, one for all sequences or one each, so that a captured HIP graph
replays a step; a sequence whose position is out of range (negative, past the
rotary tables, past a cache without a window) is left out: its row of the
result and its cache stay as they were.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from .. import _lib

GROUP = 32  # elements that share a scale and a minimum
BLOCK = 32  # slots whose values are interleaved


def _on(t: torch.Tensor):
    """The tensor's device as the current one (kernels are launched there)."""
    return torch.cuda.device(t.device)


def _need(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


def kv4_buffers(batch: int, kv_heads: int, slots: int, head_dim: int, device) -> Tuple[torch.Tensor, ...]:
    """Empty buffers of a 4-bit cache: key codes, key parameters, value codes,
    value parameters (layouts at aq_kv4_store in include/atlasinfer_amd.h)."""
    _need(head_dim in (64, 128), f"kv4: head size {head_dim} (64 and 128 supported)")
    _need(batch > 0 and kv_heads > 0 and 0 < slots <= 1 << 24, "kv4: batch, heads and slots must be positive")
    c = (slots + BLOCK - 1) // BLOCK * BLOCK
    return (torch.zeros(batch, kv_heads, c, head_dim // 2, dtype=torch.uint8, device=device),
            torch.zeros(batch, kv_heads, c, head_dim // GROUP, 2, dtype=torch.float16, device=device),
            torch.zeros(batch, kv_heads, c // BLOCK, head_dim * 16, dtype=torch.uint8, device=device),
            torch.zeros(batch, kv_heads, c // BLOCK, head_dim // GROUP, 4, 4, 4, dtype=torch.float16, device=device))


def _kv4_sizes(cache, slots: Optional[int]):
    """(B, Hkv, D, slots) of a 4-bit cache's buffers, which are checked."""
    _need(len(cache) == 4, "kv4: a cache is four buffers (kv4_buffers)")
    kc, kp, vc, vp = cache
    _need(kc.dim() == 4 and kc.shape[3] in (32, 64) and kc.shape[2] % BLOCK == 0, f"kv4: key codes {tuple(kc.shape)}")
    B, Hkv, c, D = kc.shape[0], kc.shape[1], kc.shape[2], kc.shape[3] * 2
    want = [((B, Hkv, c, D // 2), torch.uint8), ((B, Hkv, c, D // GROUP, 2), torch.float16),
            ((B, Hkv, c // BLOCK, D * 16), torch.uint8), ((B, Hkv, c // BLOCK, D // GROUP, 4, 4, 4), torch.float16)]
    for t, (shape, dtype) in zip(cache, want):
        _need(t.device.type == "cuda", "kv4: the cache must be on a HIP device")
        _need(tuple(t.shape) == shape and t.dtype == dtype and t.is_contiguous() and t.device == kc.device,
              f"kv4: a buffer {tuple(t.shape)} {t.dtype}, expected contiguous {shape} {dtype}")
    slots = c if slots is None else int(slots)
    _need(c - BLOCK < slots <= c, f"kv4: {slots} slots in buffers of {c}")
    return B, Hkv, D, slots


def _sinks(sinks: Optional[int], slots: int) -> int:
    if sinks is None:
        return -1
    _need(0 <= sinks < slots, f"{sinks} sinks in {slots} slots")
    return int(sinks)


def _strides(t: torch.Tensor):
    return _lib.ptr_array(t.stride()[:3], ctypes.c_int64)


def kv4_store(k: torch.Tensor, v: torch.Tensor, cache, start: int = 0, lengths: Optional[torch.Tensor] = None,
              slots: Optional[int] = None, sinks: Optional[int] = None) -> None:
    """Quantize positions start .. start + S - 1 (k, v fp16 [B, Hkv, S, D], any
    strides) into a 4-bit cache; of sequence b only the first ``lengths[b]``
    (int64 [B]).  ``sinks``: the cache is a window (None: it is not, and the
    positions must fit)."""
    B, Hkv, D, slots = _kv4_sizes(cache, slots)
    _need(k.dim() == 4 and k.shape == v.shape and k.shape[:2] == (B, Hkv) and k.shape[3] == D,
          f"kv4_store: k {tuple(k.shape)}, v {tuple(v.shape)} for a cache of [{B}, {Hkv}, *, {D}]")
    dev = cache[0].device
    for t in (k, v):
        _need(t.dtype == torch.float16 and t.device == dev, f"kv4_store: k and v must be fp16 on {dev}")
    if lengths is not None:
        _need(lengths.dtype == torch.int64 and lengths.shape == (B,) and lengths.is_contiguous() and lengths.device == dev,
              f"kv4_store: lengths must be int64 [{B}] on {dev}")
    S = k.shape[2]
    _need(start >= 0 and (sinks is not None or start + S <= slots),
          f"kv4_store: positions {start} .. {start + S - 1} in {slots} slots")
    sk = _sinks(sinks, slots)
    if S == 0:
        return
    k, v = _lib.strided_rows(k), _lib.strided_rows(v)
    with _on(k):
        _lib.check(_lib.load().aq_kv4_store(k.data_ptr(), v.data_ptr(), B, Hkv, S, D, _strides(k), _strides(v),
                                            int(start), _lib.ptr(lengths), *[t.data_ptr() for t in cache], slots, sk,
                                            _lib.stream_of(dev)), "aq_kv4_store")


def kv4_load(cache, count: Optional[int] = None, slots: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first ``count`` slots (all of them) of a 4-bit cache in fp16: keys
    and values [B, Hkv, count, D]."""
    B, Hkv, D, slots = _kv4_sizes(cache, slots)
    count = slots if count is None else int(count)
    _need(0 <= count <= slots, f"kv4_load: {count} of {slots} slots")
    dev = cache[0].device
    k, v = (torch.empty(B, Hkv, count, D, dtype=torch.float16, device=dev) for _ in range(2))
    if count:
        with _on(k):
            _lib.check(_lib.load().aq_kv4_load(*[t.data_ptr() for t in cache], B, Hkv, D, slots, count, k.data_ptr(),
                                               v.data_ptr(), _lib.stream_of(dev)), "aq_kv4_load")
    return k, v


def _step_arguments(what, q, k_new, v_new, pos, rope, B, Hkv, D, dev):
    """Checks of a step's tensors; (q, k_new, v_new contiguous, H, pos_stride,
    cos, sin, rows of the rotary tables)."""
    _need(q.dim() == 3 and q.shape[0] == B and q.shape[2] == D and q.shape[1] > 0 and q.shape[1] % Hkv == 0,
          f"{what}: q {tuple(q.shape)} for a cache of [{B}, {Hkv}, *, {D}]")
    _need(tuple(k_new.shape) == (B, Hkv, D) and tuple(v_new.shape) == (B, Hkv, D),
          f"{what}: k_new {tuple(k_new.shape)}, v_new {tuple(v_new.shape)}, expected {(B, Hkv, D)}")
    for t in (q, k_new, v_new):
        _need(t.dtype == torch.float16 and t.device == dev, f"{what}: q, k_new and v_new must be fp16 on {dev}")
    _need(pos.dtype == torch.int64 and pos.device == dev and pos.dim() == 1 and pos.shape[0] in (1, B)
          and pos.is_contiguous(), f"{what}: pos must be int64 [1] or [{B}] on {dev}")
    cos = sin = None
    rows = 0
    if rope is not None:
        cos, sin = rope
        rows = cos.shape[0]
        for t in (cos, sin):
            _need(t.dtype == torch.float16 and t.device == dev and t.is_contiguous() and tuple(t.shape) == (rows, D)
                  and rows > 0, f"{what}: rotary tables must be contiguous fp16 [positions, {D}] on {dev}")
    q, k_new, v_new = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
                       for t in (q, k_new, v_new))
    return q, k_new, v_new, q.shape[1], int(pos.shape[0] > 1), cos, sin, rows


def _workspace(what, size: int, workspace: Optional[torch.Tensor], dev) -> torch.Tensor:
    _need(size >= 0, f"{what}: sizes out of range")
    if workspace is None:
        return torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
    _need(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.device == dev
          and workspace.numel() >= size, f"{what}: the workspace must be uint8 of at least {size} bytes on {dev}")
    return workspace


def _result(what, out, q, dev):
    if out is None:
        return torch.empty_like(q)
    _need(out.shape == q.shape and out.dtype == torch.float16 and out.is_contiguous() and out.device == dev
          and out.data_ptr() % 16 == 0, f"{what}: out must be contiguous fp16 {tuple(q.shape)} on {dev}")
    return out


def kv4_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, cache, pos: torch.Tensor, *,
                  scale: float, slots: Optional[int] = None, sinks: Optional[int] = None, q_scale: float = 1.0,
                  rope=None, workspace: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None
                  ) -> torch.Tensor:
    """A decode step's attention over a 4-bit cache: k_new, v_new fp16 [B, Hkv,
    D] are quantized into the slot of ``pos`` (int64 [1] or [B], on the device)
    and q fp16 [B, H, D] attends to every slot in use.  ``rope``: (cos, sin) fp16
    [positions, D], q and k_new are rotated at pos first (rotate-half form);
    ``q_scale`` multiplies q before that.  ``sinks``: the cache is a window.
    ``workspace`` (uint8, aq_kv4_attention_workspace bytes) and ``out``: given, or
    allocated."""
    B, Hkv, D, slots = _kv4_sizes(cache, slots)
    dev = cache[0].device
    q, k_new, v_new, H, pos_stride, cos, sin, rows = _step_arguments("kv4_attention", q, k_new, v_new, pos, rope, B,
                                                                     Hkv, D, dev)
    L = _lib.load()
    size = int(L.aq_kv4_attention_workspace(B, H, Hkv, D, slots))
    ws = _workspace("kv4_attention", size, workspace, dev)
    out = _result("kv4_attention", out, q, dev)
    with _on(q):
        _lib.check(L.aq_kv4_attention(q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), *[t.data_ptr() for t in cache],
                                      pos.data_ptr(), pos_stride, B, H, Hkv, D, slots, _sinks(sinks, slots),
                                      scale, q_scale, _lib.ptr(cos), _lib.ptr(sin), rows, ws.data_ptr(), ws.numel(),
                                      out.data_ptr(), _lib.stream_of(dev)), "aq_kv4_attention")
    return out


def window_decode_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
                            v_cache: torch.Tensor, pos: torch.Tensor, *, scale: float, sinks: Optional[int] = 0,
                            q_scale: float = 1.0, rope=None, workspace: Optional[torch.Tensor] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """kv4_attention over an fp16 cache k_cache, v_cache [B, Hkv, slots, D]; H is
    1, 2, 4 or 8 times Hkv."""
    what = "window_decode_attention"
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[3] in (64, 128),
          f"{what}: caches {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    dev = k_cache.device
    _need(dev.type == "cuda", f"{what}: the cache must be on a HIP device")
    for t in (k_cache, v_cache):
        _need(t.dtype == torch.float16 and t.is_contiguous() and t.device == dev,
              f"{what}: the caches must be contiguous fp16 on {dev}")
    B, Hkv, slots, D = k_cache.shape
    q, k_new, v_new, H, pos_stride, cos, sin, rows = _step_arguments(what, q, k_new, v_new, pos, rope, B, Hkv, D, dev)
    L = _lib.load()
    ws = _workspace(what, int(L.aq_decode_attention_workspace(B, H, Hkv, D, slots)), workspace, dev)
    out = _result(what, out, q, dev)
    with _on(q):
        _lib.check(L.aq_window_decode_attention(q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_cache.data_ptr(),
                                                v_cache.data_ptr(), pos.data_ptr(), pos_stride, B, H, Hkv, D, slots,
                                                _sinks(sinks, slots), scale, q_scale, _lib.ptr(cos), _lib.ptr(sin),
                                                rows, ws.data_ptr(), ws.numel(), out.data_ptr(), _lib.stream_of(dev)),
                   "aq_window_decode_attention")
    return out


class DecodeCache:
    """One layer's static key/value cache of ``slots`` positions on a HIP
    device, in fp16 (``bits=16``) or 4 bits (``bits=4``), of every position
    (``sinks=None``) or of the first ``sinks`` and the last ``slots - sinks``."""

    def __init__(self, batch: int, kv_heads: int, slots: int, head_dim: int, *, bits: int = 16,
                 sinks: Optional[int] = None, device="cuda"):
        _need(bits in (4, 16), f"DecodeCache: {bits} bits (4 and 16 supported)")
        _need(head_dim in (64, 128), f"DecodeCache: head size {head_dim} (64 and 128 supported)")
        _sinks(sinks, slots)
        self.batch, self.kv_heads, self.slots, self.head_dim = batch, kv_heads, slots, head_dim
        self.bits, self.sinks = bits, sinks
        if bits == 4:
            self.buffers = kv4_buffers(batch, kv_heads, slots, head_dim, device)
        else:
            self.buffers = tuple(torch.zeros(batch, kv_heads, slots, head_dim, dtype=torch.float16, device=device)
                                 for _ in range(2))

    def workspace_bytes(self, heads: int) -> int:
        """Bytes of workspace that ``attend`` needs for this many query heads
        (layers whose calls follow each other can share one)."""
        L = _lib.load()
        f = L.aq_kv4_attention_workspace if self.bits == 4 else L.aq_decode_attention_workspace
        return int(f(self.batch, heads, self.kv_heads, self.head_dim, self.slots))

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.buffers)

    def store(self, k: torch.Tensor, v: torch.Tensor, start: int = 0, lengths: Optional[torch.Tensor] = None) -> None:
        """Write positions start .. start + S - 1 (k, v fp16 [B, Hkv, S, D]), of
        sequence b the first ``lengths[b]`` of them."""
        if self.bits == 4:
            kv4_store(k, v, self.buffers, start, lengths, self.slots, self.sinks)
            return
        S = k.shape[2]
        _need(start >= 0 and (self.sinks is not None or start + S <= self.slots),
              f"DecodeCache: positions {start} .. {start + S - 1} in {self.slots} slots")
        if S == 0:
            return
        # the newest position of each slot, by sequence when their lengths differ
        dev = self.buffers[0].device
        slot = torch.arange(self.slots, device=dev)[None]
        end = start + (torch.full((1, 1), S, device=dev) if lengths is None else lengths.clamp(0, S).view(-1, 1))
        p = slot
        if self.sinks is not None:
            w = self.slots - self.sinks
            p = torch.where(slot < self.sinks, slot, slot + torch.div((end - 1 - slot).clamp(min=0), w,
                                                                      rounding_mode="floor") * w)
        take = (p >= start) & (p < end)
        p = (p - start).clamp(0, S - 1)
        for buf, t in zip(self.buffers, (k, v)):
            new = t.gather(2, p[:, None, :, None].expand(t.shape[0], t.shape[1], self.slots, t.shape[3]))
            buf.copy_(torch.where(take[:, None, :, None], new, buf))

    def load(self, count: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The first ``count`` slots in fp16 (copies)."""
        if self.bits == 4:
            return kv4_load(self.buffers, count, self.slots)
        n = self.slots if count is None else count
        return self.buffers[0][:, :, :n].clone(), self.buffers[1][:, :, :n].clone()

    def attend(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, pos: torch.Tensor, *, scale: float,
               q_scale: float = 1.0, rope=None, workspace: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Append the step's key and value at ``pos`` and attend (kv4_attention,
        window_decode_attention)."""
        if self.bits == 4:
            return kv4_attention(q, k_new, v_new, self.buffers, pos, scale=scale, slots=self.slots, sinks=self.sinks,
                                 q_scale=q_scale, rope=rope, workspace=workspace, out=out)
        return window_decode_attention(q, k_new, v_new, *self.buffers, pos, scale=scale, sinks=self.sinks,
                                       q_scale=q_scale, rope=rope, workspace=workspace, out=out)
