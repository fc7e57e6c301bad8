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
result and its cache stay as they were (without ``out`` that row is undefined).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from .. import _lib

GROUP = 32  # elements that share a scale and a minimum
BLOCK = 32  # slots whose values are interleaved


def _refuse(what: str):
    raise ValueError(what)


def kv4_buffers(batch: int, kv_heads: int, slots: int, head_dim: int, device) -> Tuple[torch.Tensor, ...]:
    """Empty buffers of a 4-bit cache: key codes, key parameters, value codes,
    value parameters (layouts at aq_kv4_store in include/atlasinfer_amd.h)."""
    if head_dim not in (64, 128):
        _refuse(f"kv4: head size {head_dim} (64 and 128 supported)")
    if batch <= 0 or kv_heads <= 0 or not 0 < slots <= 1 << 24:
        _refuse("kv4: batch, heads and slots must be positive, slots at most 2^24")
    c = (slots + BLOCK - 1) // BLOCK * BLOCK
    return (torch.zeros(batch, kv_heads, c, head_dim // 2, dtype=torch.uint8, device=device),
            torch.zeros(batch, kv_heads, c, head_dim // GROUP, 2, dtype=torch.float16, device=device),
            torch.zeros(batch, kv_heads, c // BLOCK, head_dim * 16, dtype=torch.uint8, device=device),
            torch.zeros(batch, kv_heads, c // BLOCK, head_dim // GROUP, 4, 4, 4, dtype=torch.float16, device=device))


# The checks below run on every step of a decoding loop: no message is put
# together unless it is raised, and shapes are compared as they are.


def _kv4_sizes(cache, slots: Optional[int]):
    """(B, Hkv, D, slots, device) of a 4-bit cache's buffers, which are checked."""
    if len(cache) != 4:
        _refuse("kv4: a cache is four buffers (kv4_buffers)")
    kc, kp, vc, vp = cache
    dev = kc.device
    if kc.dim() != 4 or dev.type != "cuda":
        _refuse(f"kv4: key codes {tuple(kc.shape)} on {dev}")
    B, Hkv, c, half = kc.shape
    if half not in (32, 64) or c % BLOCK or 0 in (B, Hkv, c):
        _refuse(f"kv4: key codes {tuple(kc.shape)}")
    n, g = c // BLOCK, half // 16
    if not (kp.shape == (B, Hkv, c, g, 2) and vc.shape == (B, Hkv, n, 32 * half) and vp.shape == (B, Hkv, n, g, 4, 4, 4)
            and kc.dtype == vc.dtype == torch.uint8 and kp.dtype == vp.dtype == torch.float16
            and kc.is_contiguous() and kp.is_contiguous() and vc.is_contiguous() and vp.is_contiguous()
            and kp.device == dev and vc.device == dev and vp.device == dev):
        _refuse(f"kv4: buffers {[(tuple(t.shape), t.dtype, t.device) for t in cache]} are not those of kv4_buffers, "
                "contiguous and on one device")
    if slots is None:
        slots = c
    elif not c - BLOCK < slots <= c:
        _refuse(f"kv4: {slots} slots in buffers of {c}")
    return B, Hkv, 2 * half, slots, dev


def _sinks(sinks: Optional[int], slots: int) -> int:
    if sinks is None:
        return -1
    if not 0 <= sinks < slots:
        _refuse(f"{sinks} sinks in {slots} slots")
    return sinks


def _strides(t: torch.Tensor):
    return _lib.ptr_array(t.stride()[:3], ctypes.c_int64)


def _prompt_arguments(what, k, v, lengths, start, B, Hkv, D, slots, sinks, dev):
    """Checks of a prompt's tensors and place; its length."""
    S = k.shape[2] if k.dim() == 4 else -1
    if k.shape != (B, Hkv, S, D) or v.shape != k.shape:
        _refuse(f"{what}: k {tuple(k.shape)}, v {tuple(v.shape)} for a cache of [{B}, {Hkv}, *, {D}]")
    if not (k.dtype == v.dtype == torch.float16 and k.device == dev and v.device == dev):
        _refuse(f"{what}: k and v must be fp16 on {dev}")
    if lengths is not None and not (lengths.dtype == torch.int64 and lengths.shape == (B,) and lengths.is_contiguous()
                                    and lengths.device == dev):
        _refuse(f"{what}: lengths must be contiguous int64 [{B}] on {dev}")
    if start < 0 or (sinks is None and start + S > slots):
        _refuse(f"{what}: positions {start} .. {start + S - 1} in {slots} slots")
    return S


def kv4_store(k: torch.Tensor, v: torch.Tensor, cache, start: int = 0, lengths: Optional[torch.Tensor] = None,
              slots: Optional[int] = None, sinks: Optional[int] = None) -> None:
    """Quantize positions start .. start + S - 1 (k, v fp16 [B, Hkv, S, D], any
    strides) into a 4-bit cache; of sequence b only the first ``lengths[b]``
    (int64 [B]).  ``sinks``: the cache is a window (None: it is not, and the
    positions must fit)."""
    B, Hkv, D, slots, dev = _kv4_sizes(cache, slots)
    S = _prompt_arguments("kv4_store", k, v, lengths, start, B, Hkv, D, slots, sinks, dev)
    sk = _sinks(sinks, slots)
    if S == 0:
        return
    k, v = _lib.strided_rows(k), _lib.strided_rows(v)
    with _lib.on_device(dev):
        _lib.check(_lib.load().aq_kv4_store(k.data_ptr(), v.data_ptr(), B, Hkv, S, D, _strides(k), _strides(v), start,
                                            _lib.ptr(lengths), *[t.data_ptr() for t in cache], slots, sk,
                                            _lib.stream_of(dev)), "aq_kv4_store")


def kv4_load(cache, count: Optional[int] = None, slots: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first ``count`` slots (all of them) of a 4-bit cache in fp16: keys
    and values [B, Hkv, count, D]."""
    B, Hkv, D, slots, dev = _kv4_sizes(cache, slots)
    if count is None:
        count = slots
    elif not 0 <= count <= slots:
        _refuse(f"kv4_load: {count} of {slots} slots")
    k = torch.empty(B, Hkv, count, D, dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    if count:
        with _lib.on_device(dev):
            _lib.check(_lib.load().aq_kv4_load(*[t.data_ptr() for t in cache], B, Hkv, D, slots, count, k.data_ptr(),
                                               v.data_ptr(), _lib.stream_of(dev)), "aq_kv4_load")
    return k, v


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _step_arguments(what, q, k_new, v_new, pos, rope, out, workspace, B, Hkv, D, dev):
    """Checks of a step's tensors; (q, k_new, v_new contiguous, H, pos_stride,
    addresses of the rotary tables, their rows, out)."""
    H = q.shape[1] if q.dim() == 3 else 0
    if H == 0 or q.shape != (B, H, D) or H % Hkv:
        _refuse(f"{what}: q {tuple(q.shape)} for a cache of [{B}, {Hkv}, *, {D}]")
    if k_new.shape != (B, Hkv, D) or v_new.shape != (B, Hkv, D):
        _refuse(f"{what}: k_new {tuple(k_new.shape)}, v_new {tuple(v_new.shape)}, expected {(B, Hkv, D)}")
    if not (q.dtype == k_new.dtype == v_new.dtype == torch.float16 and q.device == dev and k_new.device == dev
            and v_new.device == dev):
        _refuse(f"{what}: q, k_new and v_new must be fp16 on {dev}")
    n = pos.numel()
    if not (pos.dtype == torch.int64 and pos.dim() == 1 and (n == B or n == 1) and pos.is_contiguous()
            and pos.device == dev):
        _refuse(f"{what}: pos must be int64 [1] or [{B}] on {dev}")
    cos = sin = None
    rows = 0
    if rope is not None:
        cos, sin = rope
        rows = cos.shape[0]
        if not (cos.shape == (rows, D) and sin.shape == (rows, D) and rows and cos.dtype == sin.dtype == torch.float16
                and cos.is_contiguous() and sin.is_contiguous() and cos.device == dev and sin.device == dev):
            _refuse(f"{what}: rotary tables must be contiguous fp16 [positions, {D}] on {dev}")
        cos, sin = cos.data_ptr(), sin.data_ptr()
    if workspace is not None and not (workspace.dtype == torch.uint8 and workspace.is_contiguous()
                                      and workspace.device == dev):
        _refuse(f"{what}: the workspace must be contiguous uint8 on {dev}")
    if out is not None and not (out.shape == q.shape and out.dtype == torch.float16 and out.is_contiguous()
                                and out.device == dev and out.data_ptr() % 16 == 0):
        _refuse(f"{what}: out must be contiguous fp16 {tuple(q.shape)} on {dev}")
    if out is None:
        out = torch.empty((B, H, D), dtype=torch.float16, device=dev)
    return _aligned(q), _aligned(k_new), _aligned(v_new), H, int(n > 1), cos, sin, rows, out


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
    B, Hkv, D, slots, dev = _kv4_sizes(cache, slots)
    q, k_new, v_new, H, pos_stride, cos, sin, rows, out = _step_arguments("kv4_attention", q, k_new, v_new, pos, rope,
                                                                          out, workspace, B, Hkv, D, dev)
    sk = _sinks(sinks, slots)
    L = _lib.load()
    if workspace is None:
        size = L.aq_kv4_attention_workspace(B, H, Hkv, D, slots)
        workspace = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
    kc, kp, vc, vp = cache
    with _lib.on_device(dev):
        _lib.check(L.aq_kv4_attention(q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), kc.data_ptr(), kp.data_ptr(),
                                      vc.data_ptr(), vp.data_ptr(), pos.data_ptr(), pos_stride, B, H, Hkv, D, slots, sk,
                                      scale, q_scale, cos, sin, rows, *_space(workspace), out.data_ptr(),
                                      _lib.stream_of(dev)), "aq_kv4_attention")
    return out


def _space(workspace):
    return (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())


def window_decode_attention(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor,
                            v_cache: torch.Tensor, pos: torch.Tensor, *, scale: float, sinks: Optional[int] = 0,
                            q_scale: float = 1.0, rope=None, workspace: Optional[torch.Tensor] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """kv4_attention over an fp16 cache k_cache, v_cache [B, Hkv, slots, D]; H is
    1, 2, 4 or 8 times Hkv."""
    what = "window_decode_attention"
    dev = k_cache.device
    if not (k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.dtype == v_cache.dtype == torch.float16
            and k_cache.is_contiguous() and v_cache.is_contiguous() and dev.type == "cuda" and v_cache.device == dev):
        _refuse(f"{what}: caches {tuple(k_cache.shape)}, {tuple(v_cache.shape)} must be contiguous fp16 of one shape on "
                "one HIP device")
    B, Hkv, slots, D = k_cache.shape
    if D not in (64, 128) or 0 in (B, Hkv, slots):
        _refuse(f"{what}: caches {tuple(k_cache.shape)} (head sizes 64 and 128 supported)")
    q, k_new, v_new, H, pos_stride, cos, sin, rows, out = _step_arguments(what, q, k_new, v_new, pos, rope, out,
                                                                          workspace, B, Hkv, D, dev)
    sk = _sinks(sinks, slots)
    L = _lib.load()
    if workspace is None:
        workspace = torch.empty(max(16, L.aq_decode_attention_workspace(B, H, Hkv, D, slots)), dtype=torch.uint8,
                                device=dev)
    with _lib.on_device(dev):
        _lib.check(L.aq_window_decode_attention(q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_cache.data_ptr(),
                                                v_cache.data_ptr(), pos.data_ptr(), pos_stride, B, H, Hkv, D, slots, sk,
                                                scale, q_scale, cos, sin, rows, *_space(workspace), out.data_ptr(),
                                                _lib.stream_of(dev)), "aq_window_decode_attention")
    return out


class DecodeCache:
    """One layer's static key/value cache of ``slots`` positions on a HIP
    device, in fp16 (``bits=16``) or 4 bits (``bits=4``), of every position
    (``sinks=None``) or of the first ``sinks`` and the last ``slots - sinks``."""

    def __init__(self, batch: int, kv_heads: int, slots: int, head_dim: int, *, bits: int = 16,
                 sinks: Optional[int] = None, device="cuda"):
        if bits not in (4, 16) or head_dim not in (64, 128):
            _refuse(f"DecodeCache: {bits} bits (4 and 16 supported), head size {head_dim} (64 and 128 supported)")
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
        sequence b the first ``lengths[b]`` of them.  In 16 bits by torch operations
        over all slots, with temporaries of the cache's size."""
        if self.bits == 4:
            kv4_store(k, v, self.buffers, start, lengths, self.slots, self.sinks)
            return
        dev = self.buffers[0].device
        S = _prompt_arguments("DecodeCache.store", k, v, lengths, start, self.batch, self.kv_heads, self.head_dim,
                              self.slots, self.sinks, dev)
        if S == 0:
            return
        # the newest position of each slot, by sequence when their lengths differ
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
        if not 0 <= n <= self.slots:
            _refuse(f"DecodeCache.load: {n} of {self.slots} slots")
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
