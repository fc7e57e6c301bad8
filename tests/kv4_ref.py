"""Plain forms of the 4-bit cache for the tests: the documented format, written
out from indices (include/atlasinfer_amd.h, aq_kv4_store)."""
import torch


def quantize(x):
    """(codes uint8 [..., D], scales, minima fp16 [..., D / 32]) of fp16 x."""
    g = x.float().reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / 15.0).half()
    s = torch.where(lo + 15.0 * s.float() >= 65520.0, (s.view(torch.int16) - 1).view(torch.float16), s)
    sf = s.float()[..., None]
    c = torch.where(sf > 0, ((g - lo[..., None]) / sf).round().clamp(0, 15), torch.zeros(()))
    bad = ~torch.isfinite(g).all(-1)
    nan = torch.tensor(float("nan")).half()
    c = torch.where(bad[..., None], torch.zeros(()), c)
    return c.to(torch.uint8).reshape(x.shape), torch.where(bad, nan, s), torch.where(bad, nan, lo.half())


def _indices(slots, D):
    """Byte and shift of (slot, element) in a head's value codes; offsets of
    (slot, group)'s scale in its value parameters."""
    s, e = torch.arange(slots)[:, None], torch.arange(D)[None]
    blk, t, r, i = s // 32, s % 32 // 16, s % 16 // 4, s % 4
    word = ((e // 64 * 4 + r) * 16 + e % 16) * 4 + e % 64 // 16
    n = 4 * t + i
    g = torch.arange(D // 32)[None]
    par = blk * (D // 32 * 64) + ((g * 4 + r) * 4 + i) * 4 + t
    return blk * 16 * D + word * 4 + n // 2, n % 2 * 4, par


def unpack(cache, slots):
    """((codes, scales, minima) of the keys, of the values), on the CPU."""
    kc, kp, vc, vp = [t.cpu() for t in cache]
    B, H, _, half = kc.shape
    D = 2 * half
    k = torch.stack([kc & 15, kc >> 4], -1).reshape(B, H, -1, D)[:, :, :slots]
    byte, shift, par = _indices(slots, D)
    v = (vc.reshape(B, H, -1)[:, :, byte].int() >> shift & 15).to(torch.uint8)
    flat = vp.reshape(B, H, -1)
    return ((k, kp[:, :, :slots, :, 0], kp[:, :, :slots, :, 1]), (v, flat[:, :, par], flat[:, :, par + 2]))


def values(codes, s, m):
    """What codes stand for, in 64 bits."""
    g = codes.double().reshape(*codes.shape[:-1], -1, 32)
    return (g * s.double()[..., None] + m.double()[..., None]).reshape(codes.shape)


def slot_of(p, slots, sinks):
    return p if p < slots else sinks + (p - sinks) % (slots - sinks)


def rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


def rope_tables(n, D, dev):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)[None]
    a = torch.cat([a, a], 1)
    return a.cos().half().to(dev), a.sin().half().to(dev)
