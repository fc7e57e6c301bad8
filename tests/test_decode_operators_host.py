"""Sampling, the 4-bit cache and window attention without a GPU: what the C
functions and their Python callers refuse, the workspace rules, and the slots
that a window of an fp16 cache keeps."""
import ctypes
import itertools

import pytest
import torch

import kv4_ref as R
from atlasinfer_amd.integration.sampling import sample_tokens
from atlasinfer_amd.integration.window_attention import window_attention
from atlasinfer_amd.memory import decode_cache as DC

AQ_EINVAL = -1
P, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4096 + 8)


@pytest.fixture(scope="module")
def lib():
    from atlasinfer_amd import _lib
    return _lib.load()


def _strides(*s):
    return (ctypes.c_int64 * 3)(*s)


class Call:
    """A C function with its arguments by name; bad(...) changes some."""

    def __init__(self, lib, name, **kw):
        self.lib, self.name, self.kw = lib, name, kw

    def bad(self, message, **changed):
        assert set(changed) <= set(self.kw)
        assert getattr(self.lib, self.name)(*{**self.kw, **changed}.values()) == AQ_EINVAL, changed
        said = self.lib.aq_last_error().decode()
        assert self.name in said and message in said, said


def test_sample_refusals(lib):
    c = Call(lib, "aq_sample", logits=P, dtype=0, B=2, V=100, stride=100, u=P, t=None, k=None, p=None, m=None, t0=1.0, k0=0,
             p0=1.0, m0=0.0, tokens=P, ws=None, ws_bytes=0, stream=None)
    for name in ("logits", "u", "tokens"):
        c.bad("null pointer", **{name: None})
    for d in (-1, 3):
        c.bad("dtype", dtype=d)
    for v in (0, -5, (1 << 18) + 1):
        c.bad("logits a row", V=v, stride=max(v, 1))
    for b, s in ((0, 100), (-1, 100), (65536, 100), (2, 99)):
        c.bad("rows", B=b, stride=s)
    for name, at in (("logits", 4097), ("u", 4098), ("tokens", 4100), ("t", 4098), ("k", 4097), ("p", 4099), ("m", 4098)):
        c.bad("misaligned", **{name: ctypes.c_void_p(at)})
    c.bad("misaligned", dtype=2, logits=ctypes.c_void_p(4098))
    c.bad("workspace", ws=ODD)


def test_sample_workspace_rule(lib):
    size = lib.aq_sample_workspace
    for bad in ((0, 100, 0, 0), (-1, 100, 0, 0), (65536, 100, 0, 0), (1, 0, 0, 0), (1, (1 << 18) + 1, 0, 0), (1, 100, 3, 0),
                (1, 100, -1, 0)):
        assert size(*bad) == -1, bad
    one = size(1, 128256, 0, 0)
    assert one > 0 and one % 16 == 0
    # rows of 2048 pieces of 16 bytes, where there are too few rows for the GPU and no top-k
    for args, parts in (((64, 128256, 0, 0), True), ((128, 128256, 0, 0), True), ((129, 128256, 0, 0), False),
                        ((257, 128256, 0, 0), False), ((65535, 128256, 0, 0), False), ((1, 2048 * 8, 1, 0), True),
                        ((1, 2048 * 8 - 1, 1, 0), False), ((1, 2048 * 4, 2, 0), True), ((1, 128256, 0, 50), False),
                        ((1, 128256, 0, 128256), True), ((1, 128256, 0, -1), True)):
        assert size(*args) == (args[0] * one if parts else 0), args


def _step(lib, name):
    kw = dict(q=P, k_new=P, v_new=P)
    kw.update(dict(kc=P, kp=P, vc=P, vp=P) if name == "aq_kv4_attention" else dict(kc=P, vc=P))
    kw.update(pos=P, pos_stride=1, B=2, H=8, Hkv=2, D=128, slots=300, sinks=4, scale=0.1, q_scale=1.0, cos=P, sin=P,
              rows=1000, ws=P, ws_bytes=1 << 30, out=P, stream=None)
    return Call(lib, name, **kw)


@pytest.mark.parametrize("name", ["aq_kv4_attention", "aq_window_decode_attention"])
def test_step_refusals(lib, name):
    c = _step(lib, name)
    for x in [n for n in c.kw if c.kw[n] is P and n not in ("cos", "sin", "ws")]:
        c.bad("null pointer", **{x: None})
    c.bad("come together", cos=None)
    c.bad("come together", sin=None)
    c.bad("rows of rope_cos", rows=0)
    c.bad("head dim", D=96)
    c.bad("multiple of Hkv" if name == "aq_kv4_attention" else "times Hkv", H=7)
    for s in (2, -1):
        c.bad("pos_stride", pos_stride=s)
    for s in (-2, 300, 301):
        c.bad("sinks", sinks=s)
    for kw in (dict(B=65536), dict(slots=(1 << 24) + 1)):
        c.bad("sizes out of range", **kw)
    for x in ("k_new", "v_new", "kc", "vc"):
        c.bad("16-byte aligned", **{x: ODD})
    # more slots than one workgroup takes: the workspace is needed in full
    size = lib.aq_kv4_attention_workspace if name == "aq_kv4_attention" else lib.aq_decode_attention_workspace
    need = size(2, 8, 2, 128, 4000)
    assert need > 0
    c.bad("workspace", slots=4000, ws_bytes=need - 1)
    c.bad("workspace" if name == "aq_kv4_attention" else "null pointer", slots=4000, ws=None)
    if name == "aq_window_decode_attention":
        c.bad("1, 2, 4 or 8", H=6)
    else:
        for x in ("q", "out", "cos", "kp", "vp"):
            c.bad("16-byte aligned", **{x: ODD})


def test_kv4_workspace_rule(lib):
    size = lib.aq_kv4_attention_workspace
    for bad in ((0, 8, 2, 128, 10), (1, 0, 2, 128, 10), (1, 8, 0, 128, 10), (1, 7, 2, 128, 10), (1, 8, 2, 80, 10), (1, 8, 2, 64, 0)):
        assert size(*bad) == -1, bad
    assert size(1, 8, 2, 128, 512) == 0 and size(64, 64, 64, 64, 1) == 0   # up to 16 blocks: one workgroup a head
    # 17 blocks in 5 spans: a tile of 16 heads' sums, maxima and denominators each
    assert size(1, 8, 2, 128, 513) == 2 * 5 * (16 * 128 + 32) * 4
    assert size(1, 34, 1, 64, 513) == 3 * 5 * (16 * 64 + 32) * 4


def test_kv4_store_and_load_refusals(lib):
    c = Call(lib, "aq_kv4_store", k=P, v=P, B=2, Hkv=2, S=10, D=64, ks=_strides(1280, 640, 64), vs=_strides(1280, 640, 64),
             start=0, lengths=None, kc=P, kp=P, vc=P, vp=P, slots=100, sinks=-1, stream=None)
    for x in ("k", "v", "ks", "vs", "kc", "kp", "vc", "vp"):
        c.bad("null pointer", **{x: None})
    c.bad("head dim", D=32)
    for kw in (dict(B=0), dict(Hkv=0), dict(slots=0), dict(slots=(1 << 24) + 1)):
        c.bad("sizes out of range", **kw)
    for s in (-2, 100):
        c.bad("sinks", sinks=s)
    for kw in (dict(S=0), dict(start=-1), dict(S=1 << 31, sinks=0), dict(start=(1 << 31) - 5, sinks=0)):
        c.bad("out of range", **kw)
    for kw in (dict(S=101), dict(start=91)):
        c.bad("slots", **kw)
    for i in range(3):
        s = [1280, 640, 64]
        s[i] += 4
        c.bad("multiples of 8", ks=_strides(*s))
        c.bad("multiples of 8", vs=_strides(*s))
    for x in ("k", "v", "kc", "kp", "vc", "vp"):
        c.bad("16-byte aligned", **{x: ODD})
    c = Call(lib, "aq_kv4_load", kc=P, kp=P, vc=P, vp=P, B=2, Hkv=2, D=64, slots=100, count=100, k=P, v=P, stream=None)
    for x in ("kc", "kp", "vc", "vp", "k", "v"):
        c.bad("null pointer", **{x: None})
        c.bad("16-byte aligned", **{x: ODD})
    for n in (0, -1, 101):
        c.bad("slots", count=n)


def test_window_attention_refusals(lib):
    s = _strides(64 * 200, 64 * 100, 64)
    c = Call(lib, "aq_window_attention", q=P, k=P, v=P, B=1, H=4, Hkv=2, M=100, N=100, D=64, qs=s, ks=s, vs=s, window=10,
             sinks=0, scale=0.1, starts=None, out=P, stream=None)
    for x in ("q", "k", "v", "qs", "ks", "vs", "out"):
        c.bad("null pointer", **{x: None})
    c.bad("head dim", D=256)
    for kw in (dict(H=5), dict(Hkv=0), dict(H=0), dict(B=0), dict(B=65536)):
        c.bad("multiple of Hkv", **kw)
    for kw in (dict(M=0), dict(M=101), dict(N=1 << 24)):
        c.bad("positions", **kw)
    for kw in (dict(window=0), dict(window=-3), dict(sinks=-1)):
        c.bad("sinks", **kw)
    for x, i in itertools.product(("qs", "ks", "vs"), range(3)):
        t = [64 * 200, 64 * 100, 64]
        t[i] += 1
        c.bad("multiples of 8", **{x: _strides(*t)})
    for x, far in itertools.product(("ks", "vs"), (-64, (1 << 23) + 8)):
        c.bad("2^23", **{x: _strides(0, 0, far)})
    c.bad("blocks of queries", B=65535, H=512, Hkv=1, M=1, N=1)
    for x in ("q", "k", "v", "out"):
        c.bad("16-byte aligned", **{x: ODD})
    c.bad("16-byte aligned", starts=ctypes.c_void_p(4098))


def test_tensors_of_the_host_are_refused():
    """Every entry point wants a HIP device and says so."""
    x = torch.zeros(2, 100)
    with pytest.raises(ValueError, match="HIP device"):
        sample_tokens(x, torch.zeros(2))
    with pytest.raises(ValueError, match="HIP device"):
        sample_tokens(x.double(), torch.zeros(2))
    h = torch.zeros(1, 2, 8, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="HIP device"):
        window_attention(h, h, h, window=4)
    cache = DC.kv4_buffers(1, 2, 8, 64, "cpu")
    with pytest.raises(ValueError, match="kv4: key codes"):
        DC.kv4_store(h, h, cache)
    with pytest.raises(ValueError, match="kv4: key codes"):
        DC.kv4_load(cache)
    row, pos = h[:, :, 0], torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="kv4: key codes"):
        DC.kv4_attention(row, row, row, cache, pos, scale=1.0)
    with pytest.raises(ValueError, match="HIP device"):
        DC.window_decode_attention(row, row, row, h, h, pos, scale=1.0)


def test_window_attention_shapes_are_refused():
    h = torch.zeros(1, 4, 8, 64, dtype=torch.float16)
    for k, v in ((h[:, :3], h[:, :3]), (h[:, :, :4], h[:, :, :4]), (h, h[:, :2]), (h[0], h[0]), (h.expand(2, 4, 8, 64),) * 2,
                 (h[..., :32], h[..., :32])):
        with pytest.raises(ValueError, match="window_attention"):
            window_attention(h, k, v)


def test_cache_arguments():
    for kw in (dict(bits=8), dict(sinks=8), dict(sinks=-1)):
        with pytest.raises(ValueError):
            DC.DecodeCache(1, 2, 8, 64, device="cpu", **kw)
    for shape in ((1, 2, 8, 80), (0, 2, 8, 64), (1, 0, 8, 64), (1, 2, 0, 64), (1, 2, (1 << 24) + 1, 64)):
        with pytest.raises(ValueError):
            DC.kv4_buffers(*shape, "cpu")
    c = DC.DecodeCache(2, 2, 8, 64, device="cpu")
    good = torch.zeros(2, 2, 4, 64, dtype=torch.float16)
    for k, kw in ((good[:1], {}), (good[:, :1], {}), (good[..., :32], {}), (good.float(), {}), (good, dict(start=-1)),
                  (good, dict(start=5)), (good, dict(lengths=torch.zeros(1, dtype=torch.int64))),
                  (good, dict(lengths=torch.zeros(2, dtype=torch.int32)))):
        with pytest.raises(ValueError, match="DecodeCache.store"):
            c.store(k, k, **kw)
    for n in (-1, 9):
        with pytest.raises(ValueError, match="DecodeCache.load"):
            c.load(n)


@pytest.mark.parametrize("slots,sinks", [(8, 0), (8, 3), (8, 7), (40, None)])
def test_fp16_cache_keeps_the_newest_position_of_a_slot(slots, sinks):
    """Pieces of prompts, by sequence: each slot holds the newest position that
    belongs to it, as a loop over the positions writes them."""
    g = torch.Generator().manual_seed(slots)
    c = DC.DecodeCache(2, 1, slots, 64, sinks=sinks, device="cpu")
    want = [torch.zeros(2, 1, slots, 64, dtype=torch.float16) for _ in range(2)]
    for start, lengths in ((0, (5, 3)), (3, (0, 9)), (5, (31, 17)), (36, (2, 0))):
        S = max(lengths)
        kv = [torch.randn(2, 1, S, 64, generator=g).half() for _ in range(2)]
        c.store(*kv, start, torch.tensor(lengths))
        for b, n in enumerate(lengths):
            for i in range(n):
                for t, x in zip(want, kv):
                    t[b, :, R.slot_of(start + i, slots, sinks)] = x[b, :, i]
        for got, t in zip(c.load(), want):
            assert torch.equal(got, t)
