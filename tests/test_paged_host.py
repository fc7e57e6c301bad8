"""The paged cache and token log probabilities without a GPU: what the C
functions and their Python callers refuse, the workspace rules, rotary
frequencies, and the 64-bit reference of the GPU tests against plain softmax."""
import ctypes
import math

import pytest
import torch

import paged_ref as R
from atlasinfer_amd.integration.decode_graph import GraphDecoder
from atlasinfer_amd.integration.logprobs import token_logprobs
from atlasinfer_amd.memory import paged_cache as PC
from test_decode_operators_host import ODD, P, Call


@pytest.fixture(scope="module")
def lib():
    from atlasinfer_amd import _lib
    return _lib.load()


def _store(lib):
    return Call(lib, "aq_paged_store", q=P, k=P, v=P, dtype=0, T=10, H=8, Hkv=2, D=64, q_row=512, q_head=64, k_row=128,
                k_head=64, v_row=128, v_head=64, starts=P, lengths=P, S=3, table=P, W=4, max_new=5, max_length=64, freq=P,
                rotary=64, interleaved=0, factor=1.0, q_out=P, kc=P, vc=P, pages=9, page_size=16, stream=None)


def _attend(lib):
    return Call(lib, "aq_paged_attention", q=P, dtype=1, T=10, H=8, Hkv=2, D=128, q_row=1024, q_head=128, kc=P, vc=P,
                pages=9, page_size=16, starts=P, lengths=P, S=3, table=P, W=400, max_new=5, max_length=6400, window=100,
                sinks=0, scale=0.1, ws=P, ws_bytes=1 << 30, out=P, stream=None)


def test_store_refusals(lib):
    c = _store(lib)
    for x in ("k", "v", "starts", "lengths", "table", "kc", "vc"):
        c.bad("null pointer", **{x: None})
    for kw in (dict(q=None), dict(H=0), dict(q_out=None)):
        c.bad("come with H", **kw)
    for d in (-1, 2):
        c.bad("dtype", dtype=d)
    for d in (0, 32, 96, 256):
        c.bad("head dim", D=d)
    for kw in (dict(T=0), dict(T=1 << 24), dict(S=0), dict(S=65536), dict(H=1025), dict(H=-1), dict(Hkv=0), dict(Hkv=1025)):
        c.bad("sizes out of range", **kw)
    for p in (0, 8, 24, 2048, -16):
        c.bad("page size", page_size=p)
    for kw in (dict(pages=0), dict(pages=1 << 31), dict(W=0), dict(W=1 << 28)):
        c.bad("pages", **kw)
    for kw in (dict(max_new=0), dict(max_length=0), dict(max_length=65)):
        c.bad("at most", **kw)
    for kw in (dict(rotary=-16), dict(rotary=8), dict(rotary=80), dict(rotary=0), dict(freq=None)):
        c.bad("rotary elements", **kw)
    for x in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head"):
        c.bad("multiples of 8", **{x: 132})
    for x in ("q", "k", "v", "q_out", "kc", "vc"):
        c.bad("16-byte aligned", **{x: ODD})
    for x in ("starts", "lengths", "table", "freq"):
        c.bad("aligned", **{x: ctypes.c_void_p(4098)})


def test_attention_refusals(lib):
    c = _attend(lib)
    for x in ("q", "kc", "vc", "starts", "lengths", "table", "out"):
        c.bad("null pointer", **{x: None})
    c.bad("dtype", dtype=2)
    c.bad("head dim", D=80)
    for kw in (dict(H=7), dict(H=0), dict(Hkv=0), dict(H=1026)):
        c.bad("multiple of Hkv", **kw)
    for kw in (dict(T=0), dict(T=1 << 24), dict(S=0), dict(S=65536), dict(max_new=0), dict(max_length=0)):
        c.bad("sizes out of range", **kw)
    c.bad("page size", page_size=48)
    for kw in (dict(pages=0), dict(W=0), dict(max_length=6401)):
        c.bad("pages", **kw)
    for kw in (dict(window=0), dict(sinks=-1)):
        c.bad("window", **kw)
    for x in ("q_row", "q_head"):
        c.bad("multiples of 8", **{x: 1028})
    for x in ("q", "kc", "vc", "out"):
        c.bad("16-byte aligned", **{x: ODD})
    for x in ("starts", "lengths", "table"):
        c.bad("aligned", **{x: ctypes.c_void_p(4098)})
    need = lib.aq_paged_attention_workspace(10, 3, 8, 2, 128, 5, 6400)
    assert need > 0
    c.bad("workspace", ws_bytes=need - 1)
    c.bad("workspace", ws=None)
    c.bad("workspace", ws=ODD)
    # more blocks than a grid takes
    c.bad("rows of", T=(1 << 24) - 1, H=1024, Hkv=512, S=1, max_new=1 << 24, q_row=1 << 17)


def test_attention_workspace_rule(lib):
    """A maximum and a denominator beside every span's sums of every row; none where
    one workgroup takes all keys."""
    size = lib.aq_paged_attention_workspace
    for bad in ((0, 1, 8, 2, 64, 1, 9), (1, 0, 8, 2, 64, 1, 9), (1, 1, 7, 2, 64, 1, 9), (1, 1, 8, 2, 80, 1, 9),
                (1, 1, 8, 2, 64, 0, 9), (1, 1, 8, 2, 64, 1, 0), (1 << 24, 1, 8, 2, 64, 1, 9), (1, 65536, 8, 2, 64, 1, 9),
                (1, 1, 8, 2, 64, 1, 1 << 31)):
        assert size(*bad) == -1, bad
    assert size(1, 1, 32, 8, 128, 1, 300) == 0  # short
    assert size(600, 600, 8, 1, 128, 1, 100000) == 0  # many
    for T, S, H, Hkv, D, new, length in ((1, 1, 32, 8, 128, 1, 701), (8, 8, 32, 8, 128, 1, 4001), (40, 8, 32, 32, 64, 5, 9000),
                                         (512, 1, 32, 8, 128, 512, 16384), (31 + 900, 32, 32, 8, 128, 900, 8000)):
        b = size(T, S, H, Hkv, D, new, length)
        spans = b // (T * H * (D + 2) * 4)
        assert b % (T * H * (D + 2) * 4) == 0 and 2 <= spans <= 64, (T, S, spans)


def test_logprobs_refusals(lib):
    c = Call(lib, "aq_token_logprobs", logits=P, dtype=0, B=2, V=100, stride=100, tokens=P, top=5, lp=P, ent=P, ranks=P, tlp=P,
             tt=P, ws=None, ws_bytes=0, stream=None)
    for x in ("logits", "tokens", "lp", "ent", "ranks", "tlp", "tt"):
        c.bad("null pointer", **{x: None})
    for d in (-1, 3):
        c.bad("dtype", dtype=d)
    for v in (0, -5, (1 << 18) + 1):
        c.bad("logits a row", V=v, stride=max(v, 1))
    for b, s in ((0, 100), (-1, 100), (65536, 100), (2, 99)):
        c.bad("rows", B=b, stride=s)
    for t in (-1, 65):
        c.bad("alternatives", top=t)
    c.bad("alternatives", V=4, stride=4)
    for name, at in (("logits", 4097), ("lp", 4098), ("ent", 4098), ("tlp", 4098), ("tokens", 4100), ("ranks", 4100), ("tt", 4100)):
        c.bad("misaligned", **{name: ctypes.c_void_p(at)})
    c.bad("misaligned", dtype=2, logits=ctypes.c_void_p(4098))
    c.bad("workspace", ws=ODD)
    size = lib.aq_token_logprobs_workspace
    for bad in ((0, 100, 0, 0), (65536, 100, 0, 0), (1, 0, 0, 0), (1, (1 << 18) + 1, 0, 0), (1, 100, 3, 0), (1, 100, 0, 65),
                (1, 4, 0, 5)):
        assert size(*bad) == -1, bad
    assert size(1, 1000, 0, 5) == 0 and size(600, 16384, 0, 5) == 0
    # parts of up to 2048 pieces of 16 bytes; more for few rows
    for B, V, dtype, parts in ((600, 16384 + 8, 0, 2), (600, 128256, 1, 8), (600, 1 << 18, 2, 32), (1, 50272, 0, 12), (64, 128256, 0, 8)):
        assert size(B, V, dtype, 7) == B * parts * (16 + 8 * 7), (B, V, dtype)


def test_python_refusals_on_the_cpu():
    i32 = dict(dtype=torch.int32)
    starts, lengths, table = torch.tensor([0, 1], **i32), torch.tensor([4], **i32), torch.zeros(1, 2, **i32)
    with pytest.raises(ValueError, match="HIP device"):
        PC.PagedBatch(starts, lengths, table, 1, 4)
    for bad in ((starts[:1], lengths, table), (starts, lengths.repeat(2), table), (starts, lengths, table[0]),
                (starts, lengths, table[:, :0]), (starts[:1], lengths[:0], table[:0])):
        with pytest.raises(ValueError, match="PagedBatch"):
            PC.PagedBatch(*bad, 1, 4)
    for kw in (dict(head_dim=96), dict(page_size=24), dict(page_size=8), dict(page_size=2048), dict(pages=0), dict(kv_heads=0),
               dict(dtype=torch.float32)):
        with pytest.raises(ValueError, match="paged cache"):
            PC.paged_buffers(**{**dict(pages=2, kv_heads=1, page_size=16, head_dim=64, device="cpu"), **kw})
    with pytest.raises(ValueError, match="HIP device"):
        token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))


def test_rotary_frequencies_are_those_of_hf():
    """Against transformers' own tables of each scaling type, from which they may be one rounding to fp32 off each."""
    transformers = pytest.importorskip("transformers")
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    for scaling in (None, dict(rope_type="linear", factor=4.0),
                    dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192),
                    dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096),
                    dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=2048, beta_fast=24.0, beta_slow=2.0,
                         attention_factor=1.5)):
        for theta in (10000.0, 500000.0):
            given = dict(scaling) if scaling else {"rope_type": "default"}
            cfg = transformers.LlamaConfig(hidden_size=512, num_attention_heads=4, num_key_value_heads=4, max_position_embeddings=32768)
            cfg.rope_theta = theta
            cfg.rope_scaling = scaling and dict(scaling)
            if hasattr(cfg, "rope_parameters"):
                cfg.rope_parameters = {**given, "rope_theta": theta}
            got, factor = PC.rotary_frequencies(128, theta, scaling)
            kind = given["rope_type"]
            if kind == "default":
                want, m = 1.0 / theta ** (torch.arange(0, 128, 2).double() / 128), 1.0
            else:
                want, m = ROPE_INIT_FUNCTIONS[kind](cfg, torch.device("cpu"))
            assert got.dtype == torch.float32 and torch.allclose(got.double(), want.double(), rtol=2e-6, atol=0), (kind, theta)
            assert abs(factor - m) <= 1e-6
    with pytest.raises(NotImplementedError):
        PC.rotary_frequencies(64, scaling=dict(rope_type="dynamic", factor=2.0))
    for n in (0, -2, 7):
        with pytest.raises(ValueError):
            PC.rotary_frequencies(n)


def test_the_reference_turns_and_attends():
    """The GPU tests' reference on one sequence whose pages are scattered, against rotations by complex numbers and torch's softmax."""
    b = R.Batch([5], [37], 2, 64, 16, torch.float16, "cpu")
    f, factor = PC.rotary_frequencies(32)
    x = torch.randn(5, 3, 64)
    for interleaved in (False, True):
        got, _ = R.turn(x, b.positions(0), f, interleaved, 1.5)
        for i, p in enumerate(b.positions(0).tolist()):
            for n in range(16):
                u, w = (2 * n, 2 * n + 1) if interleaved else (n, n + 16)
                a = p * float(f[n])
                for h in range(3):
                    y, z = float(x[i, h, u]), float(x[i, h, w])
                    assert abs(float(got[i, h, u]) - 1.5 * (y * math.cos(a) - z * math.sin(a))) < 1e-9
                    assert abs(float(got[i, h, w]) - 1.5 * (z * math.cos(a) + y * math.sin(a))) < 1e-9
        assert torch.equal(got[..., 32:], x[..., 32:].double())
    q = torch.randn(5, 4, 64).half()
    want, bound = R.attend(q, b, 0, 0.125, window=20, sinks=3)
    for i, p in enumerate(b.positions(0).tolist()):
        for h in range(4):
            seen = [j for j in range(p + 1) if p - j < 20 or j < 3]
            k = torch.stack([b.cache[0][b.table[0, j // 16], h // 2, j % 16] for j in seen]).double()
            v = torch.stack([b.cache[1][b.table[0, j // 16], h // 2, j % 16] for j in seen]).double()
            out = torch.softmax(k @ q[i, h].double() * 0.125, 0) @ v
            assert (want[i, h] - out).abs().max() < 1e-12
    assert (bound > 0).all() and (bound < 0.05).all()


def test_table_widths_past_64_bits(lib):
    """A width whose positions do not fit 64 bits is refused as any other that is too large."""
    for c in (_store(lib), _attend(lib)):
        c.bad("pages", W=1 << 60)
        c.bad("pages", W=(1 << 60) + 1)


class Pool:
    """What ``GraphDecoder._reserve`` needs of a decoder, on the CPU."""

    def __init__(self, B, pages, L, P=16):
        self.B, self.pages, self.L, self.page_size = B, pages, L, P
        self.table = torch.zeros(B, -(-L // P), dtype=torch.int32)
        GraphDecoder._release(self)

    def _device(self, values, dtype):
        return torch.tensor(values, dtype=dtype)

    def check(self, lengths):
        """Every sequence holds the pages of its positions, none twice, and the table says so."""
        for h, row, n in zip(self._held, self.table.tolist(), lengths):
            assert len(h) >= -(-n // self.page_size) and row == h + [0] * (len(row) - len(h))
        assert sorted(sum(self._held, []) + self._free) == list(range(self.pages))


@pytest.mark.parametrize("counts,steps,pages", [([16, 8], 16, 4), ([60, 3, 20], 44, 14), ([1, 1, 1, 1], 47, 12), ([33, 40], 8, 6)])
def test_pages_held_ahead_go_back(counts, steps, pages):
    """A pool of just the pages that the sequences end with serves them to the end; a position more is refused,
    and what they hold stays."""
    assert sum(-(-(n + steps) // 16) for n in counts) == pages
    p = Pool(len(counts), pages, 128)
    GraphDecoder._reserve(p, counts)
    kept = [[] for _ in counts]
    for step in range(steps + 1):
        lengths = [n + step for n in counts]
        GraphDecoder._reserve(p, lengths, ahead=64)
        p.check(lengths)
        for k, h, n in zip(kept, p._held, lengths):  # written pages stay where they are
            assert h[:len(k)] == k
            k[:] = h[:-(-n // 16)]
    before = [list(h) for h in p._held]
    with pytest.raises(RuntimeError, match="pages"):
        GraphDecoder._reserve(p, [16 * pages + 1] + lengths[1:], ahead=64)
    assert p._held == before
    p.check(lengths)


@pytest.mark.parametrize("factor", [1.0, 4.0, 40.0])
@pytest.mark.parametrize("given", [dict(mscale=1.0, mscale_all_dim=1.0), dict(mscale=0.707, mscale_all_dim=0.707),
                                   dict(mscale=1.0, mscale_all_dim=0.707), dict(mscale=0.707, mscale_all_dim=1.0),
                                   dict(mscale=2.0), dict(mscale_all_dim=2.0), dict(mscale=0.0, mscale_all_dim=1.0),
                                   dict(mscale=1.0, mscale_all_dim=0.0), dict(mscale=1.0, mscale_all_dim=0.5, attention_factor=1.7)])
def test_yarn_with_scales_of_its_factor(factor, given):
    """The factor of yarn's turned elements where a configuration scales it, against transformers' own."""
    transformers = pytest.importorskip("transformers")
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    scaling = dict(rope_type="yarn", factor=factor, original_max_position_embeddings=4096, **given)
    cfg = transformers.LlamaConfig(hidden_size=512, num_attention_heads=4, num_key_value_heads=4,
                                   max_position_embeddings=int(4096 * factor))
    cfg.rope_theta = 10000.0
    cfg.rope_scaling = dict(scaling)
    if hasattr(cfg, "rope_parameters"):
        cfg.rope_parameters = {**scaling, "rope_theta": 10000.0}
    want, m = ROPE_INIT_FUNCTIONS["yarn"](cfg, torch.device("cpu"))
    got, factor = PC.rotary_frequencies(128, 10000.0, scaling)
    assert abs(factor - m) <= 1e-6 and torch.allclose(got.double(), want.double(), rtol=2e-6, atol=0)


def test_scalings_without_what_they_need():
    """A scaling that lacks a number, or has None for it, is refused by its name."""
    whole = dict(linear=dict(factor=2.0), yarn=dict(factor=4.0, original_max_position_embeddings=4096),
                 llama3=dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192))
    for kind, numbers in whole.items():
        PC.rotary_frequencies(64, scaling=dict(rope_type=kind, **numbers))
        for key in numbers:
            for rest in ({k: x for k, x in numbers.items() if k != key}, {**numbers, key: None}):
                with pytest.raises(ValueError, match=f"{kind}.* without {key}"):
                    PC.rotary_frequencies(64, scaling=dict(rope_type=kind, **rest))


@pytest.mark.parametrize("page_size", [0, -16])
def test_pages_of_no_positions(page_size):
    p = Pool(2, 4, 64)
    p.dev = torch.device("cpu")
    with pytest.raises(ValueError, match=f"pages of {page_size} positions"):
        GraphDecoder._page_state(p, page_size, None, 2048)
