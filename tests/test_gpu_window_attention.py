"""Attention through a sliding window with sinks: prompts against 64 bits, and
the step over an fp16 cache that keeps the window."""
import pytest
import torch

import kv4_ref as R
from atlasinfer_amd.integration.window_attention import window_attention
from atlasinfer_amd.memory import decode_cache as DC

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _rnd(g, *s):
    return torch.randn(*s, generator=g, device=DEV).half()


def _reference(q, k, v, window, sinks, scale, starts):
    """Output [B, M, H, D] and error bound, in 64 bits."""
    B, H, M, D = q.shape
    N, G = k.shape[2], H // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    i = torch.arange(N - M, N, device=DEV)[:, None]
    j = torch.arange(N, device=DEV)[None]
    first = torch.zeros(B, 1, 1, device=DEV) if starts is None else starts.view(B, 1, 1)
    sees = (j <= i) & (j >= first) & ((i - j < window) | (j - first < sinks))
    sees = sees[:, None]
    k0, v0 = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
    s = (q @ k0.transpose(2, 3).contiguous() * scale).masked_fill(~sees, -float("inf"))
    w = torch.softmax(s, -1).nan_to_num(0.0)
    want = w @ v0
    # numerators rounded to fp16 (2^-11 each, 2^-25 of the largest below the
    # normal numbers); scores and sums in f32: products of D terms and the
    # exponential, 2^-17 of the scores' terms
    size = (q.abs() @ k0.abs().transpose(2, 3).contiguous() * scale).masked_fill(~sees, 0.0).amax(-1, keepdim=True)
    bound = (torch.expm1(2.0 ** -17 * size) + 2.0 ** -11 + 2.0 ** -16) * (w @ v0.abs())
    bound = bound + 2.0 ** -24 * (sees.double() @ v0.abs()) + 2.0 ** -11 * want.abs() + 2.0 ** -24
    return want.transpose(1, 2), bound.transpose(1, 2)


def _check(B, H, Hkv, M, N, D, window, sinks, starts=None, seed=0, poison=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, k, v = _rnd(g, B, M, H, D).transpose(1, 2), _rnd(g, B, N, Hkv, D).transpose(1, 2), _rnd(g, B, N, Hkv, D).transpose(1, 2)
    if poison is not None:
        poison(k, v)
    starts = None if starts is None else torch.tensor(starts, dtype=torch.int32, device=DEV)
    got = window_attention(q, k, v, window=window, sinks=sinks, starts=starts)
    want, bound = _reference(q, k, v, N if window is None else window, sinks, D ** -0.5, starts)
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max()
    return got


@pytest.mark.parametrize("D,H,Hkv", [(64, 2, 2), (128, 4, 1), (128, 6, 2)])
@pytest.mark.parametrize("N", [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 200, 513])
def test_lengths(D, H, Hkv, N):
    _check(2, H, Hkv, N, N, D, None, 0, seed=N)
    _check(1, H, Hkv, N, N, D, max(1, N // 3), min(4, N), seed=N + 1)


@pytest.mark.parametrize("M,N,window,sinks", [
    (1, 1, 1, 0), (1, 300, 20, 3), (5, 300, 64, 0), (130, 700, 1, 0), (130, 700, 1, 1), (300, 300, 64, 65),
    (300, 300, 65, 300), (257, 1000, 128, 4), (1000, 1000, 100, 64), (1000, 1000, 63, 1), (640, 640, 1000, 7),
])
def test_windows(M, N, window, sinks):
    _check(1, 4, 2, M, N, 64, window, sinks, seed=M)
    _check(1, 2, 1, M, N, 128, window, sinks, seed=M)


def test_scales():
    """A negative scale is that of the negated queries; with 0 every key seen counts alike."""
    g = torch.Generator(device=DEV).manual_seed(8)
    for D in (64, 128):
        q, k, v = _rnd(g, 2, 4, 150, D), _rnd(g, 2, 2, 150, D), _rnd(g, 2, 2, 150, D)
        starts = torch.tensor([0, 30], dtype=torch.int32, device=DEV)
        kw = dict(window=70, sinks=3, starts=starts)
        assert torch.equal(window_attention(q, k, v, scale=-0.2, **kw), window_attention(-q, k, v, scale=0.2, **kw))
        want, bound = _reference(q, k, v, 70, 3, 0.0, starts)
        assert ((window_attention(q, k, v, scale=0.0, **kw).double() - want).abs() <= bound).all()


def test_left_padding():
    """Sequences that begin late, rows of which see nothing, one of them empty."""
    got = _check(5, 4, 2, 200, 200, 64, 40, 4, starts=[0, 1, 70, 199, 200], seed=5)
    assert (got[2, :70] == 0).all() and (got[4] == 0).all()
    _check(3, 2, 2, 100, 300, 128, 1000, 0, starts=[0, 150, 250], seed=6)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_unseen_values_do_not_matter(D, bad):
    """NaN and infinities in keys and values that a query does not see: before
    the start, and future positions of queries in the same tile."""
    N = 200

    def poison(k, v):
        for t in (k, v):
            t[0, :, :30] = bad
            t[:, :, 150:, ::7] = bad
    g = torch.Generator(device=DEV).manual_seed(9)
    q, k, v = _rnd(g, 2, 2, N, D), _rnd(g, 2, 1, N, D), _rnd(g, 2, 1, N, D)
    poison(k, v)
    starts = torch.tensor([30, 0], dtype=torch.int32, device=DEV)
    for window in (300, 40):
        got = window_attention(q, k, v, window=window, sinks=2, starts=starts)[:, :150]
        want, bound = _reference(q, k, v, window, 2, D ** -0.5, starts)
        assert ((got.double() - want[:, :150]).abs() <= bound[:, :150]).all()
    # and through the window: what has left it
    k, v = _rnd(g, 1, 1, N, D), _rnd(g, 1, 1, N, D)
    k[:, :, :20], v[:, :, :20] = bad, bad
    got = window_attention(q[:1], k, v, window=30)
    want, bound = _reference(q[:1], k, v, 30, 0, D ** -0.5, None)
    assert ((got.double() - want).abs() <= bound)[:, 49:].all()


def test_prompt_in_pieces_and_streams():
    """A prompt in two pieces gives each piece's rows of the whole; on another
    stream; strided and misaligned inputs."""
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = _rnd(g, 1, 4, 300, 64), _rnd(g, 1, 2, 300, 64), _rnd(g, 1, 2, 300, 64)
    whole = window_attention(q, k, v, window=50, sinks=3)
    rest = window_attention(q[:, :, 170:], k, v, window=50, sinks=3)
    assert ((whole[:, 170:].float() - rest.float()).abs() <= 2e-2).all()  # other tiles, other roundings
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = window_attention(q, k, v, window=50, sinks=3)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(whole, other)
    odd = torch.empty(1 * 4 * 300 * 64 + 1, dtype=torch.float16, device=DEV)[1:].view(1, 4, 300, 64).copy_(q)
    wide = torch.zeros(1, 2, 300, 67, dtype=torch.float16, device=DEV)
    wide[..., :64] = k
    assert torch.equal(window_attention(odd, wide[..., :64], v, window=50, sinks=3), whole)


def test_refusals():
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)  # noqa: E731
    q, k = h(1, 4, 8, 64), h(1, 2, 8, 64)
    for args, kw in [((q, k, k), dict(window=0)), ((q, k, k), dict(sinks=-1)), ((q, k, h(1, 2, 9, 64)), {}),
                     ((h(1, 3, 8, 64), k, k), {}), ((q, h(1, 2, 7, 64), h(1, 2, 7, 64)), {}),
                     ((h(1, 4, 8, 96), h(1, 2, 8, 96), h(1, 2, 8, 96)), {}), ((q.float(), k, k), {}),
                     ((q, k, k), dict(starts=torch.zeros(1, device=DEV))), ((q.cpu(), k.cpu(), k.cpu()), {})]:
        with pytest.raises(ValueError):
            window_attention(*args, **kw)
    with pytest.raises(RuntimeError):
        window_attention(q.requires_grad_(), k, k)
    assert window_attention(h(1, 4, 0, 64), k, k).shape == (1, 0, 4, 64)


# ---------------------------------------------------------------- the step


def _step(B, H, Hkv, D, slots, sinks, positions, rope):
    g = torch.Generator(device=DEV).manual_seed(slots + B)
    kc, vc = (torch.full((B, Hkv, slots, D), float("nan"), dtype=torch.float16, device=DEV) for _ in range(2))
    for b, p in enumerate(positions):
        n = min(max(p, 0), slots)
        kc[b, :, :n], vc[b, :, :n] = _rnd(g, Hkv, n, D), _rnd(g, Hkv, n, D)
    q, kn, vn = _rnd(g, B, H, D), _rnd(g, B, Hkv, D), _rnd(g, B, Hkv, D)
    pos = torch.tensor(positions, device=DEV)
    tables = R.rope_tables(max(positions) + 1, D, DEV) if rope else None
    want_k, want_v = kc.clone(), vc.clone()
    out = torch.full((B, H, D), 77.0, dtype=torch.float16, device=DEV)
    DC.window_decode_attention(q, kn, vn, kc, vc, pos, scale=D ** -0.5, sinks=sinks, rope=tables, out=out)
    if rope:
        c, s = [t[pos.clamp(min=0)][:, None] for t in tables]
        q, kn = R.rotate(q, c, s), R.rotate(kn, c, s)
    for b, p in enumerate(positions):
        if p >= 0:
            want_k[b, :, R.slot_of(p, slots, sinks)], want_v[b, :, R.slot_of(p, slots, sinks)] = kn[b], vn[b]
    assert torch.equal(kc.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(vc.view(torch.int16), want_v.view(torch.int16))
    for b, p in enumerate(positions):
        if p < 0:
            assert (out[b] == 77.0).all()
            continue
        n = min(p + 1, slots)
        k, v = (t[b, :, :n].double().repeat_interleave(H // Hkv, 0) for t in (kc, vc))
        s = (k * q[b].double()[:, None]).sum(-1)
        w = torch.softmax(s * D ** -0.5, -1)
        want = (w[..., None] * v).sum(1)
        # scores, softmax and sums in f32 (2^-17 of the terms), one rounding to fp16
        size = (k.abs() * q[b].double().abs()[:, None]).sum(-1).amax(-1) * D ** -0.5
        bound = (torch.expm1(2.0 ** -17 * size) + 2.0 ** -17)[:, None] * (w[..., None] * v.abs()).sum(1)
        bound = bound + 2.0 ** -11 * want.abs() + 2.0 ** -24
        assert ((out[b].double() - want).abs() <= bound).all(), (b, p)


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("B,H,Hkv,D,slots,sinks,positions", [
    (1, 4, 4, 64, 40, 4, [39]), (1, 4, 4, 64, 40, 4, [40]), (2, 8, 2, 128, 100, 4, [99, 1000]),
    (3, 8, 1, 128, 37, 0, [37, -1, 74]), (2, 4, 2, 64, 5, 4, [5, 77]), (2, 2, 2, 64, 1, 0, [0, 9]),
    (2, 8, 2, 128, 1028, 4, [1027, 5000]), (16, 16, 8, 64, 300, 1, [29 * i for i in range(16)]),
    (2, 8, 2, 128, 4100, 4, [4099, 9000]), (130, 2, 1, 64, 300, 5, [7 * i for i in range(130)]),
    (2, 4, 2, 128, 200, None, [199, 3]),
])
def test_window_step(B, H, Hkv, D, slots, sinks, positions, rope):
    _step(B, H, Hkv, D, slots, sinks, positions, rope)


@pytest.mark.parametrize("bits", [4, 16])
def test_prompt_then_steps(bits):
    """A prompt stored into a window, then steps past its edge, as a decoder
    runs them: the slots hold the sinks and the last positions."""
    B, H, Hkv, D, slots, sinks, S = 2, 4, 2, 64, 24, 3, 50
    g = torch.Generator(device=DEV).manual_seed(8)
    c = DC.DecodeCache(B, Hkv, slots, D, bits=bits, sinks=sinks, device=DEV)
    k, v = _rnd(g, B, Hkv, S, D), _rnd(g, B, Hkv, S, D)
    lengths = torch.tensor([S, 17], device=DEV)
    c.store(k[:, :, :30], v[:, :, :30], lengths=lengths.clamp(max=30))
    c.store(k[:, :, 30:], v[:, :, 30:], start=30, lengths=(lengths - 30).clamp(min=0))
    hist = [[k[b, :, :n], v[b, :, :n]] for b, n in enumerate(lengths.tolist())]
    pos = lengths.clone()
    for step in range(10):
        q, kn, vn = _rnd(g, B, H, D), _rnd(g, B, Hkv, D), _rnd(g, B, Hkv, D)
        c.attend(q, kn, vn, pos, scale=0.125)
        for b in range(B):
            hist[b] = [torch.cat([x, y[b][:, None]], 1) for x, y in zip(hist[b], (kn, vn))]
        pos += 1
    got = c.load()
    for b in range(B):
        n = hist[b][0].shape[1]
        for p in range(n):
            if n <= slots or p < sinks or p >= n - (slots - sinks):
                for x, y in zip(got, hist[b]):
                    want = y[:, p]
                    if bits == 4:
                        want = R.values(*R.quantize(want.cpu())).half().to(DEV)
                    assert ((x[b, :, R.slot_of(p, slots, sinks)] - want).abs() <= 2e-3 * want.abs()).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [64, 100, 300])
def test_unseen_values_of_the_first_tile(D, N):
    """Infinities and NaN in the rows that each of the waves loads of the first tile, in
    many heads at once: queries before them do not see them."""
    g = torch.Generator(device=DEV).manual_seed(N)
    B, H = 8, 16
    q, k, v = _rnd(g, B, H, N, D), _rnd(g, B, H, N, D), _rnd(g, B, H, N, D)
    first = torch.tensor([3, 17, 31, 33, 47, 49, 62, 63], device=DEV)  # by sequence
    for b, at in enumerate(first.tolist()):
        v[b, :, at, b::5] = [float("nan"), float("inf"), -float("inf")][b % 3]
    for window, sinks in ((N, 0), (20, 4)):
        got = window_attention(q, k, v, window=window, sinks=sinks).double()
        want, bound = _reference(q, k, v, window, sinks, D ** -0.5, None)
        before = (torch.arange(N, device=DEV)[None] < first[:, None])[..., None, None]
        assert (((got - want).abs() <= bound) | ~before).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window,sinks", [(300, 0), (40, 0), (40, 11)])
def test_seen_values_that_are_not_finite(D, bad, window, sinks):
    """One of weight e^-32 or less, which rounds to zero beside the others' in fp16: it
    reaches every query that sees it, in tiles that the mask cuts and in whole ones, and
    no other."""
    N, at = 300, 10
    g = torch.Generator(device=DEV).manual_seed(D)
    q = 1.0 + 0.1 * _rnd(g, 2, 2, N, D)
    k, v = 0.1 * _rnd(g, 2, 2, N, D), _rnd(g, 2, 2, N, D)
    k[:, :, at] = -4.0  # -4 D of 1 / sqrt(D): -32 for D = 64
    v[:, :, at, 3] = bad
    got = window_attention(q, k, v, window=window, sinks=sinks)
    i = torch.arange(N, device=DEV)
    sees = (i >= at) & ((i - at < window) | (at < sinks))
    assert not got[:, sees][..., 3].isfinite().any()
    assert got[:, ~sees].isfinite().all() and got[..., :3].isfinite().all() and got[..., 4:].isfinite().all()


@pytest.mark.parametrize("D", [64, 128])
def test_scores_of_minus_infinity(D):
    """They weigh nothing beside others; a query that sees only such has no softmax
    (NaN), unlike one that sees nothing (zeros)."""
    N, n = 200, 70
    g = torch.Generator(device=DEV).manual_seed(D)
    q, k, v = _rnd(g, 2, 2, N, D).abs() + 0.1, _rnd(g, 2, 1, N, D), _rnd(g, 2, 1, N, D)
    k[:, :, :n] = -float("inf")
    starts = torch.tensor([0, 20], dtype=torch.int32, device=DEV)
    for window, sinks in ((300, 0), (90, 3)):
        got = window_attention(q, k, v, window=window, sinks=sinks, starts=starts)
        assert got[0, :n].isnan().all() and got[1, 20:n].isnan().all() and (got[1, :20] == 0).all()
        # sinks are among the first n keys: the rest see what begins at n
        want, bound = _reference(q, k, v, window, 0, D ** -0.5, starts.clamp(min=n))
        assert ((got.double() - want).abs() <= bound)[:, n:].all()
