"""The 4-bit cache: stored codes bit for bit, values read back, a step's
attention against 64 bits, windows with sinks, ragged batches, graphs."""
import pytest
import torch

import kv4_ref as R
from atlasinfer_amd.memory import decode_cache as DC

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _rnd(g, *s):
    return torch.randn(*s, generator=g, device=DEV).half()


def _store_ref(k, v, old, slots, sinks, start, lengths):
    """The cache's unpacked state after a store, position by position."""
    out = [[t.clone() for t in half] for half in old]
    for half, x in zip(out, (k, v)):
        new = R.quantize(x.cpu())
        for b in range(k.shape[0]):
            n = k.shape[2] if lengths is None else min(k.shape[2], max(0, int(lengths[b])))
            for i in range(n):
                s = R.slot_of(start + i, slots, sinks)
                for t, u in zip(half, new):
                    t[b, :, s] = u[b, :, i]
    return out


def _same(cache, want, slots):
    for half, ref in zip(R.unpack(cache, slots), want):
        for got, x in zip(half, ref):
            if got.dtype == torch.float16:  # -0 and 0 are one minimum; NaN for a group that has one
                assert torch.equal(got.isnan(), x.isnan()) and torch.equal(got.nan_to_num() + 0.0, x.nan_to_num() + 0.0)
            else:
                assert torch.equal(got, x)


@pytest.mark.parametrize("B,Hkv,S,D,slots,sinks,start", [
    (1, 1, 1, 64, 1, None, 0), (2, 3, 33, 128, 40, None, 0), (1, 2, 31, 64, 64, None, 33), (2, 2, 77, 128, 200, None, 5),
    (2, 2, 50, 128, 20, 4, 0), (1, 2, 100, 64, 33, 0, 7), (2, 1, 3, 128, 37, 5, 90), (1, 1, 300, 64, 128, 1, 0),
])
def test_store_bits(B, Hkv, S, D, slots, sinks, start):
    g = torch.Generator(device=DEV).manual_seed(S + D)
    k, v = _rnd(g, B, S, Hkv, D).transpose(1, 2), _rnd(g, B, S, Hkv, D).transpose(1, 2)
    k[..., 3] *= 30
    cache = DC.kv4_buffers(B, Hkv, slots, D, DEV)
    for t in cache:  # what is there stays where nothing is written
        t.view(torch.uint8).random_(0, 120, generator=g)
    old = R.unpack(cache, slots)
    lengths = None if B == 1 else torch.tensor([S, S // 2], device=DEV)
    want = _store_ref(k, v, old, slots, sinks, start, lengths)
    DC.kv4_store(k, v, cache, start=start, lengths=lengths, slots=slots, sinks=sinks)
    _same(cache, want, slots)
    for got, half in zip(DC.kv4_load(cache, slots=slots), want):
        x = R.values(*half)
        # one rounding to fp16 of a sum rounded to f32: half a step, and a little;
        # from 65520 on (only what was there before the store) fp16 has infinity
        got, big = got.cpu().double(), x.abs() >= 65520.0
        off = torch.where(big, 0.0, (got - x).abs())
        assert bool((off <= x.abs() * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25).all())
        assert torch.equal(got[big], x[big].sign() * float("inf"))


def test_store_extremes():
    """Equal elements, subnormals, the largest numbers, infinities and NaN."""
    x = torch.zeros(1, 1, 9, 64, dtype=torch.float16)
    x[0, 0, 1] = 3.5
    x[0, 0, 2, ::2] = 6e-8
    x[0, 0, 3, :32] = 65504.0
    x[0, 0, 3, 5] = -65504.0
    x[0, 0, 4] = torch.linspace(-65504, 65504, 64).half()
    x[0, 0, 5, 40] = float("inf")
    x[0, 0, 6, 3] = float("nan")
    x[0, 0, 7] = torch.linspace(-1, 14, 64).half()  # codes at and near ties
    x[0, 0, 8, 1] = -0.0
    k = x.to(DEV)
    cache = DC.kv4_buffers(1, 1, 9, 64, DEV)
    DC.kv4_store(k, k, cache, slots=9)
    want = _store_ref(k, k, R.unpack(DC.kv4_buffers(1, 1, 9, 64, DEV), 9), 9, None, 0, None)
    _same(cache, want, 9)
    back = DC.kv4_load(cache, slots=9)[0].cpu()
    assert torch.isfinite(back[:, :, :5]).all() and torch.isfinite(back[0, 0, 5, :32]).all()
    assert back[0, 0, 5, 32:].isnan().all() and back[0, 0, 6, :32].isnan().all()


def _attention_ref(q, cache, last, scale):
    """Output and error bound of one sequence's heads over slots 0 .. last."""
    (kc, ks, km), (vc, vs, vm) = cache
    k, v = R.values(kc, ks, km)[:, :last + 1], R.values(vc, vs, vm)[:, :last + 1]  # [Hkv, n, D]
    H, D = q.shape
    G = H // k.shape[0]
    k, v, q = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0), q.double()
    ks = ks[:, :last + 1]
    s = (k * q[:, None]).sum(-1) * scale
    w = torch.softmax(s, -1)
    want = (w[..., None] * v).sum(1)
    # scores from sums in f32 of the codes raised by 1024, times the group's scale (8
    # roundings of 2^-24 of at most 1039 s sum |q|, under 2^-11 s sum |q|), and of the
    # minima's part and the exponential: 2^-17 of the terms; values rounded to fp16
    # (2^-11; the numerators are two numbers, 2^-22 or 2^-25 of the largest), the
    # output once
    top = ks.double().amax((1, 2)).repeat_interleave(G, 0)
    ds = (2.0 ** -17 * (k.abs() * q.abs()[:, None]).sum(-1).amax(-1) + 2.0 ** -11 * top * q.abs().sum(-1)) * abs(scale)
    wv = (w[..., None] * v.abs()).sum(1)
    bound = (torch.expm1(2 * ds)[:, None] + 2.0 ** -11 + 2.0 ** -17) * wv + 2.0 ** -24 * v.abs().sum(1)
    bound = bound + 2.0 ** -11 * want.abs() + 2.0 ** -24
    return want, bound


def _step(B, H, Hkv, D, slots, sinks, positions, rope=False, q_scale=1.0, seed=0, poison=True, workspace=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = DC.kv4_buffers(B, Hkv, slots, D, DEV)
    if poison:  # NaN parameters wherever nothing was written
        for t in (cache[1], cache[3]):
            t.fill_(float("nan"))
    most = max(positions)
    k, v = _rnd(g, B, Hkv, most + 1, D), _rnd(g, B, Hkv, most + 1, D)
    lengths = torch.tensor([max(p, 0) for p in positions], device=DEV)
    DC.kv4_store(k, v, cache, lengths=lengths, slots=slots, sinks=sinks)
    q, kn, vn = _rnd(g, B, H, D), _rnd(g, B, Hkv, D), _rnd(g, B, Hkv, D)
    pos = torch.tensor(positions, device=DEV)
    tables = R.rope_tables(most + 1, D, DEV) if rope else None
    before = R.unpack(cache, slots)
    out = torch.full((B, H, D), 77.0, dtype=torch.float16, device=DEV)
    DC.kv4_attention(q, kn, vn, cache, pos, scale=D ** -0.5, slots=slots, sinks=sinks, q_scale=q_scale, rope=tables,
                     out=out, workspace=workspace)
    qr, kr = q, kn
    if q_scale != 1.0:
        qr = (qr.float() * q_scale).half()
    if rope:
        c, s = [t[pos.clamp(min=0)][:, None] for t in tables]
        qr, kr = R.rotate(qr, c, s), R.rotate(kr, c, s)
    want = [[t.clone() for t in half] for half in before]
    for half, x in zip(want, (kr, vn)):
        new = R.quantize(x.cpu())
        for b, p in enumerate(positions):
            if p >= 0:
                for t, u in zip(half, new):
                    t[b, :, R.slot_of(p, slots, sinks)] = u[b]
    _same(cache, want, slots)
    for b, p in enumerate(positions):
        if p < 0:
            assert (out[b] == 77.0).all()
            continue
        ref, bound = _attention_ref(qr[b].cpu(), [[t[b] for t in half] for half in want], min(p, slots - 1), D ** -0.5)
        off = (out[b].cpu().double() - ref).abs()
        assert (off <= bound).all(), (b, p, (off / bound).max())


@pytest.mark.parametrize("D,H,Hkv", [(64, 4, 4), (64, 6, 2), (128, 8, 2), (128, 8, 1), (128, 17, 1), (64, 40, 1)])
@pytest.mark.parametrize("pos", [0, 1, 15, 16, 31, 32, 33, 127, 128, 200])
def test_step(D, H, Hkv, pos):
    _step(2, H, Hkv, D, 201, None, [pos, pos], seed=pos)


@pytest.mark.parametrize("B,H,Hkv,D,slots,sinks,positions", [
    (1, 32, 8, 128, 768, None, [700]),
    (3, 8, 2, 128, 1000, None, [999, -1, 40]),       # one sequence left out
    (2, 4, 2, 64, 5000, None, [4999, 4097]),         # many spans
    (2, 4, 2, 64, 50, 4, [49, 50]),                  # the window's edge
    (3, 8, 2, 128, 100, 4, [150, 99, 1234]),         # past it
    (2, 2, 2, 128, 33, 0, [33, 500]),                # no sinks, a block of one slot
    (1, 4, 1, 64, 5, 4, [77]),                       # a window of one position
    (40, 4, 4, 64, 300, None, [7 * i for i in range(40)]),
])
@pytest.mark.parametrize("rope", [False, True])
def test_step_positions(B, H, Hkv, D, slots, sinks, positions, rope):
    _step(B, H, Hkv, D, slots, sinks, positions, rope=rope, q_scale=1.0 if rope else 0.125, seed=slots)


def test_shared_position_and_bounds():
    """pos of one element; a position past the cache, or past the rotary tables,
    leaves everything as it was."""
    g = torch.Generator(device=DEV).manual_seed(1)
    cache = DC.kv4_buffers(2, 1, 10, 64, DEV)
    DC.kv4_store(_rnd(g, 2, 1, 10, 64), _rnd(g, 2, 1, 10, 64), cache, slots=10)
    q, kn, vn = _rnd(g, 2, 2, 64), _rnd(g, 2, 1, 64), _rnd(g, 2, 1, 64)
    before = [t.clone() for t in cache]
    tables = R.rope_tables(8, 64, DEV)
    for p, kw in [(10, {}), (-1, {}), (8, dict(rope=tables)), (1 << 40, dict(sinks=2)), (8, dict(rope=tables, sinks=2))]:
        out = torch.full((2, 2, 64), 5.0, dtype=torch.float16, device=DEV)
        DC.kv4_attention(q, kn, vn, cache, torch.tensor([p], device=DEV), scale=1.0, slots=10, out=out, **kw)
        assert (out == 5.0).all() and all(torch.equal(a, b) for a, b in zip(cache, before))
    one = DC.kv4_attention(q, kn, vn, cache, torch.tensor([7], device=DEV), scale=0.125, slots=10)
    two = DC.kv4_attention(q, kn, vn, cache, torch.tensor([7, 7], device=DEV), scale=0.125, slots=10)
    assert torch.equal(one, two)


def test_scales():
    """A negative scale is that of the negated queries; with 0 every slot counts alike."""
    g = torch.Generator(device=DEV).manual_seed(3)
    B, H, Hkv, D, slots = 2, 6, 3, 64, 90
    cache = DC.kv4_buffers(B, Hkv, slots, D, DEV)
    DC.kv4_store(_rnd(g, B, Hkv, 80, D), _rnd(g, B, Hkv, 80, D), cache, slots=slots)
    q, kn, vn = _rnd(g, B, H, D), _rnd(g, B, Hkv, D), _rnd(g, B, Hkv, D)
    pos = torch.tensor([80, 50], device=DEV)
    a = DC.kv4_attention(q, kn, vn, cache, pos, scale=-0.2, slots=slots)
    assert torch.equal(a, DC.kv4_attention(-q, kn, vn, cache, pos, scale=0.2, slots=slots))
    got = DC.kv4_attention(q, kn, vn, cache, pos, scale=0.0, slots=slots)
    v = R.values(*R.unpack(cache, slots)[1]).repeat_interleave(H // Hkv, 1)
    for b, p in enumerate(pos.tolist()):
        seen = v[b, :, :p + 1]
        bound = 2.0 ** -10 * seen.abs().mean(1) + 2.0 ** -11 * seen.mean(1).abs() + 2.0 ** -24
        assert ((got[b].cpu().double() - seen.mean(1)).abs() <= bound).all()


def test_steps_in_a_graph():
    """A captured step replayed over growing positions gives the eager steps'
    results, bit for bit, past the window's edge too."""
    B, H, Hkv, D, slots, sinks = 2, 8, 2, 128, 40, 3
    g = torch.Generator(device=DEV).manual_seed(2)
    tables = R.rope_tables(100, D, DEV)
    a, b = DC.DecodeCache(B, Hkv, slots, D, bits=4, sinks=sinks, device=DEV), DC.DecodeCache(B, Hkv, slots, D, bits=4,
                                                                                          sinks=sinks, device=DEV)
    k, v = _rnd(g, B, Hkv, 30, D), _rnd(g, B, Hkv, 30, D)
    a.store(k, v)
    b.store(k, v)
    q, kn, vn = _rnd(g, B, H, D), _rnd(g, B, Hkv, D), _rnd(g, B, Hkv, D)
    pos = torch.tensor([30, 25], device=DEV)
    ws = torch.empty(max(16, a.workspace_bytes(H)), dtype=torch.uint8, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    scratch = DC.DecodeCache(B, Hkv, slots, D, bits=4, sinks=sinks, device=DEV)
    with torch.cuda.stream(s):
        scratch.attend(q, kn, vn, pos, scale=0.1, rope=tables, workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a.attend(q, kn, vn, pos, scale=0.1, rope=tables, workspace=ws)
    for i in range(20):
        for t in (q, kn, vn):
            t.copy_(_rnd(g, *t.shape))
        graph.replay()
        want = b.attend(q, kn, vn, pos, scale=0.1, rope=tables)
        assert torch.equal(out, want)
        assert all(torch.equal(x, y) for x, y in zip(a.buffers, b.buffers))
        pos += 1


def test_refusals():
    cache = DC.kv4_buffers(2, 2, 40, 64, DEV)
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)  # noqa: E731
    pos = torch.zeros(2, dtype=torch.int64, device=DEV)
    ok = dict(scale=1.0, slots=40)
    with pytest.raises(ValueError):
        DC.kv4_attention(h(2, 3, 64), h(2, 2, 64), h(2, 2, 64), cache, pos, **ok)  # 3 heads on 2
    with pytest.raises(ValueError):
        DC.kv4_attention(h(2, 4, 64), h(2, 2, 64), h(2, 1, 64), cache, pos, **ok)
    with pytest.raises(ValueError):
        DC.kv4_attention(h(2, 4, 64).float(), h(2, 2, 64), h(2, 2, 64), cache, pos, **ok)
    with pytest.raises(ValueError):
        DC.kv4_attention(h(2, 4, 64), h(2, 2, 64), h(2, 2, 64), cache, pos.int(), **ok)
    with pytest.raises(ValueError):
        DC.kv4_attention(h(2, 4, 64), h(2, 2, 64), h(2, 2, 64), cache, pos, scale=1.0, slots=70)
    with pytest.raises(ValueError):
        DC.kv4_attention(h(2, 4, 64), h(2, 2, 64), h(2, 2, 64), cache, pos, scale=1.0, slots=40, sinks=40)
    with pytest.raises(ValueError):
        DC.kv4_attention(h(2, 4, 64), h(2, 2, 64), h(2, 2, 64), cache[:3], pos, **ok)
    with pytest.raises(ValueError):
        DC.kv4_store(h(2, 2, 41, 64), h(2, 2, 41, 64), cache, slots=40)
    with pytest.raises(ValueError):
        DC.kv4_store(h(2, 2, 3, 64), h(2, 2, 3, 64), cache, slots=40, lengths=pos.int())
    with pytest.raises(ValueError):
        DC.kv4_load(cache, 41, slots=40)
    with pytest.raises(ValueError):
        DC.kv4_buffers(1, 1, 10, 96, DEV)
    DC.kv4_store(h(2, 2, 0, 64), h(2, 2, 0, 64), cache, slots=40)  # nothing to do


@pytest.mark.parametrize("bits", [4, 16])
def test_positions_of_31_bits(bits):
    """Positions far past a window take the slots of the near ones they are equal to
    modulo it; the last one that is run is 2^31 - 2."""
    g = torch.Generator(device=DEV).manual_seed(9)
    B, H, Hkv, D, slots, sinks = 2, 4, 2, 128, 75, 5
    k, v = _rnd(g, B, Hkv, slots, D), _rnd(g, B, Hkv, slots, D)
    q, kn, vn = _rnd(g, B, H, D), _rnd(g, B, Hkv, D), _rnd(g, B, Hkv, D)
    far = torch.tensor([2 ** 31 - 2, 2 ** 31 - 1000], device=DEV)
    near = sinks + (far - sinks) % (slots - sinks) + 3 * (slots - sinks)
    caches = [DC.DecodeCache(B, Hkv, slots, D, bits=bits, sinks=sinks, device=DEV) for _ in range(3)]
    for c in caches:
        c.store(k, v)
    outs = [c.attend(q, kn, vn, p, scale=0.1) for c, p in zip(caches, (far, near))]
    assert torch.equal(*outs)
    assert all(torch.equal(a, b) for a, b in zip(caches[0].buffers, caches[1].buffers))
    out = torch.full((B, H, D), 3.0, dtype=torch.float16, device=DEV)
    caches[2].attend(q, kn, vn, torch.tensor([2 ** 31 - 1], device=DEV), scale=0.1, out=out)
    assert (out == 3.0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mean", [3.0, 10.0])
@pytest.mark.parametrize("slots", [2, 700])
def test_scores_of_biased_queries(D, mean, slots):
    """Queries far from zero on average, as biases of their projection make them:
    two slots of near scores and values 1 and -1, whose output is tanh of half the
    scores' difference, so that it shows their errors and hardly its own rounding."""
    g = torch.Generator(device=DEV).manual_seed(D + int(mean))
    B, H, Hkv = 24, 8, 2
    q = mean + 0.25 * torch.randint(-1, 2, (B, H, D), generator=g, device=DEV)
    q[torch.rand(B, H, D, generator=g, device=DEV) < 0.8] = mean
    q = q.half()  # whole multiples of 1/4
    # groups of codes 0 .. 15, the lowest of them 0: the minimum is 0, the scale from 1.3 to 2
    codes = torch.randint(0, 16, (B, Hkv, D // 32, 32), generator=g, device=DEV).float()
    codes[..., 0], codes[..., 1] = 0.0, 15.0
    k0 = codes * (1.3 + 0.7 * torch.rand(B, Hkv, D // 32, 1, generator=g, device=DEV))
    k1 = k0[..., torch.randperm(32, generator=g, device=DEV)]
    k0, k1 = k0.half().view(B, Hkv, 1, D), k1.half().view(B, Hkv, D)
    one = torch.ones(B, Hkv, D, dtype=torch.float16, device=DEV)
    cache = DC.kv4_buffers(B, Hkv, slots, D, DEV)
    DC.kv4_store(k0, one[:, :, None], cache, slots=slots)
    got = DC.kv4_attention(q, k1, -one, cache, torch.ones(1, dtype=torch.int64, device=DEV), scale=D ** -0.5,
                           slots=slots).cpu().double()
    (c, s, m), values = R.unpack(cache, slots)
    assert (m[:, :, :2] == 0).all()
    k = R.values(c, s, m)[:, :, :2].repeat_interleave(H // Hkv, 1)
    assert torch.equal(R.values(*values)[:, :, :2], torch.tensor([1.0, -1.0]).double().view(1, 1, 2, 1).expand(B, Hkv, 2, D))
    score = (k * q.cpu().double()[:, :, None]).sum(-1) * D ** -0.5  # [B, H, 2], all terms positive
    delta = score[..., 0] - score[..., 1]
    assert delta.abs().max() < 12
    # sums of codes times quarters are exact, so a score has the roundings of up to four
    # products and sums with the scales, 2^-24 of the score each, and of the exponent's
    # argument, 2^-24 of it: 5 2^-24 of both scores; scale and log2(e) round, 2^-23 of the
    # difference; half of that reaches the output, and the weights' roundings (2^-20 of 1)
    # and its own
    off = 5 * 2.0 ** -24 * score.sum(-1) + 2.0 ** -23 * delta.abs()
    want = torch.tanh(0.5 * delta)
    bound = 0.5 * off + 2.0 ** -20 + 2.0 ** -11 * want.abs() + 2.0 ** -25
    err = (got - want[..., None]).abs()
    assert (err <= bound[..., None]).all(), (err / bound[..., None]).max()
