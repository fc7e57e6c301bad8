"""Log probabilities, entropies, ranks and alternatives of tokens against 64 bits."""
import pytest
import torch

from atlasinfer_amd import _lib
from atlasinfer_amd.integration.logprobs import token_logprobs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _check(x, tokens, top, got=None):
    """x [B, V] on the device.  Bounds, with R = max - min of a row's finite logits in its sums:
    an exponential's argument is a difference (exact to 2^-24 of itself) times log2(e)
    (2^-24), the exponential 2^-22: relative error of a term e^-y is (2 y 2^-24 + 2^-22),
    and y e^-y <= 1/e, so of Z and of E / Z (terms y e^-y, y^2 e^-y <= 4 / e^2 of the
    largest) with at most 64 terms a lane, 2 more scalings each and 12 joins: 2^-16 is ample
    for up to 2^18 terms (2^10 a lane, each addition 2^-24).  The log adds 2^-22 of itself."""
    got = token_logprobs(x, tokens, top) if got is None else got
    B, V = x.shape
    y = x.double().nan_to_num(-float("inf"), float("inf"), -float("inf"))
    m = y.amax(1, keepdim=True)
    none = (m == -float("inf"))[:, 0]
    d = torch.where(y == m, 0.0, y - m)
    w = d.exp()
    z = w.sum(1, keepdim=True)
    lp = d - z.log()
    p = w / z
    entropy = -(p * torch.where(p > 0, lp, 0.0)).sum(1)
    order = torch.sort(y + 0.0, dim=1, descending=True, stable=True).indices  # -0 as 0
    valid = (tokens >= 0) & (tokens < V)
    t = tokens.clamp(0, V - 1)[:, None]
    rank = torch.where(valid, (order == t).int().argmax(1), -1)
    want = lp.gather(1, t)[:, 0]
    want[none | ~valid] = float("nan")
    lp[none] = float("nan")
    entropy[none] = float("nan")
    assert torch.equal(got.ranks, rank)
    assert torch.equal(got.top_tokens, order[:, :top])
    for a, b in ((got.logprobs, want), (got.top_logprobs, lp.gather(1, order[:, :top])), (got.entropies, entropy)):
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(torch.isinf(a), torch.isinf(b))
        ok = torch.isfinite(b)
        off = (a.double() - b)[ok].abs()
        assert (off <= 2.0 ** -16 + 2.0 ** -21 * b[ok].abs()).all(), off.max()
    return got


def _logits(g, B, V, dtype):
    x = torch.randn(B, V, generator=g, device=DEV) * (1 + 3 * torch.rand(B, 1, generator=g, device=DEV))
    x.scatter_add_(1, torch.randint(0, V, (B, 5), generator=g, device=DEV), 10 * torch.rand(B, 5, generator=g, device=DEV))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (2, 7), (5, 63), (2, 64), (3, 65), (4, 129), (2, 1000), (7, 2049), (1, 8191),
                                 (2, 32000), (1, 50257), (3, 50272), (2, 128256), (600, 1031), (1, 262144), (130, 4099)])
def test_sizes(dtype, B, V):
    g = torch.Generator(device=DEV).manual_seed(B + V)
    x = _logits(g, B, V, dtype)
    tokens = torch.randint(0, V, (B,), generator=g, device=DEV)
    tokens[::2] = x[::2].float().argmax(1)
    for top in sorted({0, 1, min(5, V), min(20, V), min(64, V)}):
        _check(x, tokens, top)
    for n in (0, V - 1, V // 2):
        _check(x, torch.full_like(tokens, n), 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties(dtype):
    """Rows of few values, constant rows, blocks of equal large ones: by index."""
    g = torch.Generator(device=DEV).manual_seed(2)
    for V in (50, 1500, 40000, 128256):
        x = torch.randint(-3, 3, (6, V), generator=g, device=DEV).to(dtype)
        x[1] = 0.0
        x[1, ::2] = -0.0
        x[2] = -7.5
        x[3] = torch.arange(V, device=DEV) // max(1, V // 9)
        x[4, V // 2:] = 3.0
        x[5, :V // 3] = -float("inf")
        for n in (0, 1, V // 2, V - 1):
            for top in (1, 7, min(50, V)):
                _check(x, torch.full((6,), n, device=DEV), top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [10, 777, 50272])
def test_masked_and_not_finite(dtype, V):
    """Vocabularies masked to a few tokens by -inf or the type's lowest value, rows with
    nothing left, +inf, NaN."""
    g = torch.Generator(device=DEV).manual_seed(V)
    low, inf, nan = torch.finfo(dtype).min, float("inf"), float("nan")
    x = _logits(g, 12, V, dtype)
    keep = torch.randint(0, V, (12, 4), generator=g, device=DEV)
    masked = torch.full_like(x, -inf).scatter_(1, keep, x.gather(1, keep))
    x[0], x[1] = masked[0], masked[1].clamp(min=low)
    x[2], x[3], x[4] = -inf, low, nan
    x[5, V // 2], x[6, ::3] = inf, inf
    x[7, ::2], x[8, 1:] = nan, nan
    x[9] = low
    x[9, 3] = -inf
    x[10, ::2] = low
    x[11] = -inf
    x[11, V - 1] = low
    for n in (0, 3, V // 2, V - 1):
        for top in (0, 1, min(20, V)):
            _check(x, torch.full((12,), n, device=DEV), top)
    _check(x, keep[:, 0].contiguous(), min(10, V))


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_ones_in_few_lanes(dtype):
    """A short list that overflows: equal steps that put every large logit into the same threads' pieces."""
    V = 131072
    E = 4 if dtype == torch.float32 else 8
    x = torch.randn(2, V, device=DEV)
    piece = torch.arange(V, device=DEV) // E % 256
    x[0, piece < 3] += 50.0
    x[1, piece == 255] = torch.linspace(60, 90, int((piece == 255).sum()), device=DEV)
    x = x.to(dtype)
    for top in (5, 64):
        _check(x, torch.tensor([5, V - 1], device=DEV), top)


def test_tokens_outside():
    x = torch.randn(4, 100, device=DEV)
    _check(x, torch.tensor([-1, 100, 1 << 40, -(1 << 50)], device=DEV), 3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    """Rows on any element, rows apart, a transposed view, one row of a view."""
    g = torch.Generator(device=DEV).manual_seed(5)
    wide = _logits(g, 5, 9000, dtype)
    tokens = torch.tensor([3, 1, 4, 1, 5], device=DEV)
    for skip in (0, 1, 3, 7):
        for V in (1, 5, 100, 8003):
            _check(wide[:, skip:skip + V], tokens % V, min(9, V))
    x = _logits(g, 300, 5, dtype).t()
    assert x.stride(1) != 1
    _check(x, tokens, 9)
    _check(wide[3:4, 1:8000], tokens[:1], 64)
    flat = wide.view(-1)
    for V in (4097, 4099):  # odd rows back to back
        _check(flat[1:1 + 5 * V].view(5, V), tokens, 20)


def test_no_workspace_and_repeats():
    """One workgroup a row gives the same tokens and ranks; a call repeats itself bit for bit."""
    L = _lib.load()
    x = torch.randn(3, 100000, device=DEV).half()
    tokens = torch.tensor([0, 77777, 99999], device=DEV)
    assert L.aq_token_logprobs_workspace(3, 100000, 0, 20) > 0
    a, b = token_logprobs(x, tokens, 20), token_logprobs(x, tokens, 20)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    out = [torch.empty_like(t) for t in a]
    _lib.check(L.aq_token_logprobs(x.data_ptr(), 0, 3, 100000, 100000, tokens.data_ptr(), 20, *[t.data_ptr() for t in out],
                                   None, 0, torch.cuda.current_stream().cuda_stream), "aq_token_logprobs")
    _check(x, tokens, 20, type(a)(*out))


def test_streams_and_graph():
    xs = [torch.randn(2, 60000, device=DEV).half() for _ in range(2)]
    tokens = torch.tensor([5, 6], device=DEV)
    want = [token_logprobs(x, tokens, 8) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(4):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(token_logprobs(x, tokens, 8))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))
    x = xs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = token_logprobs(x, tokens, 8)
    for n in range(4):
        x.copy_(torch.randn_like(x))
        tokens.add_(100)
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, token_logprobs(x, tokens, 8)))


def test_python_refusals():
    x, t = torch.randn(3, 50, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for args in ((x[0], t), (x.double(), t), (x.long(), t), (x, t.int()), (x, t[:2]), (x, t.cpu()), (x, t, 51), (x, t, -1),
                 (torch.randn(3, 100, device=DEV), t, 65), (x[:, :0], t), (torch.empty(1, (1 << 18) + 1, device=DEV), t[:1]),
                 (x, torch.zeros(6, dtype=torch.int64, device=DEV)[::2])):
        with pytest.raises(ValueError):
            token_logprobs(*args)
    with pytest.raises(RuntimeError, match="gradients"):
        token_logprobs(x.clone().requires_grad_(), t)
    out = token_logprobs(x[:0], t[:0], 4)
    assert out.logprobs.shape == (0,) and out.top_tokens.shape == (0, 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_fewer_lanes_than_alternatives(dtype):
    """Rows that fewer threads share than alternatives are asked for, whole and off the 16-byte grid: everything is listed."""
    x = torch.randn(3, 600, device=DEV).to(dtype)
    tokens = torch.tensor([0, 99, 63], device=DEV)
    for V in (64, 255, 256, 263, 300, 503, 504, 511, 512, 517, 518, 519, 526, 540):
        for skip in (0, 1, 5):
            _check(x[:, skip:skip + V], tokens, 64)
            _check(x[:, skip:skip + V], tokens, 9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e4, 1e6, 1.6e7, 1e8, 1e20, 5e29, 2e30, 1e37])
def test_large_logits(dtype, size):
    """Rows of either sign up to the type's range, alone and with ordinary ones; whole rows near one large number."""
    g = torch.Generator(device=DEV).manual_seed(3)
    for V in (300, 50272):
        x = torch.randn(8, V, generator=g, device=DEV)
        x[0] *= size
        x[1] = x[1].abs() * -size - size
        x[2, ::7] -= size
        x[3, V // 3] += size
        x[4] = x[4] * 3 + size
        x[5] = x[5] * 3 - size
        x[6] = torch.where(x[6] > 1, -size, size)
        x[7, V // 2:] = -size
        x = x.to(dtype)
        for n in (0, V // 3, V - 1):
            _check(x, torch.full((8,), n, device=DEV), min(9, V))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 5, 8, 17, 64])
def test_short_rows_to_the_last_bits(dtype, V):
    """Rows of one piece a lane, logits of a few units, where the sums' own roundings are few.  Relative to Z, in
    units of 2^-24: 18 additions (8 a lane, 6 of a wave's lanes, 4 waves), three exponentials of 2^-22 and their
    products (15), exponents off by 1.5 of the mean distance D from the maximum (D <= log V < 4.2: 7) and 1.5 of a lane's
    distance, which the lanes near the maximum, e^-y of the sum, weigh by y e^-y <= 1/e: 1, in all
    below 64, so 2^-18 of log Z.  E has the same on each of its terms and one product more; log and subtractions
    add 2^-22 of their results."""
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (2.0 * torch.randn(400, V, generator=g, device=DEV)).to(dtype)
    tokens = torch.randint(0, V, (400,), generator=g, device=DEV)
    got = token_logprobs(x, tokens, min(5, V))
    y = x.double()
    d = y - y.amax(1, keepdim=True)
    z = d.exp().sum(1, keepdim=True)
    lp, mean = d - z.log(), -(d.exp() / z * d).sum(1)
    want = lp.gather(1, tokens[:, None])[:, 0]
    assert ((got.logprobs.double() - want).abs() <= 2.0 ** -18 + 2.0 ** -22 * want.abs()).all()
    top = torch.sort(lp, dim=1, descending=True, stable=True).values[:, :min(5, V)]
    assert ((got.top_logprobs.double() - top).abs() <= 2.0 ** -18 + 2.0 ** -22 * top.abs()).all()
    entropy = z.log()[:, 0] + mean
    assert ((got.entropies.double() - entropy).abs() <= 2.0 ** -18 * (1 + 2 * mean) + 2.0 ** -22 * entropy).all()
