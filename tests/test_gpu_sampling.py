"""aq_sample against a plain form in 64 bits: every filter, ties, rows that
leave nothing, all types, ragged sizes, settings per row, graphs."""
import math

import pytest
import torch

from atlasinfer_amd.integration.sampling import sample_tokens

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def reference(x, u, t, k, p, m):
    """One row at a time, on the CPU."""
    out = []
    for row, ui, ti, ki, pi, mi in zip(x.double().cpu(), u.double().cpu(), t, k, p, m):
        row = torch.where(row.isnan(), -torch.tensor(float("inf"), dtype=torch.float64), row) + 0.0
        top = row.max()
        order = torch.sort(row, descending=True, stable=True).indices
        if not ti > 0 or top == -float("inf"):
            out.append(int(order[0]))
            continue
        w = torch.where(row == top, 1.0, torch.exp((row - top) / ti).nan_to_num(0.0))
        w = torch.where(row == -float("inf"), 0.0, w)
        keep = order[:ki] if 0 < ki < len(row) else order
        before = torch.cumsum(w[keep], 0) - w[keep]
        if pi < 1:
            keep = keep[(before < pi * w[keep].sum()) | (torch.arange(len(keep)) == 0)]
        if mi > 0:
            keep = keep[(w[keep] >= min(mi, 1.0))]
        mask = torch.zeros_like(w)
        mask[keep] = w[keep]
        c = torch.cumsum(mask, 0)
        hit = (c > ui * c[-1]).nonzero()
        out.append(int(hit[0]) if len(hit) else int(mask.nonzero()[-1]))
    return torch.tensor(out)


def _logits(g, B, V, dtype, spread=2.5):
    x = torch.randn(B, V, generator=g, device=DEV) * spread
    x[:, :: max(1, V // 20)] += 6 * torch.rand(B, len(range(0, V, max(1, V // 20))), generator=g, device=DEV)
    return x.to(dtype)


f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 63, 1000, 8191, 8193, 32000, 50272])
@pytest.mark.parametrize("t,k,p,m", [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (0.8, 0, 0.9, 0.0),
                                     (1.3, 0, 1.0, 0.05), (0.9, 400, 0.95, 0.01), (1.0, 1, 0.5, 1.0), (5.0, 0, 0.5, 0.0)])
def test_settings(dtype, V, t, k, p, m):
    g = torch.Generator(device=DEV).manual_seed(V + int(10 * t))
    B = 4
    x, u = _logits(g, B, V, dtype), torch.rand(B, generator=g, device=DEV)
    got = sample_tokens(x, u, t, k, p, m)
    want = reference(x, u, [f32(t)] * B, [k] * B, [f32(p)] * B, [f32(m)] * B)
    assert torch.equal(got.cpu(), want)


def test_settings_per_row():
    g = torch.Generator(device=DEV).manual_seed(3)
    B, V = 40, 5000
    x, u = _logits(g, B, V, torch.float16), torch.rand(B, generator=g, device=DEV)
    t = torch.rand(B, generator=g, device=DEV) * 1.5
    t[::9] = 0.0
    k = torch.randint(0, 200, (B,), generator=g, device=DEV, dtype=torch.int32)
    k[::7] = 0
    p, m = torch.rand(B, generator=g, device=DEV), torch.rand(B, generator=g, device=DEV) * 0.2
    p[::5] = 1.0
    m[::4] = 0.0
    got = sample_tokens(x, u, t, k, p, m)
    assert torch.equal(got.cpu(), reference(x, u, t.tolist(), k.tolist(), p.tolist(), m.tolist()))
    # the same token whatever else is in the batch, and on every call
    for i in (0, 7, 39):
        one = sample_tokens(x[i:i + 1], u[i:i + 1], t[i:i + 1], k[i:i + 1], p[i:i + 1], m[i:i + 1])
        assert one.item() == got[i].item()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_ties(dtype):
    """Equal logits are taken by index: a row of one value, of two, with both
    zeros, cut inside a tie."""
    V = 9000
    rows = [torch.zeros(V), torch.arange(V) % 2 * 1.0, torch.where(torch.arange(V) % 3 == 0, -0.0, 0.0),
            torch.where(torch.arange(V) < 4, 1.0, 0.0)]
    x = torch.stack(rows).to(dtype).to(DEV)
    for u0 in (0.0, 0.25, 0.5, 0.99999, 1.0):
        u = torch.full((4,), u0, device=DEV)
        for k, p in [(0, 1.0), (7, 1.0), (5000, 1.0), (0, 0.5), (3000, 0.5), (0, 0.001), (8999, 0.75)]:
            got = sample_tokens(x, u, 1.0, k, p)
            assert torch.equal(got.cpu(), reference(x, u, [1.0] * 4, [k] * 4, [f32(p)] * 4, [0.0] * 4)), (u0, k, p)


def test_rows_that_leave_nothing():
    """Infinities and NaN: no token at all, one, several of +inf; greedy too."""
    inf, nan = float("inf"), float("nan")
    V = 3000
    x = torch.full((7, V), -inf)
    x[1, 17] = -5.0
    x[2, ::100] = inf
    x[3] = torch.randn(V, generator=torch.Generator().manual_seed(0))
    x[3, :1500] = -inf
    x[4] = nan
    x[5], x[5, 2000] = nan, 1.0
    x[6], x[6, 5], x[6, 9] = 0.0, inf, nan
    for dtype in (torch.float16, torch.float32):
        y = x.to(dtype).to(DEV)
        for t in (0.0, 1.0, 1e-30, 1e30, inf):
            for k, p, m in [(0, 1.0, 0.0), (2, 0.9, 0.0), (0, 0.4, 0.1)]:
                u = torch.full((7,), 0.6, device=DEV)
                got = sample_tokens(y, u, t, k, p, m)
                want = reference(y, u, [f32(t)] * 7, [k] * 7, [f32(p)] * 7, [f32(m)] * 7)
                assert torch.equal(got.cpu(), want), (dtype, t, k, p, m)


def test_strides_largest_vocabulary_and_distribution():
    g = torch.Generator(device=DEV).manual_seed(5)
    wide = torch.randn(3, 70001, generator=g, device=DEV).half()
    u = torch.rand(3, generator=g, device=DEV)
    assert torch.equal(sample_tokens(wide[:, 1:60000], u, 0.9, 0, 0.9), sample_tokens(wide[:, 1:60000].contiguous(), u, 0.9, 0, 0.9))
    assert torch.equal(sample_tokens(wide[:, ::2], u, 0.9, 30), sample_tokens(wide[:, ::2].contiguous(), u, 0.9, 30))
    x = torch.randn(1, 1 << 18, generator=g, device=DEV)
    u = torch.tensor([0.37], device=DEV)
    assert torch.equal(sample_tokens(x, u, 1.1, 0, 0.8).cpu(), reference(x, u, [f32(1.1)], [0], [f32(0.8)], [0.0]))
    # evenly spaced numbers give each token its share, to one number in n
    n = 4096
    row = torch.tensor([[0.0, 1.0, -1.0, 2.0]], device=DEV).expand(n, 4).contiguous()
    tok = sample_tokens(row, (torch.arange(n, device=DEV) + 0.5) / n)
    share = torch.bincount(tok, minlength=4).cpu() / n
    assert ((share - torch.softmax(row[0].cpu(), 0)).abs() <= 1.0 / n).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 16384), (1, 50272), (3, 50273), (2, 128256), (100, 20011), (1, 1 << 18)])
def test_rows_in_parts(dtype, B, V):
    """Long rows of small batches are shared by workgroups: the same tokens as
    the plain form's and as one workgroup's, misaligned rows, ties past the
    list's room, greedy and top-k rows among others, a row without a token."""
    from atlasinfer_amd import _lib
    g = torch.Generator(device=DEV).manual_seed(V + B)
    n = min(B, 4)
    wide = torch.empty(B, V + 3, dtype=dtype, device=DEV)
    wide[:, 1:V + 1] = _logits(g, B, V, dtype, 1.5)
    x, u = wide[:, 1:V + 1], torch.rand(B, generator=g, device=DEV)
    for t, k, p, m in [(0.8, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (1.2, 0, 1.0, 0.03), (3.0, 0, 0.6, 0.01)]:
        assert _lib.load().aq_sample_workspace(B, V, 0, k) > 0 or dtype == torch.float32 or B > 64
        got = sample_tokens(x, u, t, k, p, m)
        want = reference(x[:n], u[:n], [f32(t)] * n, [k] * n, [f32(p)] * n, [f32(m)] * n)
        assert torch.equal(got[:n].cpu(), want), (t, k, p, m)
        # one workgroup a row: the same call with settings that rule the parts out
        one = torch.empty_like(got)
        _lib.check(_lib.load().aq_sample(x.data_ptr(), [torch.float16, torch.bfloat16, torch.float32].index(dtype), B, V,
                                         x.stride(0), u.data_ptr(), None, None, None, None, t, k, p, m, one.data_ptr(),
                                         None, 0, _lib.stream_of(DEV)), "aq_sample")
        assert torch.equal(one, got)
    flat = torch.zeros(4, V, dtype=dtype, device=DEV)  # one value; two; none; one number among -inf
    flat[1, ::3] = 1.0
    flat[2] = -float("inf")
    flat[3] = -float("inf")
    flat[3, V // 2] = -3.0
    v = torch.tensor([0.999, 0.3, 0.5, 0.7], device=DEV)
    for p in (1.0, 0.7):
        assert torch.equal(sample_tokens(flat, v, 1.0, 0, p).cpu(), reference(flat, v, [1.0] * 4, [0] * 4, [f32(p)] * 4, [0.0] * 4))
    # rows of every kind in one call
    y, w = x[:n].contiguous(), u[:n].contiguous()
    t = torch.tensor([0.0, 0.7, 1.0, 1.5][:n], device=DEV)
    k = torch.tensor([0, 40, 0, 0][:n], dtype=torch.int32, device=DEV)
    p = torch.tensor([0.9, 0.9, 1.0, 0.95][:n], device=DEV)
    assert torch.equal(sample_tokens(y, w, t, k, p).cpu(), reference(y, w, t.tolist(), k.tolist(), p.tolist(), [0.0] * n))


def test_in_a_graph():
    g = torch.Generator(device=DEV).manual_seed(6)
    x, u = _logits(g, 3, 20000, torch.float16), torch.rand(3, generator=g, device=DEV)
    t = torch.ones(3, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sample_tokens(x, u, t, 50, 0.9)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(x, u, t, 50, 0.9)
    whole, u2 = _logits(g, 2, 128256, torch.float16), torch.rand(2, generator=g, device=DEV)
    parts = torch.cuda.CUDAGraph()
    sample_tokens(whole, u2, 0.9, 0, 0.95)
    with torch.cuda.graph(parts):
        out2 = sample_tokens(whole, u2, 0.9, 0, 0.95)
    for i in range(8):
        whole.copy_(_logits(g, 2, 128256, torch.float16))
        parts.replay()
        assert torch.equal(out2, sample_tokens(whole, u2, 0.9, 0, 0.95))
        x.copy_(_logits(g, 3, 20000, torch.float16))
        u.copy_(torch.rand(3, generator=g, device=DEV))
        t.fill_(0.2 * i)
        graph.replay()
        assert torch.equal(out, sample_tokens(x, u, t, 50, 0.9))


def test_refusals():
    x, u = torch.zeros(2, 10, device=DEV), torch.zeros(2, device=DEV)
    for args, kw in [((x[0], u), {}), ((x.double(), u), {}), ((x.cpu(), u), {}), ((x, u.double()), {}), ((x, u[:1]), {}),
                     ((x, u), dict(temperature=torch.ones(1, device=DEV))), ((x, u), dict(top_k=torch.ones(2, device=DEV))),
                     ((x, u), dict(top_p=torch.ones(2))), ((x, u), dict(out=torch.zeros(2, dtype=torch.int32, device=DEV))),
                     ((torch.zeros(1, (1 << 18) + 1, device=DEV), u[:1]), {}), ((torch.zeros(2, 0, device=DEV), u), {})]:
        with pytest.raises(ValueError):
            sample_tokens(*args, **kw)
    assert sample_tokens(x[:0], u[:0]).shape == (0,)


def test_more_long_rows_than_workgroups_fit():
    """More than 256 rows are never split, however long."""
    g = torch.Generator(device=DEV).manual_seed(21)
    x = torch.randn(300, 17000, generator=g, device=DEV).half()
    u = torch.rand(300, generator=g, device=DEV)
    got = sample_tokens(x, u, 0.9, 0, 0.8)
    parts = torch.cat([sample_tokens(x[i:i + 75], u[i:i + 75], 0.9, 0, 0.8) for i in range(0, 300, 75)])
    assert torch.equal(got, parts)


@pytest.mark.parametrize("V", [1001, 32000, 50273])
def test_rows_of_the_lowest_numbers(V):
    """Rows whose largest logit is the lowest number fp32 has, or near it (what
    masking with finfo.min leaves): -inf, NaN and what lies before and behind the row
    weigh nothing there either."""
    low, inf = torch.finfo(torch.float32).min, float("inf")
    x = torch.full((5, V), low)
    x[1, ::3] = -inf
    x[2] = -inf
    x[2, [V // 3, V - 2]] = low
    x[3] = torch.linspace(low, low * 0.999, V)
    x[3, ::4] = float("nan")
    x[4, 7:] = -inf
    wide = torch.zeros(5, V + 3, device=DEV)
    wide[:, 1:V + 1] = x.to(DEV)
    y = wide[:, 1:V + 1]
    for u0 in (0.0, 0.37, 0.99999):
        u = torch.full((5,), u0, device=DEV)
        for t in (0.01, 1.0, 2e33, inf):  # 2e33: the numbers of row 3 differ in weight
            for k, p, m in [(0, 1.0, 0.0), (0, 0.7, 0.0), (700, 1.0, 0.0), (5, 0.6, 0.1), (0, 1.0, 0.5)]:
                got = sample_tokens(y, u, t, k, p, m)
                # temperatures above 1e34 count as 1e34, weights below 2^-43 round to nothing
                # (the running mass exceeds 0 at the first that does not)
                tt = min(f32(t), f32(1e34))
                z = x.double().nan_to_num(nan=-inf, neginf=-inf)
                z = torch.where((z - z.amax(-1, keepdim=True)) / tt < -43 * math.log(2.0), -inf, z)
                want = reference(z, u, [tt] * 5, [k] * 5, [f32(p)] * 5, [f32(m)] * 5)
                assert torch.equal(got.cpu(), want), (u0, t, k, p, m)


def test_lowest_numbers_of_bf16():
    V, low = 9001, torch.finfo(torch.bfloat16).min
    x = torch.full((2, V), low)
    x[1, 5:] = -float("inf")
    for t in (1.0, 1e34):
        got = sample_tokens(x.bfloat16().to(DEV), torch.full((2,), 0.6, device=DEV), t)
        assert torch.equal(got.cpu(), reference(x, torch.full((2,), 0.6), [f32(t)] * 2, [0] * 2, [1.0] * 2, [0.0] * 2))


def test_tiny_temperatures():
    """Temperatures of a fraction of the step between fp32 numbers: what lies below
    the largest number weighs nothing, -inf among it."""
    x = torch.full((1, 3000), -float("inf"), device=DEV)
    x[0, 1234] = 1.0
    u = torch.full((1,), 0.9999999, device=DEV)
    for steps in (0.3, 0.9, 1.1, 1.3, 1.45, 1.6, 3.0):
        t = steps * 2.0 ** -24 / 41.6  # the distance at which weights end, in steps below 1
        for p in (1.0, 0.9):
            assert sample_tokens(x, u, t, 0, p).item() == 1234, (steps, p)
            assert sample_tokens(x, torch.zeros_like(u), t, 0, p).item() == 1234, (steps, p)


@pytest.mark.parametrize("n,d,t", [(7, 7.161129951477051, 3.6800928115844727), (3, 15.558229446411133, 14.161710739135742),
                                   (3, 12.468780517578125, 11.349573135375977), (2, 4.920184135437012, 7.098325252532959),
                                   (7, 14.07146167755127, 7.2313008308410645)])
def test_weights_at_a_border(n, d, t):
    """n tokens d below the largest, with n exp(-d / t) = 1 + e, e from 7e-12 to 1.4e-11:
    at u = 1/2 the last of them is the token, by a margin of e / 2, which is 15 to 30 units
    of 2^-42; their roundings are n / 2 units at most."""
    x = torch.tensor([[-d] * n + [0.0]], device=DEV)
    assert sample_tokens(x, torch.full((1,), 0.5, device=DEV), t).item() == n - 1
