"""The paged cache: new tokens with rotary positions into it, and attention over
it, against 64 bits."""
import pytest
import torch

import paged_ref as R
from atlasinfer_amd.memory.paged_cache import (PagedBatch, Rotary, paged_attention, paged_attention_workspace,
                                               paged_buffers, paged_store, rotary_frequencies)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F16, BF16 = torch.float16, torch.bfloat16


def _batch(b, max_new=None, max_length=None):
    n, x = b.bounds()
    return PagedBatch(b.starts, b.lengths, b.table, max_new or n, max_length or x)


# ---------------------------------------------------------------- store


def _check_store(news, contexts, H, Hkv, D, P, dtype, rotary, interleaved, factor=1.0, before=0, after=0, seed=0):
    b = R.Batch(news, contexts, Hkv, D, P, dtype, DEV, seed, before=before, after=after)
    x = b.normal(b.T, H + 2 * Hkv, D).to(dtype)  # the three side by side, as one product gives them
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    rope = None
    if rotary:
        rope = Rotary(rotary_frequencies(rotary, 500000.0, device=DEV)[0], interleaved, factor)
    was = [t.clone() for t in b.cache]
    q_out = torch.full((b.T, H, D), 7.0, dtype=dtype, device=DEV) if H else None
    got = paged_store(k, v, b.cache, _batch(b), q=q if H else None, rope=rope, q_out=q_out)
    assert got is q_out
    h = R.HALF[dtype]
    left = [torch.ones(t.shape[:1] + t.shape[2:3], dtype=torch.bool, device=DEV) for t in was]
    for i in range(len(news)):
        rows = slice(b.first[i], b.first[i + 1])
        p = b.positions(i)
        for t, out in ((k, b.held(0, i)[:, contexts[i]:].transpose(0, 1)), (q, got[rows] if H else None)):
            if out is None:
                continue
            want, size = R.turn(t[rows], p, rope.frequencies if rope else None, interleaved, factor)
            # cos, sin and the products in f32: 2^-21 of the terms
            assert ((out.double() - want).abs() <= h * want.abs() + 2.0 ** -21 * size * (1 + h) + 2.0 ** -25 * (size > 0)).all()
            if rope:
                assert torch.equal(out[..., rotary:], t[rows][..., rotary:])
            else:
                assert torch.equal(out, t[rows])
        assert torch.equal(b.held(1, i)[:, contexts[i]:].transpose(0, 1), v[rows])
        page = b.table[i].long()[p // P]
        for t in left:
            t[page, p % P] = False
    for t, w, keep in zip(b.cache, was, left):  # every other slot as it was
        assert torch.equal(t.transpose(1, 2)[keep], w.transpose(1, 2)[keep])
    if H:
        assert (got[:before] == 7).all() and (got[b.first[-1]:] == 7).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,rotary", [(64, 0), (64, 16), (64, 64), (128, 128), (128, 32), (128, 112)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_store(dtype, D, rotary, interleaved):
    _check_store([3, 0, 1, 37], [5, 9, 0, 40], 4, 2, D, 16, dtype, rotary, interleaved, 1.2, before=2, after=3)


@pytest.mark.parametrize("news,contexts,P", [([1], [0], 16), ([1], [15], 16), ([1], [16], 16), ([300], [0], 128),
                                             ([1] * 40, list(range(40)), 16), ([0, 0, 5, 0], [3, 0, 60, 0], 64)])
def test_store_places(news, contexts, P):
    _check_store(news, contexts, 6, 3, 64, P, F16, 64, False)
    _check_store(news, contexts, 0, 1, 128, P, BF16, 128, True)


def test_store_many_sequences():
    """More than a workgroup's threads can look at in one go."""
    news = [(7 * i) % 3 for i in range(700)]
    _check_store(news, [(11 * i) % 50 for i in range(700)], 2, 1, 64, 16, F16, 64, False)


@pytest.mark.parametrize("far", [1 << 16, (1 << 20) + 12345, (1 << 26) + 77])
def test_store_far_positions(far):
    """Angles of far positions; only the last pages of the table are looked at."""
    P, D, n = 1024, 128, 9
    k, v = torch.randn(n, 2, D, device=DEV).half(), torch.randn(n, 2, D, device=DEV).half()
    cache = paged_buffers(3, 2, P, D, device=DEV)
    W = (far + n) // P + 1
    table = torch.full((1, W), -1, dtype=torch.int32, device=DEV)
    table[0, far // P:] = torch.tensor([2, 1], dtype=torch.int32, device=DEV)[:W - far // P]
    f = rotary_frequencies(D, device=DEV)[0]
    b = PagedBatch(torch.tensor([0, n], dtype=torch.int32, device=DEV), torch.tensor([far + n], dtype=torch.int32, device=DEV),
                   table, n, far + n)
    paged_store(k, v, cache, b, rope=Rotary(f))
    p = torch.arange(far, far + n, device=DEV)
    want, size = R.turn(k, p, f, False, 1.0)
    got = cache[0][table[0].long()[p // P], :, p % P].double()
    assert ((got - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -21 * size * 1.01 + 2.0 ** -25).all()


def test_store_leaves_out():
    """Sequences that pass the host's bounds, rows without one, pages outside the
    cache: nothing else is touched, the others are as ever."""
    P, D, Hkv, H = 16, 64, 2, 2
    news, contexts = [4, 6, 2, 3], [20, 1, 30, 0]
    b = R.Batch(news, contexts, Hkv, D, P, F16, DEV)
    q, k, v = b.normal(b.T, H, D).half(), b.normal(b.T, Hkv, D).half(), b.normal(b.T, Hkv, D).half()
    was = [t.clone() for t in b.cache]
    table = b.table.clone()
    table[0, 1] = 10 ** 6  # sequence 0's new tokens lie in its second page
    lengths = b.lengths.clone()
    lengths[3] = 2  # fewer positions than new tokens
    batch = PagedBatch(b.starts, lengths, table, 4, 32)  # sequence 1 has more than 4 new ones
    q_out = torch.full_like(q, 7.0)
    paged_store(k, v, b.cache, batch, q=q, q_out=q_out)
    at = b.first
    assert torch.equal(q_out[at[0]:at[1]], q[at[0]:at[1]])  # its queries need no page
    assert (q_out[at[1]:at[2]] == 7).all() and (q_out[at[3]:] == 7).all()
    assert torch.equal(q_out[at[2]:at[3]], q[at[2]:at[3]])
    page = b.table[2].long()
    for t, w, new in zip(b.cache, was, (k, v)):
        assert torch.equal(t[page[1], :, 14:].transpose(0, 1), new[at[2]:at[3]])
        t[page[1], :, 14:] = w[page[1], :, 14:]
        assert torch.equal(t, w)


# ---------------------------------------------------------------- attention


def _check(news, contexts, H, Hkv, D, P=16, dtype=F16, window=None, sinks=0, scale=None, seed=0, before=0, after=0,
           poison=None, whole=False, keys=1.0):
    b = R.Batch(news, contexts, Hkv, D, P, dtype, DEV, seed, before=before, after=after)
    b.cache[0].mul_(keys)
    if poison is not None:
        poison(b)
    q = b.normal(b.T, H, D).to(dtype)
    scale = D ** -0.5 if scale is None else scale
    max_length = b.table.shape[1] * P if whole else None  # a bound as long as the table
    out = torch.full((b.T, H, D), 7.0, dtype=dtype, device=DEV)
    got = paged_attention(q, b.cache, _batch(b, max_length=max_length), scale=scale, window=window, sinks=sinks, out=out)
    assert got is out and (out[:before] == 7).all() and (out[b.first[-1]:] == 7).all()
    for i in range(len(news)):
        if news[i]:
            want, bound = R.attend(q[b.first[i]:b.first[i + 1]], b, i, scale, window, sinks)
            off = (out[b.first[i]:b.first[i + 1]].double() - want).abs()
            assert (off <= bound).all(), (i, (off / bound).max())
    again = paged_attention(q, b.cache, _batch(b, max_length=max_length), scale=scale, window=window, sinks=sinks)
    assert torch.equal(again[before:b.first[-1]], out[before:b.first[-1]])
    return b, q, out


HEADS = [(2, 2, 64), (4, 1, 128), (10, 2, 64), (8, 1, 128), (3, 3, 128)]


@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 513])
def test_single_tokens(H, Hkv, D, L):
    _check([1], [L - 1], H, Hkv, D, seed=L)
    _check([1, 1, 1], [L - 1, 0, L // 2], H, Hkv, D, 32, BF16, seed=L + 1)


@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("n,context", [(2, 0), (3, 77), (8, 8), (9, 200), (33, 0), (40, 1000), (129, 0), (128, 64), (300, 5)])
def test_chunks(H, Hkv, D, n, context):
    _check([n], [context], H, Hkv, D, seed=n)
    _check([n, 1, n // 2], [context, context + 3, 0], H, Hkv, D, 64, BF16, seed=n + 1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_mixtures(dtype, D):
    """Prompts, chunks, single tokens and idle sequences in one call, rows around them that belong to none."""
    _check([1, 0, 200, 1, 5, 0, 33, 1], [700, 90, 0, 0, 1200, 0, 321, 2000], 8, 2, D, dtype=dtype, before=3, after=5)
    _check([0, 0, 1], [10, 0, 40], 5, 1, D, dtype=dtype)


@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("news,contexts,window,sinks", [
    ([1], [300], 20, 3), ([1], [300], 1, 0), ([5], [295], 64, 0), ([130], [570], 1, 1), ([300], [0], 64, 65),
    ([300], [0], 65, 300), ([257], [743], 128, 4), ([1000], [0], 63, 1), ([640], [0], 1000, 7),
    ([1, 100, 1, 7], [3000, 900, 5, 2000], 256, 17)])
def test_windows(H, Hkv, D, news, contexts, window, sinks):
    _check(news, contexts, H, Hkv, D, window=window, sinks=sinks, seed=len(news))
    _check(news, contexts, H, Hkv, D, 128, BF16, window=window, sinks=sinks, seed=len(news))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("news,contexts", [([1], [9000]), ([1, 1], [4097, 9000]), ([3, 1], [6000, 100]), ([70], [7000]),
                                           ([200], [9000])])
def test_long_contexts(D, news, contexts):
    """Keys split among workgroups and merged; a generous bound on the length."""
    _check(news, contexts, 4, 1, D, seed=1)
    _check(news, contexts, 2, 2, D, 32, BF16, seed=2, whole=True)
    _check(news, contexts, 4, 1, D, window=5000, sinks=70, seed=3)


def test_many_sequences():
    _check([(5 * i) % 4 for i in range(300)], [(37 * i) % 200 for i in range(300)], 4, 2, 64)
    _check([1] * 150, [(91 * i) % 400 for i in range(150)], 2, 1, 128, dtype=BF16)


def test_thousands_of_sequences():
    """More sequences than one look at 64 of 64 finds: rows and blocks in their places."""
    S = 4500
    news = [(7 * i) % 3 for i in range(S)]
    news[2000], news[4400] = 40, 150
    contexts = [(13 * i) % 40 for i in range(S)]
    b = R.Batch(news, contexts, 1, 64, 16, F16, DEV)
    q = b.normal(b.T, 2, 64).half()
    got = paged_attention(q, b.cache, _batch(b), scale=0.125)
    for i in list(range(0, S, 371)) + [1999, 2000, 2001, 4400, 4498, 4499]:
        if news[i]:
            want, bound = R.attend(q[b.first[i]:b.first[i + 1]], b, i, 0.125)
            assert ((got[b.first[i]:b.first[i + 1]].double() - want).abs() <= bound).all(), i
    _check_store([(5 * i) % 2 for i in range(S)], [(11 * i) % 30 for i in range(S)], 1, 1, 64, 16, F16, 64, False)


def test_shared_and_freed_pages():
    """Sequences that share the pages of a common beginning; pages that have left the window, given back."""
    P, n = 16, 64
    b = R.Batch([1, 30, 2], [100, 80, n], 2, 64, P, F16, DEV)
    b.table[1, :n // P] = b.table[0, :n // P]
    b.table[2, :n // P] = b.table[0, :n // P]
    for i in (1, 2):
        b.pages[i][:n // P] = b.pages[0][:n // P]
    q = b.normal(b.T, 4, 64).half()
    got = paged_attention(q, b.cache, _batch(b), scale=0.1)
    for i in range(3):
        want, bound = R.attend(q[b.first[i]:b.first[i + 1]], b, i, 0.1)
        assert ((got[b.first[i]:b.first[i + 1]].double() - want).abs() <= bound).all()
    # nothing before position 100 - 39 is seen by any row through a window of 40, but for 3 sinks
    b = R.Batch([1, 70], [100, 100], 2, 128, P, F16, DEV)
    q = b.normal(b.T, 4, 128).half()
    want = paged_attention(q, b.cache, _batch(b), scale=0.1, window=40, sinks=3)
    b.table[:, 1:61 // P] = torch.tensor([-1, 1 << 30], dtype=torch.int32, device=DEV)
    assert torch.equal(paged_attention(q, b.cache, _batch(b), scale=0.1, window=40, sinks=3), want)


def test_large_scores_and_scales():
    """Peaked rows (keys 30 times as large), a negative scale, and 0, with which every key seen counts alike."""
    for D in (64, 128):
        for news, contexts in (([1, 1], [300, 1000]), ([150], [100])):
            _check(news, contexts, 4, 2, D, keys=30.0)
            _check(news, contexts, 4, 2, D, scale=-0.2)
            _check(news, contexts, 4, 2, D, scale=0.0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_unseen_values_do_not_matter(D, dtype, bad):
    """NaN and infinities where no row may look: behind the sequence's end in its
    last page, in pages of nobody, before the window, in the future of a row."""

    def behind(b):
        for t in b.cache:
            seen = torch.zeros(t.shape[0], t.shape[2], dtype=torch.bool, device=DEV)
            for i, x in enumerate(b.len):
                j = torch.arange(x, device=DEV)
                seen[b.table[i].long()[j // b.P], j % b.P] = True
            t.transpose(1, 2)[~seen] = bad
    for news, contexts in (([1], [40]), ([1, 1], [500, 3]), ([9, 70], [30, 8]), ([200], [33])):
        _check(news, contexts, 4, 2, D, dtype=dtype, poison=behind)

    def left(b):  # what has left every row's window, but for the sinks
        behind(b)
        for i, x in enumerate(b.contexts):
            j = torch.arange(3, max(3, x - 29), device=DEV)
            for t in b.cache:
                t[b.table[i].long()[j // b.P], :, j % b.P] = bad
    for news, contexts in (([1], [400]), ([1, 1], [500, 70]), ([9, 70], [100, 300])):
        _check(news, contexts, 4, 2, D, dtype=dtype, window=30, sinks=3, poison=left)

    # in the future of a chunk's rows: those before it do not see it
    n, context, first = 150, 50, 120
    b = R.Batch([n], [context], 2, D, 16, dtype, DEV)
    q = b.normal(n, 4, D).to(dtype)
    for step in (1, 7):
        j = torch.arange(first, n + context, step, device=DEV)
        for t in b.cache:
            t[b.table[0].long()[j // 16], :, j % 16] = bad
        got = paged_attention(q, b.cache, _batch(b), scale=0.1)
        want, bound = R.attend(q, b, 0, 0.1)
        rows = slice(0, first - context)
        assert ((got[rows].double() - want[rows]).abs() <= bound[rows]).all()
    for news, at in ((4, 2), (7, 3)):  # a few rows of one tile
        b = R.Batch([news], [90], 2, D, 16, dtype, DEV)
        q = b.normal(news, 4, D).to(dtype)
        j = 90 + at
        for t in b.cache:
            t[int(b.table[0, j // 16]), :, j % 16] = bad
        got = paged_attention(q, b.cache, _batch(b), scale=0.1)
        want, bound = R.attend(q, b, 0, 0.1)
        assert ((got[:at].double() - want[:at]).abs() <= bound[:at]).all()


@pytest.mark.parametrize("n", [1, 3, 200])
def test_seen_values_that_are_not_finite(n):
    """They reach the elements of every row that sees them, and no other element."""
    b = R.Batch([n], [100], 1, 128, 16, F16, DEV)
    q = b.normal(n, 2, 128).half()
    b.cache[1][int(b.table[0, 2]), 0, 5, 17] = float("inf")
    b.cache[1][int(b.table[0, 2]), 0, 6, 18] = float("nan")
    b.cache[0][int(b.table[0, 2]), 0, 5] *= -40.0  # weight next to none for some rows
    got = paged_attention(q, b.cache, _batch(b), scale=0.1)
    assert not torch.isfinite(got[..., 17]).any() and torch.isnan(got[..., 18]).all()
    rest = torch.ones(128, dtype=torch.bool, device=DEV)
    rest[[17, 18]] = False
    assert torch.isfinite(got[..., rest]).all()
    # only scores of -inf: no answer
    b.cache[0].zero_()
    b.cache[0][..., 0] = -float("inf")
    q[..., 0] = 1.0
    assert torch.isnan(paged_attention(q, b.cache, _batch(b), scale=0.1)).all()


def test_left_out_and_pages_of_zeros():
    """Sequences that pass the host's bounds keep their rows; a page outside the
    cache reads as zeros, keys and values alike."""
    news, contexts = [1, 6, 2, 3, 100], [20, 1, 300, 0, 3]
    b = R.Batch(news, contexts, 2, 64, 16, F16, DEV)
    q = b.normal(b.T, 4, 64).half()
    lengths = b.lengths.clone()
    lengths[3] = 2
    table = b.table.clone()
    table[2, 1], table[2, 4] = -1, 1 << 30
    out = torch.full_like(q, 7.0)
    paged_attention(q, b.cache, PagedBatch(b.starts, lengths, table, 4, 304), scale=0.1, out=out)
    at = b.first
    assert (out[at[1]:at[2]] == 7).all() and (out[at[3]:] == 7).all()  # 6 and 100 new ones, and 3 of 2
    for t in b.cache:
        t[[b.pages[2][1], b.pages[2][4]]] = 0.0
    for i in (0, 2):
        want, bound = R.attend(q[at[i]:at[i + 1]], b, i, 0.1)
        assert ((out[at[i]:at[i + 1]].double() - want).abs() <= bound).all()
    out.fill_(7.0)
    paged_attention(q, b.cache, PagedBatch(b.starts, lengths, table, 100, 200), scale=0.1, out=out)
    assert (out[at[2]:at[3]] == 7).all() and not (out[at[4]:] == 7).any()  # now 302 are too many


def test_caches_past_4_gib():
    """Pages whose bytes lie past 2^32 and 2^33, keys and values."""
    pages, Hkv, P, D = 600000, 2, 64, 64
    cache = [torch.empty(pages, Hkv, P, D, dtype=F16, device=DEV) for _ in range(2)]
    used = [pages - 1, 3, 262144 + 5, 131072, 524288 + 1]
    b = R.Batch([1, 40], [150, 60], Hkv, D, P, F16, DEV)
    small = [t.clone() for t in b.cache]
    table = b.table.clone()
    place = {p: used[n] for n, p in enumerate(b.pages[0] + b.pages[1])}
    for i in range(2):
        for n, p in enumerate(b.pages[i]):
            table[i, n] = place[p]
            for t, s in zip(cache, small):
                t[place[p]] = s[p]
    n, x = b.bounds()
    batch = PagedBatch(b.starts, b.lengths, table, n, x)
    q, k, v = b.normal(b.T, 4, D).half(), b.normal(b.T, Hkv, D).half(), b.normal(b.T, Hkv, D).half()
    paged_store(k, v, cache, batch)
    paged_store(k, v, b.cache, _batch(b))
    for p, at in place.items():
        assert all(torch.equal(t[at], s[p]) for t, s in zip(cache, b.cache))
    assert torch.equal(paged_attention(q, cache, batch, scale=0.1), paged_attention(q, b.cache, _batch(b), scale=0.1))


def test_strides_workspace_and_empty():
    b = R.Batch([1, 30], [5000, 700], 2, 128, 16, F16, DEV)
    q = b.normal(b.T, 8, 128).half()
    batch = _batch(b)
    want = paged_attention(q, b.cache, batch, scale=0.1)
    wide = torch.zeros(b.T, 8, 256, dtype=F16, device=DEV)
    for x in (wide[..., :128], wide[..., 3:131]):  # the second is not 16-byte aligned
        x.copy_(q)
        assert torch.equal(paged_attention(x, b.cache, batch, scale=0.1), want)
    x = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(paged_attention(x, b.cache, batch, scale=0.1), want)
    size = paged_attention_workspace(b.T, 8, 2, 128, batch)
    ws = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(paged_attention(q, b.cache, batch, scale=0.1, workspace=ws), want)
    if size:
        with pytest.raises(RuntimeError, match="workspace"):
            paged_attention(q, b.cache, batch, scale=0.1, workspace=ws[:16])
    assert paged_attention(q[:0], b.cache, batch, scale=0.1).shape == (0, 8, 128)
    assert paged_store(q[:0, :2], q[:0, :2], b.cache, batch) is None


def test_two_streams_and_graphs():
    """Store and attention of a step, captured and replayed with new lengths, pages and tokens; two streams at once."""
    P, D, H, Hkv, S = 16, 128, 8, 2, 5
    b = R.Batch([1] * S, [700, 3, 64, 2000, 15], Hkv, D, P, F16, DEV, spare=8)
    f = rotary_frequencies(D, device=DEV)[0]
    batch = PagedBatch(b.starts, b.lengths, b.table, 1, b.table.shape[1] * P)
    q, k, v = b.normal(S, H, D).half(), b.normal(S, Hkv, D).half(), b.normal(S, Hkv, D).half()
    size = paged_attention_workspace(S, H, Hkv, D, batch)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)

    def step(cache):
        return paged_attention(paged_store(k, v, cache, batch, q=q, rope=Rotary(f)), cache, batch, scale=0.09, workspace=ws)
    mine = [t.clone() for t in b.cache]
    step(mine)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(mine)
    for t, s in zip(mine, b.cache):
        t.copy_(s)
    for n in range(5):
        g.replay()
        want = step(b.cache)
        assert torch.equal(out, want) and all(torch.equal(t, s) for t, s in zip(mine, b.cache))
        b.lengths += 1
        b.lengths[1] += n
        b.lengths.clamp_(max=b.table.shape[1] * P)
        b.table.clamp_(min=0)
        for t in (q, k, v):
            t.normal_()
    both, streams = [], [torch.cuda.Stream() for _ in range(2)]
    works = [(b.normal(S, H, D).half(), torch.empty_like(ws)) for _ in streams]
    want = [paged_attention(x, b.cache, batch, scale=0.09) for x, _ in works]
    torch.cuda.synchronize()
    for _ in range(4):
        both = []
        for (x, w), s in zip(works, streams):
            with torch.cuda.stream(s):
                both.append(paged_attention(x, b.cache, batch, scale=0.09, workspace=w))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(both, want))


def test_python_refusals():
    b = R.Batch([3], [20], 2, 64, 16, F16, DEV)
    batch = _batch(b)
    q, k, v = b.normal(3, 4, 64).half(), b.normal(3, 2, 64).half(), b.normal(3, 2, 64).half()
    f = rotary_frequencies(64, device=DEV)[0]

    def store(k=k, v=v, cache=b.cache, batch=batch, **kw):
        return paged_store(k, v, cache, batch, **kw)

    def attend(q=q, cache=b.cache, batch=batch, **kw):
        return paged_attention(q, cache, batch, **{"scale": 0.1, **kw})
    kc, vc = b.cache
    caches = [(kc, vc[:1]), (kc.float(), vc.float()), (kc, vc.bfloat16()), (kc[:, :, :8].contiguous(), vc[:, :, :8].contiguous()),
              (kc[..., ::2], vc[..., ::2]), (kc[..., :32].contiguous(), vc[..., :32].contiguous()), (kc.cpu(), vc.cpu())]
    for c in caches:
        for f_ in (store, attend):
            with pytest.raises(ValueError):
                f_(cache=c)
    for kw in (dict(k=k[:2]), dict(v=v[:, :1]), dict(k=k.bfloat16()), dict(k=k.cpu()), dict(k=k[0]), dict(q=q[:2]), dict(q=q.float()),
               dict(q=q[..., :32]), dict(q_out=q), dict(q=q, q_out=q.bfloat16()), dict(q=q, q_out=q), dict(rope=Rotary(f.half())),
               dict(rope=Rotary(f[:4])), dict(rope=Rotary(f.repeat(2))), dict(rope=Rotary(f.cpu())), dict(rope=Rotary(f[:0]))):
        with pytest.raises(ValueError):
            store(**kw)
    for kw in (dict(q=q[:, :3]), dict(q=q.bfloat16()), dict(q=q[0]), dict(q=q[..., :32]), dict(window=0), dict(sinks=-1),
               dict(out=q.float()), dict(out=q[:2]), dict(out=q.cpu()), dict(workspace=torch.empty(4, device=DEV)),
               dict(batch=PagedBatch(b.starts, b.lengths, b.table, 3, 1000))):
        with pytest.raises(ValueError):
            attend(**kw)
    for f_, kw in ((store, dict(k=k.clone().requires_grad_())), (attend, dict(q=q.clone().requires_grad_()))):
        with pytest.raises(RuntimeError, match="gradients"):
            f_(**kw)
        with torch.no_grad():
            f_(**kw)
    for bad in ((b.starts.long(), b.lengths, b.table), (b.starts, b.lengths.cpu(), b.table), (b.starts, b.lengths, b.table.long()),
                (b.starts[::1].repeat(2)[::2], b.lengths, b.table)):
        with pytest.raises(ValueError):
            PagedBatch(*bad, 3, 23)
    for n, x in ((0, 23), (3, 0)):
        with pytest.raises(ValueError):
            PagedBatch(b.starts, b.lengths, b.table, n, x)
    with pytest.raises(AttributeError):
        batch.max_length = 7


def test_graphs_that_share_a_workspace():
    """Two captured attentions of different batches in one workspace, replayed in turns
    with eager calls in it between them."""
    P, D, H, Hkv = 16, 128, 8, 2
    shapes = [([1, 1, 1], [3000, 700, 41]), ([200, 1], [2500, 1200])]
    bs = [R.Batch(new, length, Hkv, D, P, F16, DEV) for new, length in shapes]
    batches = [_batch(b) for b in bs]
    qs = [b.normal(b.T, H, D).half() for b in bs]
    ws = torch.empty(max(paged_attention_workspace(b.T, H, Hkv, D, x) for b, x in zip(bs, batches)), dtype=torch.uint8, device=DEV)
    assert ws.numel() > 0

    def attend(i):
        return paged_attention(qs[i], bs[i].cache, batches[i], scale=0.09, workspace=ws)
    attend(0), attend(1)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in bs], []
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            outs.append(attend(i))
    for n in range(4):
        for i, g in enumerate(graphs):
            qs[i].normal_()
            outs[i].zero_()
            g.replay()
            attend(1 - i)
        for i in range(2):
            assert torch.equal(outs[i], paged_attention(qs[i], bs[i].cache, batches[i], scale=0.09)), (n, i)


def test_output_over_its_queries():
    b = R.Batch([3], [20], 2, 64, 16, F16, DEV)
    q = b.normal(b.T, 4, 64).half()
    with pytest.raises(ValueError, match="must not be q"):
        paged_attention(q, b.cache, _batch(b), scale=0.1, out=q)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("spans", [2, 5, 16, 17, 18, 19, 20, 21, 31, 32, 33, 34, 35, 48, 49, 63, 64])
def test_every_number_of_spans(D, spans):
    """Chunks whose keys are split into so many spans of 8 tiles of 64, the last of 7 tiles: none is lost in the
    merge, whatever rest the number leaves by the spans that it takes at once."""
    L = 64 * (8 * spans - 1)
    for n, H, dtype, window in ((33, 1, F16, None), (9, 4, BF16, None), (128, 1, F16, L - 40)):
        # one sequence and key/value head, more rows than the kernel for few takes: the workspace tells the spans
        b = R.Batch([n], [L - n], 1, D, 16, dtype, DEV)
        rows = paged_attention_workspace(n, H, 1, D, _batch(b)) // (n * H * (D + 2) * 4)
        assert rows == spans
        _check([n], [L - n], H, 1, D, dtype=dtype, window=window, seed=spans)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("news,contexts,H,Hkv", [([1], [1], 4, 4), ([1], [4], 4, 1), ([1, 1, 1], [12, 30, 39], 8, 2), ([5], [3], 6, 2),
                                                 ([3, 2], [20, 9], 8, 1), ([1, 1], [700, 90], 8, 1), ([40, 1, 3], [5, 17, 9], 4, 2)])
def test_steps_lose_no_bits_of_their_numerators(D, dtype, news, contexts, H, Hkv):
    """Sequences of up to 32 rows hold a numerator as two numbers of the type: h^2 of it is lost where the bound
    of ``attend`` has h, and the rest of that bound stays.  Few keys, small scores: the output's own rounding and
    the scores' leave room for no more."""
    b = R.Batch(news, contexts, Hkv, D, 16, dtype, DEV, seed=11)
    q = b.normal(b.T, H, D).to(dtype)
    scale = 0.25 * D ** -0.5
    out = paged_attention(q, b.cache, _batch(b), scale=scale)
    v = b.cache[1]
    h = R.HALF[dtype]
    for i in range(len(news)):
        if news[i] * H // Hkv > 32:
            continue
        rows = q[b.first[i]:b.first[i + 1]]
        b.cache[1] = v
        want, bound = R.attend(rows, b, i, scale)
        b.cache[1] = v.abs()
        size, _ = R.attend(rows, b, i, scale)
        tight = bound - 1.01 * (h - h * h) * (size + want.abs())
        off = (out[b.first[i]:b.first[i + 1]].double() - want).abs()
        assert (tight > 0).all() and (off <= tight).all(), (i, (off / tight).max())


@pytest.mark.parametrize("n", [1, 3, 200])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("key", [0, 101])
def test_seen_infinities_keep_their_signs(n, dtype, key):
    """With weights above zero an infinity among the values is what the row answers there, whichever tile it is in:
    101 lies in one that the mask cuts for n = 3 and 200."""
    b = R.Batch([n], [101], 1, 64, 16, dtype, DEV)
    q = b.normal(n, 2, 64).to(dtype)
    page, slot = int(b.table[0, key // 16]), key % 16
    b.cache[1][page, 0, slot, 5] = float("inf")
    b.cache[1][page, 0, slot, 40] = -float("inf")
    got = paged_attention(q, b.cache, _batch(b), scale=0.1)
    assert (got[..., 5] == float("inf")).all() and (got[..., 40] == -float("inf")).all()
    got[..., [5, 40]] = 0.0
    assert torch.isfinite(got).all()


def test_one_row_of_an_odd_pitch():
    """A single row, or a single head, keeps the pitch of the buffer that it is a view of, whatever torch calls it:
    answered as any other strides are."""
    b = R.Batch([1], [50], 1, 128, 16, F16, DEV)
    wide = b.normal(2, 4 * 128 + 7).half()
    one = torch.as_strided(b.normal(128).half(), (1, 1, 128), (3, 5, 1))
    for q in (wide[:1, :512].view(1, 4, 128), one):
        assert q.is_contiguous() and any(s % 8 for s in q.stride())
        want = paged_attention(q.clone(memory_format=torch.contiguous_format), b.cache, _batch(b), scale=0.1)
        assert torch.equal(paged_attention(q, b.cache, _batch(b), scale=0.1), want)
        paged_store(q[:, :1], q[:, :1], b.cache, _batch(b), q=q)
