"""A paged batch, rotary positions and attention over pages in 64 bits, one
sequence at a time."""
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step of rounding


class Batch:
    """Sequences of ``news`` new tokens after ``contexts`` positions, their pages
    in random order in a cache of [pages, Hkv, P, D] (keys and values normal)."""

    def __init__(self, news, contexts, Hkv, D, P=16, dtype=torch.float16, dev="cpu", seed=0, spare=2, before=0, after=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.news, self.contexts, self.P, self.dev, self.g = news, contexts, P, dev, g
        self.len = [n + c for n, c in zip(news, contexts)]
        counts = [(x + P - 1) // P for x in self.len]
        pages = sum(counts) + spare
        order = torch.randperm(pages, generator=g, device=dev).tolist()
        W = max(1, max(counts))
        # entries behind a sequence's pages are never looked at
        self.table = torch.full((len(news), W), -7, dtype=torch.int32)
        self.pages = []
        for i, n in enumerate(counts):
            self.pages.append(order[:n])
            self.table[i, :n] = torch.tensor(order[:n], dtype=torch.int32)
            order = order[n:]
        self.table = self.table.to(dev)
        self.first = [before]
        for n in news:
            self.first.append(self.first[-1] + n)
        self.T = self.first[-1] + after
        self.starts = torch.tensor(self.first, dtype=torch.int32, device=dev)
        self.lengths = torch.tensor(self.len, dtype=torch.int32, device=dev)
        self.cache = [self.normal(pages, Hkv, P, D).to(dtype) for _ in range(2)]

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device=self.dev)

    def bounds(self):
        return max(1, max(self.news)), max(1, max(self.len))

    def positions(self, i):
        return torch.arange(self.contexts[i], self.len[i], device=self.dev)

    def held(self, which, i):
        """Keys (0) or values (1) [Hkv, length, D] of sequence i."""
        x = self.cache[which][self.pages[i]].transpose(0, 1)
        return x.reshape(x.shape[0], -1, x.shape[-1])[:, :self.len[i]]


def turn(x, positions, frequencies, interleaved, factor):
    """x [n, heads, D] turned, and the size of the terms (for bounds), in 64 bits."""
    x = x.double().clone()
    size = x.abs()
    if frequencies is None:
        return x, torch.zeros_like(size)
    n = frequencies.numel()
    a = (positions.double()[:, None] * frequencies.double())[:, None]
    i = torch.arange(n, device=x.device)
    p, r = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    u, w = x[..., p].clone(), x[..., r].clone()
    x[..., p], x[..., r] = factor * (u * a.cos() - w * a.sin()), factor * (w * a.cos() + u * a.sin())
    both = (u.abs() + w.abs()) * abs(factor)
    size[...] = 0.0
    size[..., p], size[..., r] = both, both
    return x, size


def attend(q, b, i, scale, window=None, sinks=0):
    """Output [n, H, D] of sequence i's rows and its error bound.  Values that a
    row does not see count as zero whatever they are.

    Numerators are rounded to the data's type (h = half a step) and their sum is that
    of the rounded ones: |error| <= h sum w |v - out|, second order in a factor
    of 1.01; fp16 numerators below 2^-14 are off by 2^-25 of a largest of at least 1.
    Scores in f32: D + 2 roundings of the terms' size and one of the largest score's
    (both maxima are below the size), the exponential 2^-21; sums in f32, at
    most 16 terms of a product and then one addition per 16 keys, and one more per part.
    The output's own rounding is h |out|."""
    n, H, D = q.shape
    k, v = b.held(0, i).double(), b.held(1, i).double()
    Hkv, L, _ = k.shape
    h = HALF[b.cache[0].dtype]
    k, v = k.repeat_interleave(H // Hkv, 0), v.repeat_interleave(H // Hkv, 0)
    p, j = b.positions(i)[:, None], torch.arange(L, device=q.device)[None]
    sees = (j <= p) & ((p - j < (window or L + 1)) | (j < sinks))
    q = q.double().transpose(0, 1)
    k0, v0 = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
    s = (q @ k0.transpose(1, 2).contiguous() * scale).masked_fill(~sees, -float("inf"))
    w = torch.softmax(s, -1)
    want, size = w @ v0, w @ v0.abs()
    terms = (q.abs() @ k0.abs().transpose(1, 2).contiguous() * abs(scale)).masked_fill(~sees, 0.0).amax(-1, keepdim=True)
    rel = torch.expm1(2.0 * (D + 4) * 2.0 ** -24 * terms) + 2.0 ** -21 + (L / 16 + 64) * 2.0 ** -24
    bound = 1.01 * (rel + h) * (size + want.abs()) + h * want.abs() + 2.0 ** -24
    bound = bound + 2.0 ** -24 * (sees.double() @ v0.abs() + sees.double().sum(-1)[None, :, None] * want.abs())
    return want.transpose(0, 1), bound.transpose(0, 1)
