"""Sampling, the 4-bit cache, the window's step and window attention on streams
other than the default one, two at once, and in graphs that share a workspace one
after the other."""
import pytest
import torch

from atlasinfer_amd.integration.sampling import sample_tokens
from atlasinfer_amd.integration.window_attention import window_attention
from atlasinfer_amd.memory import decode_cache as DC

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _rnd(g, *s):
    return torch.randn(*s, generator=g, device=DEV).half()


class Work:
    """One of everything, with its own inputs; run() gives its outputs."""

    def __init__(self, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        B, H, Hkv, D, slots = 3, 8, 2, 128, 2100
        self.logits, self.u = torch.randn(4, 50000, generator=g, device=DEV), torch.rand(4, generator=g, device=DEV)
        self.caches = [DC.DecodeCache(B, Hkv, slots, D, bits=b, sinks=4, device=DEV) for b in (4, 16)]
        self.k, self.v = _rnd(g, B, Hkv, 2000, D), _rnd(g, B, Hkv, 2000, D)
        self.q, self.kn, self.vn = _rnd(g, B, H, D), _rnd(g, B, Hkv, D), _rnd(g, B, Hkv, D)
        self.pos = torch.tensor([2000, 1500, 3], device=DEV)
        self.pq = _rnd(g, B, H, 2000, D)
        self.ws = [torch.empty(max(16, c.workspace_bytes(H)), dtype=torch.uint8, device=DEV) for c in self.caches]

    def run(self):
        out = [sample_tokens(self.logits, self.u, top_p=0.9), sample_tokens(self.logits, self.u, 0.7, 40)]
        for c, ws in zip(self.caches, self.ws):
            c.store(self.k, self.v)
            out.append(c.attend(self.q, self.kn, self.vn, self.pos, scale=0.09, workspace=ws))
        return out + [window_attention(self.pq, self.k, self.v, window=300, sinks=4)]


def test_two_streams_at_once():
    works = [Work(1), Work(2)]
    want = [w.run() for w in works]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in works]
    for _ in range(5):
        got = []
        for w, s in zip(works, streams):
            with torch.cuda.stream(s):
                got.append(w.run())
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_graphs_that_share_a_workspace():
    """Replayed one after the other on a stream; what one leaves there the other
    does not read."""
    works = [Work(3), Work(4)]
    works[1].ws = works[0].ws
    want = [w.run() for w in works]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for w in works:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(w.run())
        graphs.append(g)
    for _ in range(4):
        for i in (0, 1):
            for o in outs[i]:
                o.zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want[i], outs[i]))
        sum(w.logits.sum() for w in works).item()  # eager work between the replays
