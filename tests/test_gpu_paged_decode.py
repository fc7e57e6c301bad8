"""GraphDecoder over a paged cache: prompts of different lengths in one batch,
chunks, windows, log probabilities of the chosen tokens and of given texts --
against HF's own forward of each sequence alone, and replays against eager steps."""
import pytest
import torch

from atlasinfer_amd.integration.decode_graph import GraphDecoder
from test_gpu_decode_options import _model

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _prompts(lengths, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randint(0, 512, (n,), generator=g, device=DEV) for n in lengths]


def _close(got, want):
    """Within 2e-2 of the row's largest logit (the bound of the plain decoder's
    tests: the linears round in another order)."""
    assert ((got.float() - want.float()).abs().amax(-1) <= 2e-2 * want.float().abs().amax(-1)).all()


@pytest.mark.parametrize("kind", ["opt", "llama"])
@pytest.mark.parametrize("lengths,options", [
    ([20], {}), ([5, 33, 1], {}), ([40, 2, 17, 8, 31, 1, 64, 3], dict(chunk=23)), ([9, 50], dict(page_size=64, chunk=7)),
    ([30, 3, 12], dict(window=16)), ([1, 45], dict(window=12, sinks=4, chunk=10))])
def test_steps_follow_hf(kind, lengths, options):
    """Teacher-forced with HF's tokens of each prompt alone."""
    m = _model(kind, 2)
    n = 20
    prompts = _prompts(lengths)
    window, sinks = options.get("window"), options.get("sinks", 0)
    refs = []
    for p in prompts:
        with torch.no_grad():
            if window is None:
                refs.append(m.generate(p[None], attention_mask=torch.ones_like(p[None]), max_new_tokens=n, do_sample=False,
                                       return_dict_in_generate=True, output_logits=True))
            else:  # the plain decoder's window, which has tests of its own
                refs.append(GraphDecoder(m, 1, 100, window=window, sinks=sinks))
    gd = GraphDecoder(m, len(prompts), 100, **{"page_size": 16, **options})
    first = gd.prefill(prompts)
    if window is None:
        assert all(int(f) == int(r.sequences[0, len(p)]) for f, r, p in zip(first, refs, prompts))
        for t in range(1, n):
            gd.tok.copy_(torch.stack([r.sequences[0, len(p) + t - 1] for r, p in zip(refs, prompts)]))
            _close(gd.step(), torch.cat([r.logits[t] for r in refs]))
    else:
        assert torch.equal(first, torch.cat([r.prefill(p[None]) for r, p in zip(refs, prompts)]))
        for t in range(1, n):
            for i, r in enumerate(refs):
                gd.tok[i] = r.tok[0]
            _close(gd.step(), torch.cat([r.step() for r in refs]))


@pytest.mark.parametrize("kind,lengths", [("opt", [7]), ("llama", [4, 9, 30]), ("llama", [3, 1, 20, 6, 8, 11, 2, 40])])
@pytest.mark.parametrize("options", [{}, dict(sampling=True, logprobs=4), dict(window=14, sinks=2, logprobs=0)])
def test_replays_are_the_eager_steps(kind, lengths, options):
    m = _model(kind, 1)
    B = len(lengths)
    g, e = (GraphDecoder(m, B, 90, graph=x, page_size=16, **options) for x in (True, False))
    for seq in range(2):
        prompts = _prompts(lengths[::-1] if seq else lengths, seq)
        if "sampling" in options:
            for d in (g, e):
                d.set_sampling(temperature=0.5 + seq, top_p=0.9, generator=torch.Generator(device=DEV).manual_seed(seq))
        assert torch.equal(g.prefill(prompts), e.prefill(prompts))
        for t in range(40):
            lg = g.step().clone()
            assert torch.equal(lg, e.step()), t
            assert torch.equal(g.tok, e.tok), t
        assert torch.equal(g.out, e.out)
        if "logprobs" in options:
            assert all(torch.equal(a, b) for a, b in zip(g.chosen, e.chosen))


def test_generate_takes_both_forms():
    """Equal prompts as a matrix and as a list; the paged cache gives the plain one's tokens where logits are apart."""
    m = _model("llama", 3)
    gd = GraphDecoder(m, 3, 80, page_size=16)
    ids = torch.stack(_prompts([12, 12, 12]))
    a, b = gd.generate(ids, 20), gd.generate(list(ids), 20)
    assert a.shape == (3, 32) and isinstance(b, list) and torch.equal(a, torch.stack(b))
    plain = GraphDecoder(m, 3, 80).generate(ids, 20)
    assert torch.equal(a[:, :13], plain[:, :13])
    out = gd.generate(_prompts([3, 40, 1]), 5)
    assert [len(t) for t in out] == [8, 45, 6]


@pytest.mark.parametrize("paged", [False, True])
def test_chosen_tokens_logprobs(paged):
    m = _model("llama", 4)
    gd = GraphDecoder(m, 3, 50, logprobs=6, sampling=True, **(dict(page_size=16) if paged else {}))
    gd.set_sampling(temperature=[0.0, 1.0, 1.5])
    gd.prefill(torch.stack(_prompts([8, 8, 8])))
    for t in range(1, 15):
        lp = torch.log_softmax(gd.step().double(), -1)
        want = lp.gather(1, gd.tok[:, None])[:, 0]
        assert ((gd.chosen.logprobs[:, t] - want).abs() <= 1e-4).all()
        assert ((gd.chosen.entropies[:, t] + (lp.exp() * lp).sum(-1)).abs() <= 1e-4).all()
        assert torch.equal(gd.chosen.ranks[:, t], (lp > want[:, None]).sum(1))
        top = torch.sort(lp, dim=1, descending=True, stable=True)
        assert torch.equal(gd.chosen.top_tokens[:, t], top.indices[:, :6])
        assert ((gd.chosen.top_logprobs[:, t] - top.values[:, :6]).abs() <= 1e-4).all()
    assert gd.chosen.ranks[0, 1:15].eq(0).all()


@pytest.mark.parametrize("kind", ["opt", "llama"])
@pytest.mark.parametrize("chunk", [2048, 13])
def test_score(kind, chunk):
    """More texts than the batch, of one token too, against HF's logits of each alone."""
    m = _model(kind, 5)
    texts = _prompts([30, 1, 2, 75, 17, 44, 16])
    gd = GraphDecoder(m, 3, 80, page_size=16, chunk=chunk)
    got = gd.score(texts, top=5)
    assert len(got) == len(texts)
    for text, s in zip(texts, got):
        assert s.logprobs.shape == s.ranks.shape == (len(text) - 1,) and s.top_tokens.shape == (len(text) - 1, 5)
        if len(text) == 1:
            continue
        with torch.no_grad():
            x = m(text[None]).logits[0, :-1].float()
        want = torch.log_softmax(x.double(), -1)
        # logits within 2e-2 of their row's largest: a log probability within twice that
        bound = 4e-2 * x.abs().amax(-1)
        assert ((s.logprobs - want.gather(1, text[1:, None])[:, 0]).abs() <= bound).all()
        assert ((s.top_logprobs - torch.topk(want, 5).values).abs() <= bound[:, None]).all()
    again = gd.score(texts[:2], top=5)
    assert all(torch.equal(a, b) for x, y in zip(again, gd.score(texts[:2], top=5)) for a, b in zip(x, y))
    with pytest.raises(RuntimeError):
        gd.step()
    gd.generate(texts[:3], 4)  # and decoding goes on as ever


def test_pool_of_pages():
    """A pool smaller than batch times max_len serves prompts that fit; what does not is refused, and the decoder
    lives on."""
    m = _model("llama", 6)
    big = GraphDecoder(m, 3, 96, page_size=16)
    small = GraphDecoder(m, 3, 96, page_size=16, pages=8)
    prompts = _prompts([60, 3, 20])  # 4 + 1 + 2 pages, steps in them up to 61 .. 64
    want = big.generate(prompts, 4)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(small.generate(prompts, 4), want))
    with pytest.raises(RuntimeError, match="pages"):
        small.prefill(_prompts([60, 60, 60]))
    with pytest.raises(RuntimeError):
        small.step()
    small.prefill(prompts)
    with pytest.raises(RuntimeError, match="pages"):
        for _ in range(40):
            small.step()
    assert all(torch.equal(a, b) for a, b in zip(small.generate(prompts, 4), want))


def test_refusals():
    m = _model("llama", 7, quantize=False)
    for bad, error in ((dict(pages=4), ValueError), (dict(page_size=24), ValueError), (dict(page_size=16, kv_bits=4), ValueError),
                       (dict(page_size=16, chunk=0), ValueError), (dict(logprobs=65), ValueError), (dict(logprobs=-1), ValueError)):
        with pytest.raises(error):
            GraphDecoder(m, 2, 64, **bad)
    with pytest.raises(NotImplementedError):
        GraphDecoder(m, 2, 64).score(_prompts([4, 5]))
    with pytest.raises(ValueError):
        GraphDecoder(m, 2, 64).generate(_prompts([4, 5]), 3)
    gd = GraphDecoder(m, 2, 64, page_size=16)
    for prompts in (_prompts([4]), _prompts([4, 64]), _prompts([4, 0])):
        with pytest.raises(ValueError):
            gd.prefill(prompts)
    with pytest.raises(NotImplementedError):
        GraphDecoder(m.float(), 2, 64, page_size=16)


def test_positions_past_a_table():
    """A decoder that would pass the learned positions' table is refused, one that just reaches its end runs."""
    m = _model("opt", 3, quantize=False)
    known = m.config.max_position_embeddings
    with pytest.raises(ValueError, match="positions"):
        GraphDecoder(m, 1, known + 1, page_size=16)
    gd = GraphDecoder(m, 1, known, page_size=16)
    got, = gd.score(_prompts([known]))
    assert torch.isfinite(got.logprobs).all() and got.logprobs.shape == (known - 1,)


def test_a_pool_of_the_final_need():
    """Prompts of uneven lengths end with every page of the pool: pages held ahead by one serve the other."""
    m = _model("llama", 9)
    prompts = _prompts([16, 8])
    want = GraphDecoder(m, 2, 96, page_size=16).generate(prompts, 17)  # 32 and 24 positions in the cache
    tight = GraphDecoder(m, 2, 96, page_size=16, pages=4)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(tight.generate(prompts, 17), want))
    with pytest.raises(RuntimeError, match="pages"):
        tight.step()


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("paged", [False, True])
def test_chosen_holds_one_text(graph, paged):
    """A short text after a longer one, and the first after the steps that come before a capture: nothing of
    another stands behind its tokens."""
    m = _model("llama", 4)
    gd = GraphDecoder(m, 2, 50, graph=graph, logprobs=3, **(dict(page_size=16) if paged else {}))
    for n in (1, 20, 4):
        gd.generate(torch.stack(_prompts([6, 6], n)), n)
        assert (gd.chosen.logprobs[:, :n] < 0).all() and (gd.chosen.entropies[:, :n] > 0).all()
        assert (gd.chosen.top_logprobs[:, :n] < 0).all()
        for t in gd.chosen + (gd.out,):
            assert (t[:, n:] == 0).all()
