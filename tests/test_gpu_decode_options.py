"""GraphDecoder's options on the GPU: a sliding window with sinks, the 4-bit
cache and sampling -- captured steps against eager ones bit for bit, and against
HF's own forward with the same attention written out."""
import pytest
import torch

import kv4_ref as R
from atlasinfer_amd.integration.decode_graph import GraphDecoder
from atlasinfer_amd.integration.sampling import sample_tokens
from atlasinfer_amd.integration.window_attention import window_prompts
from integration import model_modifier as MM

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _model(kind, seed=0, quantize=True, **more):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(seed)
    if kind == "opt":
        cfg = transformers.OPTConfig(vocab_size=512, hidden_size=256, ffn_dim=512, num_hidden_layers=2,
                                     num_attention_heads=4, max_position_embeddings=256, word_embed_proj_dim=256)
        m = transformers.OPTForCausalLM(cfg)
    else:
        cls, mod = ((transformers.LlamaConfig, transformers.LlamaForCausalLM) if kind == "llama"
                    else (transformers.MistralConfig, transformers.MistralForCausalLM))
        cfg = cls(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                  num_key_value_heads=2, max_position_embeddings=256, **more)
        m = mod(cfg)
    m = m.half().to(DEV).eval()
    if quantize:
        MM.apply_atlas_quantization_to_model(m, kind, {"block_size": -1}, excluded_layers=["embed_tokens",
                                                                                          "embed_positions"])
    return m


def _reference_attention(window, sinks, quantize):
    """HF attention interface in f32: window and sinks, and for steps (one query)
    keys and values as the 4-bit cache holds them."""
    def back(t):
        c, s, m = R.quantize(t.cpu())
        return R.values(c, s, m).float().to(t.device)

    def attend(module, q, k, v, attention_mask, scaling=None, dropout=0.0, **kw):
        M, N, G = q.shape[2], k.shape[2], q.shape[1] // k.shape[1]
        kf, vf = (back(k), back(v)) if quantize and M == 1 else (k.float(), v.float())
        s = q.float() @ kf.repeat_interleave(G, 1).transpose(2, 3).contiguous() * scaling
        i, j = torch.arange(N - M, N, device=q.device)[:, None], torch.arange(N, device=q.device)[None]
        sees = j <= i if window is None else (j <= i) & ((i - j < window) | (j < sinks))
        o = torch.softmax(s.masked_fill(~sees, -float("inf")), -1) @ vf.repeat_interleave(G, 1)
        return o.half().transpose(1, 2).contiguous(), None
    return attend


@pytest.mark.parametrize("kind", ["opt", "llama"])
@pytest.mark.parametrize("batch", [1, 3, 8])
@pytest.mark.parametrize("window,sinks,kv_bits", [(None, 0, 4), (16, 0, 16), (12, 4, 16), (12, 3, 4)])
def test_steps_follow_hf_with_the_same_attention(kind, batch, window, sinks, kv_bits):
    """Teacher-forced: fed HF's tokens, every step's logits lie within 2e-2 of
    the largest of HF's (the bound of the plain decoder's test: the linears round
    in another order), past the window's edge."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface
    m = _model(kind, 2)
    S, n = 20, 24
    ids = torch.randint(0, 512, (batch, S), device=DEV)
    name = f"ref_{window}_{sinks}_{kv_bits}"
    AttentionInterface.register(name, _reference_attention(window, sinks, kv_bits == 4))
    AttentionMaskInterface.register(name, lambda *a, **k: None)
    before = m.config._attn_implementation
    m.set_attn_implementation(name)
    with torch.no_grad():
        ref = m.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=n, do_sample=False,
                         return_dict_in_generate=True, output_logits=True)
    m.set_attn_implementation(before)
    gd = GraphDecoder(m, batch=batch, max_len=64, window=window, sinks=sinks, kv_bits=kv_bits)
    gd.prefill(ids)
    assert m.config._attn_implementation == before
    for t in range(1, n):
        gd.tok.copy_(ref.sequences[:, S + t - 1])
        got, want = gd.step().float(), ref.logits[t].float()
        assert ((got - want).abs().amax(-1) <= 2e-2 * want.abs().amax(-1)).all(), t


@pytest.mark.parametrize("kind,batch", [("opt", 1), ("llama", 1), ("llama", 5), ("llama", 8)])
@pytest.mark.parametrize("options", [dict(kv_bits=4), dict(window=10, sinks=2), dict(window=10, sinks=2, kv_bits=4),
                                     dict(sampling=True), dict(sampling=True, kv_bits=4, window=20)])
def test_replays_are_the_eager_steps(kind, batch, options):
    m = _model(kind, 1)
    ids = torch.randint(0, 512, (batch, 9), device=DEV)
    g, e = GraphDecoder(m, batch, 60, **options), GraphDecoder(m, batch, 60, graph=False, **options)
    for seq in range(2):
        if "sampling" in options:
            for d in (g, e):
                d.set_sampling(temperature=0.5 + seq, top_k=[3, 0][seq], top_p=0.9,
                               generator=torch.Generator(device=DEV).manual_seed(seq))
        assert torch.equal(g.prefill(ids), e.prefill(ids))
        for t in range(30):
            lg = g.step().clone()
            assert torch.equal(lg, e.step()), t
            assert torch.equal(g.tok, e.tok), t
        torch.cuda.synchronize()
        assert torch.equal(g.out, e.out)


def test_sampled_tokens_are_those_of_the_logits():
    m = _model("llama", 3)
    ids = torch.randint(0, 512, (4, 7), device=DEV)
    gd = GraphDecoder(m, 4, 50, sampling=True)
    gd.set_sampling(temperature=[0.0, 0.7, 1.0, 2.0], top_k=[0, 5, 0, 50], top_p=[1.0, 1.0, 0.8, 0.95], min_p=0.001)
    gd.prefill(ids)
    for t in range(1, 20):
        lg = gd.step()
        want = sample_tokens(lg, gd.u[t], gd.settings["temperature"], gd.settings["top_k"], gd.settings["top_p"],
                             gd.settings["min_p"])
        assert torch.equal(gd.tok, want) and torch.equal(gd.out[:, t], want)
        assert gd.tok[0] == lg[0].float().argmax()
    # temperature 0 is the greedy decoder; equal generators give equal tokens, others others
    greedy = GraphDecoder(m, 4, 50).generate(ids, 12)
    assert torch.equal(gd.generate(ids, 12, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0), greedy)
    run = lambda s: gd.generate(ids, 30, temperature=1.5, generator=torch.Generator().manual_seed(s))  # noqa: E731
    assert torch.equal(run(1), run(1)) and not torch.equal(run(1), run(2))
    assert torch.equal(gd.settings["temperature"], torch.full((4,), 1.5, device=DEV))


def test_a_configured_window_is_taken():
    """A Mistral whose configuration has a window shorter than max_len decodes as
    HF's own sliding cache does; the cache holds the window alone."""
    m = _model("mistral", 4, sliding_window=12)
    ids = torch.randint(0, 512, (2, 30), device=DEV)
    with torch.no_grad():
        ref = m.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=20, do_sample=False,
                         return_dict_in_generate=True, output_logits=True)
    gd = GraphDecoder(m, 2, 64)
    assert gd.window == 12 and gd.caches[0].slots == 12
    gd.prefill(ids)
    for t in range(1, 20):
        gd.tok.copy_(ref.sequences[:, 30 + t - 1])
        got, want = gd.step().float(), ref.logits[t].float()
        assert ((got - want).abs().amax(-1) <= 2e-2 * want.abs().amax(-1)).all(), t
    assert GraphDecoder(m, 2, 12).window is None  # it reaches back to the first position


def test_cache_sizes_and_refusals():
    m = _model("llama", 5, quantize=False)
    full = GraphDecoder(m, 2, 200)
    four = GraphDecoder(m, 2, 200, kv_bits=4)
    held = sum(t.numel() * 2 for t in full.k + full.v)
    # 5 bits for 16, slots in blocks of 32
    assert sum(c.nbytes() for c in four.caches) * 16 == held // 200 * 224 * 5
    for kw in (dict(kv_bits=8), dict(window=0), dict(window=5, sinks=-1), dict(sinks=4)):
        with pytest.raises(ValueError):
            GraphDecoder(m, 2, 64, **kw)
    with pytest.raises(NotImplementedError):
        GraphDecoder(m.float(), 2, 64, kv_bits=4)
    m.half()
    with pytest.raises(ValueError):
        full.generate(torch.randint(0, 512, (2, 5), device=DEV), 5, temperature=0.5)
    with pytest.raises(RuntimeError):  # an exception inside leaves the model as it was
        with window_prompts(m, 8):
            raise RuntimeError
    assert m.config._attn_implementation == "sdpa"


def test_every_prompt_draws_its_numbers():
    """set_sampling's numbers serve the prompt that follows; prompts without it, and
    the first one, draw their own, from the last generator."""
    gd = GraphDecoder(_model("llama"), batch=2, max_len=24, sampling=True)
    ids = torch.randint(0, 512, (2, 5), device=DEV)
    gd.prefill(ids)
    one = gd.u.clone()
    assert one.min() >= 0 and one.max() < 1 and one.unique().numel() > 40
    gd.step()
    gd.set_sampling(temperature=1.2, generator=torch.Generator().manual_seed(3))
    two = gd.u.clone()
    assert torch.equal(two.cpu(), torch.rand(24, 2, generator=torch.Generator().manual_seed(3)))
    gd.step()  # takes them, so that the next prompt may not
    g = torch.Generator().manual_seed(3)
    torch.rand(24, 2, generator=g)
    gd.prefill(ids)
    assert torch.equal(gd.u.cpu(), torch.rand(24, 2, generator=g))
    gd.set_sampling(generator=torch.Generator().manual_seed(4))
    three = gd.u.clone()
    gd.prefill(ids)
    assert torch.equal(gd.u, three)
    gd.prefill(ids)
    assert not torch.equal(gd.u, three)


@pytest.mark.parametrize("options", [dict(window=64), dict(window=100, sinks=2), dict(sinks=52), dict(window=40, sinks=24),
                                     dict(window=64, kv_bits=4)])
def test_a_window_that_reaches_max_len_replaces_the_configured_one(options):
    """A Mistral with a configured window, decoded with one that reaches back to the
    first position: the prompt, longer than the configured window, sees every position
    before it as the steps do."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface
    m = _model("mistral", 4, sliding_window=12)
    ids = torch.randint(0, 512, (2, 30), device=DEV)
    four = options.get("kv_bits") == 4
    name = f"ref_whole_{four}"
    AttentionInterface.register(name, _reference_attention(None, 0, four))
    AttentionMaskInterface.register(name, lambda *a, **k: None)
    before = m.config._attn_implementation
    m.config.sliding_window = None  # HF's cache would keep the window alone
    m.set_attn_implementation(name)
    with torch.no_grad():
        ref = m.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=20, do_sample=False,
                         return_dict_in_generate=True, output_logits=True)
    m.set_attn_implementation(before)
    m.config.sliding_window = 12
    gd = GraphDecoder(m, 2, 64, **options)
    assert gd.window is None
    gd.prefill(ids)
    assert m.config._attn_implementation == before
    for t in range(1, 20):
        gd.tok.copy_(ref.sequences[:, 30 + t - 1])
        got, want = gd.step().float(), ref.logits[t].float()
        assert ((got - want).abs().amax(-1) <= 2e-2 * want.abs().amax(-1)).all(), t


def test_generate_keeps_the_generator():
    """A generator given once serves every generate that names no other."""
    gd = GraphDecoder(_model("llama"), batch=2, max_len=24, sampling=True)
    ids = torch.randint(0, 512, (2, 5), device=DEV)
    gd.set_sampling(temperature=1.3, generator=torch.Generator().manual_seed(7))
    g = torch.Generator().manual_seed(7)
    torch.rand(24, 2, generator=g)
    for kw in ({}, dict(top_k=9), {}):
        gd.generate(ids, 6, **kw)
        assert torch.equal(gd.u.cpu(), torch.rand(24, 2, generator=g)), kw
    gd.generate(ids, 6, generator=torch.Generator().manual_seed(8))
    assert torch.equal(gd.u.cpu(), torch.rand(24, 2, generator=torch.Generator().manual_seed(8)))
    gd.generate(ids, 6, generator=None)  # back to torch's default one
    assert not torch.equal(gd.u.cpu(), torch.rand(24, 2, generator=g))
    a = gd.u.clone()
    gd.generate(ids, 6)
    assert not torch.equal(gd.u, a)
