"""GraphDecoder's decode step on the CPU (eager, no capture): with plain
fp32 OPT, Llama and Mistral models it must generate what HF's own generate
generates, token for token, with the same logits at every step.  This checks
the step's indexing (cache slot, positional embedding and rotary rows at
the device-side position, the causal mask, the output slot) before any
graph is captured on the GPU."""
import pytest
import torch

from atlasinfer_amd.integration.decode_graph import GraphDecoder

transformers = pytest.importorskip("transformers")


def _model(kind):
    torch.manual_seed(0)
    if kind == "opt":
        cfg = transformers.OPTConfig(vocab_size=256, hidden_size=128, ffn_dim=256, num_hidden_layers=2,
                                     num_attention_heads=4, max_position_embeddings=128, word_embed_proj_dim=128)
        return transformers.OPTForCausalLM(cfg).eval()
    cls = transformers.LlamaConfig if kind == "llama" else transformers.MistralConfig
    cfg = cls(vocab_size=256, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
              num_key_value_heads=2, max_position_embeddings=128)
    model_cls = transformers.LlamaForCausalLM if kind == "llama" else transformers.MistralForCausalLM
    return model_cls(cfg).eval()


@pytest.mark.parametrize("kind", ["opt", "llama", "mistral"])
def test_eager_step_matches_hf_generate(kind):
    m = _model(kind)
    ids = torch.randint(0, 256, (2, 7))
    with torch.no_grad():
        ref = m.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=10, do_sample=False,
                         return_dict_in_generate=True, output_logits=True)
    gd = GraphDecoder(m, batch=2, max_len=32, graph=False)
    first = gd.prefill(ids)
    assert torch.equal(first, ref.sequences[:, 7])
    for t in range(9):
        lg = gd.step()
        rel = ((lg - ref.logits[t + 1]).abs().max() / ref.logits[t + 1].abs().max()).item()
        assert rel < 1e-5, (t, rel)
    assert torch.equal(gd.generate(ids, 10), ref.sequences)


def test_cache_bound_is_enforced():
    gd = GraphDecoder(_model("opt"), batch=1, max_len=10, graph=False)
    ids = torch.randint(0, 256, (1, 6))
    with pytest.raises(ValueError):
        gd.generate(ids, 5)  # 6 + 5 positions > 10
    gd.prefill(ids)
    for _ in range(4):  # positions 6..9
        gd.step()
    with pytest.raises(RuntimeError):
        gd.step()
    with pytest.raises(ValueError):
        gd.prefill(torch.randint(0, 256, (2, 6)))  # batch differs


def test_unsupported_model_type():
    cfg = transformers.GPT2Config(n_layer=1, n_embd=64, n_head=2, vocab_size=64)
    with pytest.raises(NotImplementedError):
        GraphDecoder(transformers.GPT2LMHeadModel(cfg).eval(), batch=1, max_len=8)


def test_norm_folds_only_fp16_norms():
    """The batch-1 GEMV prologue reads the norm's weight (and LayerNorm's
    bias) as fp16: a norm kept in fp32 or bf16 inside an fp16 model must not
    be folded (nor take aq_decode_norm), whatever its class."""
    for kind in ("opt", "llama"):
        m = _model(kind).half()
        gd = GraphDecoder(m, batch=1, max_len=16, graph=False)
        layer = gd.layers[0]
        norm = layer.self_attn_layer_norm if kind == "opt" else layer.input_layernorm
        assert gd._norm_folds(norm)
        for dt in (torch.float32, torch.bfloat16):
            norm.to(dt)
            assert not gd._norm_folds(norm), (kind, dt)
        norm.half()
        if kind == "opt":
            norm.bias.data = norm.bias.data.float()  # weight fp16, bias not
            assert not gd._norm_folds(norm)
            norm.bias = None
            assert not gd._norm_folds(norm)


def test_options_need_the_gpu_path():
    """A window shorter than max_len (asked for, or the model's own), the 4-bit
    cache and sampling run on the GPU path only; a longer window changes nothing."""
    m = _model("mistral")
    for kw in (dict(window=8), dict(kv_bits=4), dict(sampling=True)):
        with pytest.raises(NotImplementedError):
            GraphDecoder(m, batch=1, max_len=16, graph=False, **kw)
    m.config.sliding_window = 8
    with pytest.raises(NotImplementedError):
        GraphDecoder(m, batch=1, max_len=16, graph=False)
    assert GraphDecoder(m, batch=1, max_len=8, graph=False).window is None


def test_window_prompts_reach_the_attention(monkeypatch):
    """The context hands every layer's queries, keys and values, the window and
    the model's scale to window_attention, and leaves the model as it was."""
    from atlasinfer_amd.integration import window_attention as W
    seen = []

    def plain(q, k, v, window, sinks, scale):
        seen.append((tuple(q.shape), tuple(k.shape), window, sinks, scale))
        G, N = q.shape[1] // k.shape[1], k.shape[2]
        s = q @ k.repeat_interleave(G, 1).transpose(2, 3) * scale
        i, j = torch.arange(N)[:, None], torch.arange(N)[None]
        s = s.masked_fill(~((j <= i) & ((i - j < window) | (j < sinks))), -float("inf"))
        return (s.softmax(-1) @ v.repeat_interleave(G, 1)).transpose(1, 2).contiguous()

    monkeypatch.setattr(W, "window_attention", plain)
    ids = torch.randint(0, 256, (2, 11))
    for kind, heads, scale in (("opt", 4, 1.0), ("llama", 2, 32 ** -0.5), ("mistral", 2, 32 ** -0.5)):
        m = _model(kind)
        with torch.no_grad():
            whole = m(input_ids=ids).logits
            seen.clear()
            with W.window_prompts(m, 100):
                same = m(input_ids=ids).logits
            with W.window_prompts(m, 3, 1):
                short = m(input_ids=ids).logits
            assert torch.equal(m(input_ids=ids).logits, whole)
        assert seen == [((2, 4, 11, 32), (2, heads, 11, 32), w, s, scale) for w, s in [(100, 0)] * 2 + [(3, 1)] * 2]
        assert (same - whole).abs().max() < 1e-5 and (short - whole).abs().max() > 1e-4
        assert torch.allclose(short[:, :4], whole[:, :4], atol=1e-5)  # these see everything through window and sink


def test_a_longer_window_than_the_configured_one_needs_the_gpu_path():
    """Where the steps would see every position but the model's own forward applies
    its configured window to the prompt, the torch form of the step is refused."""
    m = _model("mistral")
    m.config.sliding_window = 4
    for kw in (dict(window=64), dict(window=30, sinks=2), dict(sinks=28)):
        with pytest.raises(NotImplementedError):
            GraphDecoder(m, batch=1, max_len=32, graph=False, **kw)
    assert GraphDecoder(m, batch=1, max_len=4, graph=False, window=9).window is None
    m.config.sliding_window = None
    ids = torch.randint(0, 256, (1, 20))
    with torch.no_grad():
        ref = m.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=5, do_sample=False)
    assert torch.equal(GraphDecoder(m, batch=1, max_len=32, graph=False, window=64).generate(ids, 5), ref)


def test_window_prompts_nest_and_keep_to_their_thread(monkeypatch):
    """The innermost context counts, in whatever order they end; two models at once;
    another thread is refused, and the model is left as it was."""
    import threading
    from atlasinfer_amd.integration import window_attention as W
    seen = []

    def plain(q, k, v, window, sinks, scale):
        seen.append((window, sinks))
        return q.transpose(1, 2).contiguous()

    monkeypatch.setattr(W, "window_attention", plain)
    a, b = _model("llama"), _model("mistral")
    before = a.config._attn_implementation
    ids = torch.randint(0, 256, (1, 5))

    def ran(m):
        seen.clear()
        with torch.no_grad():
            m(input_ids=ids)
        assert len(set(seen)) <= 1
        return seen[0] if seen else None

    def elsewhere(f):
        out = []

        def run():
            try:
                out.append(f())
            except Exception as e:
                out.append(e)
        t = threading.Thread(target=run)
        t.start()
        t.join()
        return out[0]

    def enter(m):
        with W.window_prompts(m, 9):
            return ran(m)

    with W.window_prompts(a, 3, 1):
        assert ran(a) == (3, 1) and ran(b) is None
        with W.window_prompts(b, 4), W.window_prompts(a, 5):
            assert ran(a) == (5, 0) and ran(b) == (4, 0)
        assert ran(a) == (3, 1) and ran(b) is None
        assert isinstance(elsewhere(lambda: ran(a)), RuntimeError)
        assert isinstance(elsewhere(lambda: enter(a)), RuntimeError)
        assert elsewhere(lambda: enter(b)) == (9, 0)  # another model
        assert ran(a) == (3, 1) and ran(b) is None
    assert ran(a) is None and a.config._attn_implementation == b.config._attn_implementation == before
    assert elsewhere(lambda: enter(a)) == (9, 0)
    one, two = W.window_prompts(a, 3), W.window_prompts(a, 4)
    one.__enter__()
    two.__enter__()
    one.__exit__(None, None, None)
    assert ran(a) == (4, 0)
    two.__exit__(None, None, None)
    assert ran(a) is None and a.config._attn_implementation == before


def test_lists_of_prompts_need_pages():
    """Both ways in refuse them in the same words, and the decoder lives on."""
    gd = GraphDecoder(_model("llama"), batch=2, max_len=20, graph=False)
    ids = torch.randint(0, 256, (2, 5))
    want = gd.generate(ids, 6)
    for call in (gd.prefill, lambda p: gd.generate(p, 3)):
        for prompts in ([ids[0], ids[1, :3]], list(ids), tuple(ids), ids.tolist()):
            with pytest.raises(ValueError, match="several lengths need page_size"):
                call(prompts)
    assert torch.equal(gd.generate(ids, 6), want)
