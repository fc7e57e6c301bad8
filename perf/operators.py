"""Operators of a decoding loop whose speed counts, beside their plain forms.

Kinds of cases (``case["op"]``):

* ``sample``      -- the next token of every sequence from its logits and one
                     random number: temperature, top-k, top-p, min-p.
* ``kv4_prompt``  -- a prompt's keys and values into the 4-bit cache and back.
* ``kv4_step``    -- attention of one decode step over the 4-bit cache, the
                     step's key and value appended.
* ``ring_step``   -- the same over an fp16 cache that keeps a sliding window
                     and the first few positions (sinks).
* ``window``      -- attention of a prompt (or a piece of one) through a
                     sliding window with sinks.

Sizes are those of the OPT-1.3b, Llama-3-8B and Mistral-7B layers and generic
ones; logits have the spread and the few high tokens of a language model's,
keys have channels that stand out.  The 4-bit cache's layout is the one
declared in include/atlasinfer_amd.h (aq_kv4_store).
"""
import math

import torch

own = False

DEV = torch.device("cuda", 0)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
GROUP = 32  # elements of a 4-bit row that share a scale and a minimum
BLOCK = 32  # slots whose values are interleaved

MAX_LOGITS = 64 * 128256
MAX_PROMPT = 4 * 8 * 8192 * 128
MAX_CACHE = 32 * 8 * 16384 * 128
MAX_RING = 8 * 8 * 4100 * 128
MAX_SCORES = 32 * 8192 * 8192


def listed():
    return [
        # one sequence of a small model with the common settings: the smallest call
        dict(name="sample-b1-opt", op="sample", b=1, v=50272, dtype="fp16", t=0.8, k=50, p=0.95, m=0.0, per_row=False),
        # a serving batch, nucleus sampling alone: the whole row's mass counts
        dict(name="sample-b64-llama3", op="sample", b=64, v=128256, dtype="fp16", t=0.7, k=0, p=0.9, m=0.0,
             per_row=False),
        # many sequences of processed (fp32) logits, each with settings of its own
        dict(name="sample-b256-mixed", op="sample", b=256, v=32000, dtype="fp32", t=1.0, k=200, p=0.95, m=0.02,
             per_row=True),
        # a chat turn of one sequence into the cache
        dict(name="kv4-prompt-77", op="kv4_prompt", b=1, hkv=8, s=77, d=128, start=0),
        # a batch of long prompts
        dict(name="kv4-prompt-4x8192", op="kv4_prompt", b=4, hkv=8, s=8192, d=128, start=0),
        # a token of one sequence early in a conversation
        dict(name="kv4-step-b1", op="kv4_step", b=1, h=32, hkv=8, d=128, slots=768, pos=700, ragged=False, sinks=-1,
             rope=True),
        # a serving batch with histories of a few thousand tokens
        dict(name="kv4-step-b8", op="kv4_step", b=8, h=32, hkv=8, d=128, slots=4160, pos=4000, ragged=False, sinks=-1,
             rope=True),
        # a large batch with long histories of any length
        dict(name="kv4-step-b32-16k", op="kv4_step", b=32, h=32, hkv=8, d=128, slots=16384, pos=16383, ragged=True,
             sinks=-1, rope=True),
        # a small model far past its window
        dict(name="ring-step-b1-opt", op="ring_step", b=1, h=32, hkv=32, d=64, slots=1028, pos=5000, ragged=False,
             sinks=4, rope=False),
        # a serving batch past a window of 4096
        dict(name="ring-step-b8", op="ring_step", b=8, h=32, hkv=8, d=128, slots=4100, pos=9000, ragged=True, sinks=4,
             rope=True),
        # a prompt of odd length through a small model with a short window
        dict(name="window-1017-opt", op="window", b=1, h=32, hkv=32, d=64, m=1017, n=1017, window=256, sinks=4,
             padded=False),
        # a long prompt through a window of 4096
        dict(name="window-8192", op="window", b=1, h=32, hkv=8, d=128, m=8192, n=8192, window=4096, sinks=4,
             padded=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_heads(rng):
    if rng.random() < 0.4:
        return dict(h=32, hkv=32, d=64)
    hkv = rng.choice([1, 2, 4, 8])
    return dict(h=hkv * rng.choice([1, 2, 4, 8]), hkv=hkv, d=128)


def draw(rng):
    op = rng.choice(["sample", "sample", "kv4_prompt", "kv4_step", "kv4_step", "ring_step", "window"])
    if op == "sample":
        v = _log_int(rng, 1000, 256000)
        b = min(_log_int(rng, 1, 256), MAX_LOGITS // v)
        return dict(op=op, b=b, v=v, dtype=rng.choice(["fp16", "fp16", "bf16", "fp32"]),
                    t=0.0 if rng.random() < 0.1 else round(rng.uniform(0.3, 1.5), 3),
                    k=0 if rng.random() < 0.5 else _log_int(rng, 1, v),
                    p=1.0 if rng.random() < 0.3 else round(rng.uniform(0.3, 0.99), 3),
                    m=0.0 if rng.random() < 0.6 else round(rng.uniform(0.005, 0.3), 3), per_row=rng.random() < 0.3)
    if op == "kv4_prompt":
        b, hkv, d = _log_int(rng, 1, 32), rng.choice([1, 2, 8, 32]), rng.choice([64, 128])
        s = min(_log_int(rng, 1, 8192), MAX_PROMPT // (b * hkv * d))
        return dict(op=op, b=b, hkv=hkv, s=s, d=d, start=rng.choice([0, 0, _log_int(rng, 1, 500)]))
    if op in ("kv4_step", "ring_step"):
        heads = _draw_heads(rng)
        most = MAX_CACHE if op == "kv4_step" else MAX_RING
        b = _log_int(rng, 1, 64)
        slots = max(16, min(_log_int(rng, 16, 32768), most // (b * heads["hkv"] * heads["d"])))
        ring = op == "ring_step" or rng.random() < 0.3
        sinks = rng.choice([0, 1, 4, 5]) if ring else -1
        pos = rng.randrange(slots, 4 * slots) if ring and rng.random() < 0.7 else rng.randrange(slots)
        return dict(op=op, b=b, slots=slots, pos=pos, ragged=rng.random() < 0.5, sinks=sinks,
                    rope=heads["d"] == 128, **heads)
    heads = _draw_heads(rng)
    b = _log_int(rng, 1, 8)
    n = _log_int(rng, 1, 8192)
    n = max(1, min(n, int(math.sqrt(MAX_SCORES // (b * heads["h"])))))
    m = n if rng.random() < 0.7 else rng.randint(1, n)
    return dict(op=op, b=b, m=m, n=n, window=_log_int(rng, 1, max(1, n)), sinks=rng.choice([0, 1, 4, 16]),
                padded=b > 1 and rng.random() < 0.5, **heads)


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return dict(case, **{"sample": _prepare_sample, "kv4_prompt": _prepare_prompt, "kv4_step": _prepare_kv4,
                         "ring_step": _prepare_ring, "window": _prepare_window}[case["op"]](case, g))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float16)


def _keys(g, *shape):
    """N(0, 1) with four channels that stand out, as keys have."""
    k = _normal(g, *shape)
    k[..., torch.randperm(shape[-1], generator=g, device=DEV)[:4]] *= 4.0
    return k


def _prepare_sample(c, g):
    b, v = c["b"], c["v"]
    x = torch.randn(b, v, generator=g, device=DEV)
    x *= 1.5 + 2.0 * torch.rand(b, 1, generator=g, device=DEV)
    part = v // 24  # 24 high tokens, one in each part of the vocabulary
    top = torch.randint(0, part, (b, 24), generator=g, device=DEV) + torch.arange(24, device=DEV) * part
    x.scatter_add_(1, top, 10.0 * torch.rand(b, 24, generator=g, device=DEV))
    u = torch.rand(b, generator=g, device=DEV)
    if c["per_row"]:  # about the case's values, each row its own
        r = torch.rand(4, b, generator=g, device=DEV)
        t = c["t"] * (0.5 + r[0])
        k = (c["k"] * (0.5 + r[1])).int()
        p = (1.0 - (1.0 - c["p"]) * 2.0 * r[2]).clamp(min=0.05)
        m = c["m"] * 2.0 * r[3]
        return dict(logits=x.to(DTYPES[c["dtype"]]), u=u, temperature=t, top_k=k, top_p=p, min_p=m)
    return dict(logits=x.to(DTYPES[c["dtype"]]), u=u, temperature=c["t"], top_k=c["k"], top_p=c["p"], min_p=c["m"])


def _blocks(slots):
    return (slots + BLOCK - 1) // BLOCK * BLOCK


def _empty_cache(b, hkv, slots, d):
    n = _blocks(slots)
    return [torch.zeros(b, hkv, n, d // 2, dtype=torch.uint8, device=DEV),
            torch.zeros(b, hkv, n, d // GROUP, 2, dtype=torch.float16, device=DEV),
            torch.zeros(b, hkv, n // BLOCK, d * 16, dtype=torch.uint8, device=DEV),
            torch.zeros(b, hkv, n // BLOCK, d // GROUP, 4, 4, 4, dtype=torch.float16, device=DEV)]


def _prepare_prompt(c, g):
    b, hkv, s, d = c["b"], c["hkv"], c["s"], c["d"]
    # a forward pass hands them over as views of [b, s, heads, d]
    return dict(keys=_keys(g, b, s, hkv, d).transpose(1, 2), values=_normal(g, b, s, hkv, d).transpose(1, 2),
                cache=_empty_cache(b, hkv, c["start"] + s, d))


def _positions(c, g):
    lo = c["slots"] if c["pos"] >= c["slots"] else 0
    if not c["ragged"]:
        return torch.full((c["b"],), c["pos"], dtype=torch.int64, device=DEV)
    pos = torch.randint(lo, c["pos"] + 1, (c["b"],), generator=g, device=DEV)
    pos[0] = c["pos"]
    return pos


def _rope(c):
    """cos, sin [positions, d] fp16 in the rotate-half form."""
    n, d = max(c["slots"], c["pos"] + 1), c["d"]
    inv = 500000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * inv[None]
    a = torch.cat([a, a], dim=1)
    return a.cos().half(), a.sin().half()


def _step_inputs(c, g):
    b, h, hkv, d = c["b"], c["h"], c["hkv"], c["d"]
    cos, sin = _rope(c) if c["rope"] else (None, None)
    return dict(q=_normal(g, b, h, d), k_new=_keys(g, b, hkv, d), v_new=_normal(g, b, hkv, d), positions=_positions(c, g),
                cos=cos, sin=sin, scale=d ** -0.5)


def _prepare_kv4(c, g):
    cache = k_codes, k_params, v_codes, v_params = _empty_cache(c["b"], c["hkv"], c["slots"], c["d"])
    _random_codes(k_codes, g)
    _random_codes(v_codes, g)
    # groups of 32 normal elements span about 4 and start about -2; one group
    # of the keys has channels that stand out
    k_params[..., 0] = (0.27 + 0.03 * _normal(g, *k_params.shape[:-1])).clamp_(min=0.15)
    k_params[..., 1] = -2.0 + 0.3 * _normal(g, *k_params.shape[:-1])
    k_params[..., 0, :] *= 2.5
    v_params[..., :2] = (0.27 + 0.03 * _normal(g, *v_params.shape[:-1], 1)).clamp_(min=0.15)
    v_params[..., 2:] = -2.0 + 0.3 * _normal(g, *v_params.shape[:-1], 2)
    return dict(cache=cache, **_step_inputs(c, g))


def _random_codes(codes, g):
    """Pairs of 4-bit numbers, the middle ones more often (means of two)."""
    codes.random_(0, 256, generator=g)
    other = torch.empty_like(codes).random_(0, 256, generator=g)
    codes.copy_((codes & other) + (((codes ^ other) & 0xEE) >> 1))


def _prepare_ring(c, g):
    b, hkv, slots, d = c["b"], c["hkv"], c["slots"], c["d"]
    return dict(k_cache=_keys(g, b, hkv, slots, d), v_cache=_normal(g, b, hkv, slots, d), **_step_inputs(c, g))


def _prepare_window(c, g):
    b, h, hkv, d, m, n = c["b"], c["h"], c["hkv"], c["d"], c["m"], c["n"]
    starts = torch.randint(0, max(1, n // 2), (b,), generator=g, device=DEV, dtype=torch.int32) if c["padded"] else None
    # a forward pass hands them over as views of [b, s, heads, d]
    return dict(q=_normal(g, b, m, h, d).transpose(1, 2), k=_keys(g, b, n, hkv, d).transpose(1, 2),
                v=_normal(g, b, n, hkv, d).transpose(1, 2), starts=starts, scale=d ** -0.5)


# ---------------------------------------------------------------- the operators


def run(state):
    return {"sample": _run_sample, "kv4_prompt": _run_prompt, "kv4_step": _run_kv4, "ring_step": _run_ring,
            "window": _run_window}[state["op"]](state)


def _run_sample(s):
    if own:
        from atlasinfer_amd.integration.sampling import sample_tokens
        return sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                             min_p=s["min_p"])
    return _sample(s)


def _per_row(x, b, dtype):
    return x.to(dtype).view(b, 1) if torch.is_tensor(x) else torch.full((b, 1), x, dtype=dtype, device=DEV)


def _sample(s):
    """In 64 bits: the token is decided by where a sum passes a border."""
    x = s["logits"].double()
    b, v = x.shape
    # a setting is a 32-bit number, also where it is given as a Python float
    t, k = _per_row(s["temperature"], b, torch.float32).double(), _per_row(s["top_k"], b, torch.int64)
    p, m = _per_row(s["top_p"], b, torch.float32).double(), _per_row(s["min_p"], b, torch.float32).double()
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: the lower index first
    w = torch.exp((xs - xs[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(v, device=DEV)[None]
    w = torch.where((rank < k) | (k <= 0), w, 0.0)
    c = torch.cumsum(w, dim=1)
    keep = ((c - w < p * c[:, -1:]) | (p >= 1)) & (w >= m.clamp(max=1.0)) & (w > 0) & ((rank == 0) | (t > 0))
    keep |= rank == 0
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    c = torch.cumsum(w, dim=1)
    return torch.argmax((c > s["u"].double()[:, None] * c[:, -1:]).int(), dim=1)


def _quantize(x):
    """Codes 0 .. 15 of x [..., d] and the scale and minimum of each group of
    32 [..., d / 32, 2]: the scale is (max - min) / 15 in fp16, one step less where 15 of it above the
    minimum would pass the largest fp16."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    scale = ((high - low) / 15.0).half()
    scale = torch.where(low + 15.0 * scale.float() >= 65520.0, (scale.view(torch.int16) - 1).view(torch.float16), scale)
    s = scale.float().unsqueeze(-1)
    codes = torch.round((x - low.unsqueeze(-1)) / torch.where(s > 0, s, 1.0)).clamp(0, 15) * (s > 0)
    return codes.to(torch.uint8).flatten(-2), torch.stack([scale, low.half()], dim=-1)


def _values(codes, params):
    x, params = codes.unflatten(-1, (-1, GROUP)).float(), params.float()
    return (x * params[..., :1] + params[..., 1:]).flatten(-2)


def _nibbles(n):
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _of_nibbles(b):
    return torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)


def _pack_values(codes):
    """[b, heads, 32 n, d] -> [b, heads, n, 16 d]: slot 16 t + 4 r + i, element 64 a + 16 e + l."""
    x = codes.reshape(*codes.shape[:2], -1, 2, 4, 4, codes.shape[-1] // 64, 4, 16)  # n t r i a e l
    return _nibbles(x.permute(0, 1, 2, 6, 4, 8, 7, 3, 5).flatten(-2)).flatten(3)  # n a r l e (t i)


def _unpack_values(packed):
    b, hkv, n, size = packed.shape
    x = _of_nibbles(packed.reshape(b, hkv, n, -1, 4, 16, 4, 4)).unflatten(-1, (2, 4))  # n a r l e t i
    return x.permute(0, 1, 2, 7, 4, 8, 3, 6, 5).reshape(b, hkv, n * BLOCK, size // 16)


def _pack_params(params):
    """[b, heads, 32 n, groups, 2] -> [b, heads, n, groups, 4, 4, 4]."""
    b, hkv, slots, groups, _ = params.shape
    x = params.reshape(b, hkv, -1, 2, 4, 4, groups, 2)  # n t r i g p
    return x.permute(0, 1, 2, 6, 4, 5, 7, 3).reshape(b, hkv, -1, groups, 4, 4, 4)


def _unpack_params(packed):
    b, hkv, n, groups = packed.shape[:4]
    x = packed.reshape(b, hkv, n, groups, 4, 4, 2, 2)  # n g r i p t
    return x.permute(0, 1, 2, 7, 4, 5, 3, 6).reshape(b, hkv, n * BLOCK, groups, 2)


def _cache_values(cache):
    """Keys and values [b, heads, slots, d] that a 4-bit cache stands for."""
    k_codes, k_params, v_codes, v_params = cache
    return _values(_of_nibbles(k_codes), k_params), _values(_unpack_values(v_codes), _unpack_params(v_params))


def _run_prompt(s):
    if own:
        from atlasinfer_amd.memory.decode_cache import kv4_load, kv4_store
        kv4_store(s["keys"], s["values"], s["cache"], start=s["start"])
        return (*kv4_load(s["cache"], s["start"] + s["s"]), *s["cache"])
    k_codes, k_params, v_codes, v_params = s["cache"]
    lo, hi = s["start"], s["start"] + s["s"]
    codes, k_params[:, :, lo:hi] = _quantize(s["keys"])
    k_codes[:, :, lo:hi] = _nibbles(codes)
    held, params = _unpack_values(v_codes), _unpack_params(v_params)
    held[:, :, lo:hi], params[:, :, lo:hi] = _quantize(s["values"])
    v_codes.copy_(_pack_values(held))
    v_params.copy_(_pack_params(params))
    keys, values = _cache_values(s["cache"])
    return keys[:, :, :hi].half(), values[:, :, :hi].half(), *s["cache"]


def _rotate(x, cos, sin):
    """fp16(fp16(x cos) + fp16(r sin)) as fp16 tensors give it."""
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


def _slot(positions, slots, sinks):
    if sinks < 0:
        return positions
    return torch.where(positions < slots, positions, sinks + (positions - sinks) % (slots - sinks))


def _rotated(s):
    q, k = s["q"], s["k_new"]
    if s["cos"] is None:
        return q, k
    cos, sin = s["cos"][s["positions"]].unsqueeze(1), s["sin"][s["positions"]].unsqueeze(1)
    return _rotate(q, cos, sin), _rotate(k, cos, sin)


def _attend(q, keys, values, positions, slots, scale):
    """Softmax attention of q [b, h, d] over the slots written so far."""
    b, h, d = q.shape
    hkv = keys.shape[1]
    scores = q.to(keys.dtype).view(b, hkv, h // hkv, d) @ keys[:, :, :slots].transpose(2, 3) * scale
    unseen = torch.arange(slots, device=DEV)[None] > positions[:, None]
    scores.masked_fill_(unseen[:, None, None], -math.inf)
    return (torch.softmax(scores, dim=-1) @ values[:, :, :slots]).view(b, h, d)


def _run_kv4(s):
    if own:
        from atlasinfer_amd.memory.decode_cache import kv4_attention
        out = kv4_attention(s["q"], s["k_new"], s["v_new"], s["cache"], s["positions"], slots=s["slots"],
                            sinks=None if s["sinks"] < 0 else s["sinks"], scale=s["scale"],
                            rope=None if s["cos"] is None else (s["cos"], s["sin"]))
        return (out, *s["cache"])
    k_codes, k_params, v_codes, v_params = s["cache"]
    q, k = _rotated(s)
    slot = _slot(s["positions"], s["slots"], s["sinks"])
    rows = torch.arange(s["b"], device=DEV)
    codes, k_params[rows, :, slot] = _quantize(k)
    k_codes[rows, :, slot] = _nibbles(codes)
    block, at = slot // BLOCK, slot % BLOCK
    held = _unpack_values(v_codes[rows, :, block].unsqueeze(2))
    params = _unpack_params(v_params[rows, :, block].unsqueeze(2))
    held[rows, :, at], params[rows, :, at] = _quantize(s["v_new"])
    v_codes[rows, :, block] = _pack_values(held).squeeze(2)
    v_params[rows, :, block] = _pack_params(params).squeeze(2)
    keys, values = _cache_values(s["cache"])
    return (_attend(q, keys, values, s["positions"], s["slots"], s["scale"]).half(), *s["cache"])


def _run_ring(s):
    if own:
        from atlasinfer_amd.memory.decode_cache import window_decode_attention
        out = window_decode_attention(s["q"], s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["positions"],
                                      sinks=s["sinks"], scale=s["scale"],
                                      rope=None if s["cos"] is None else (s["cos"], s["sin"]))
        return out, s["k_cache"], s["v_cache"]
    q, k = _rotated(s)
    slot = _slot(s["positions"], s["slots"], s["sinks"])
    rows = torch.arange(s["b"], device=DEV)
    s["k_cache"][rows, :, slot] = k
    s["v_cache"][rows, :, slot] = s["v_new"]
    out = _attend(q, s["k_cache"].float(), s["v_cache"].float(), s["positions"], s["slots"], s["scale"])
    return out.half(), s["k_cache"], s["v_cache"]


def _visible(s, m, n):
    """[b or 1, m, n]: the keys that each query sees."""
    i = torch.arange(n - m, n, device=DEV)[None, :, None]
    j = torch.arange(n, device=DEV)[None, None]
    first = 0 if s["starts"] is None else s["starts"].view(-1, 1, 1)
    return (j <= i) & (j >= first) & ((i - j < s["window"]) | (j - first < s["sinks"]))


def _run_window(s):
    if own:
        from atlasinfer_amd.integration.window_attention import window_attention
        return window_attention(s["q"], s["k"], s["v"], window=s["window"], sinks=s["sinks"], scale=s["scale"],
                                starts=s["starts"])
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, h, m, d = q.shape
    hkv, n = k.shape[1], k.shape[2]
    scores = q.reshape(b, hkv, -1, d) @ k.transpose(2, 3)  # [b, hkv, (h / hkv) m, n]
    scores = scores.mul_(s["scale"]).view(b, hkv, -1, m, n)
    scores.masked_fill_(~_visible(s, m, n)[:, None, None], -math.inf)
    w = torch.exp(scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)))
    total = w.sum(-1, keepdim=True)
    out = (w.view(b, hkv, -1, n) @ v).view(b, hkv, -1, m, d) / torch.where(total > 0, total, 1.0)
    return out.view(b, h, m, d).transpose(1, 2).contiguous().half()


# ---------------------------------------------------------------- work, and results in 64 bits


def work(case):
    c = case
    if c["op"] == "sample":
        size = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": c["b"] * (c["v"] * size + 12), "flops": 2 * c["b"] * c["v"]}
    d = c["d"]
    if c["op"] == "kv4_prompt":
        # both in and back out in fp16, the 4-bit rows written and read
        rows = 2 * c["b"] * c["hkv"] * c["s"]
        return {"bytes": rows * (4 * d + 2 * (d // 2 + d // 8)), "flops": 6 * rows * d}
    if c["op"] in ("kv4_step", "ring_step"):
        row = d // 2 + d // 8 if c["op"] == "kv4_step" else 2 * d
        held = min(c["pos"] + 1, c["slots"])
        if c["ragged"] and c["pos"] < c["slots"]:
            held = (held + 1) // 2  # on average
        return {"bytes": 2 * c["b"] * c["hkv"] * held * row + 4 * c["b"] * (c["h"] + c["hkv"]) * d,
                "flops": 4 * c["b"] * c["h"] * held * d}
    # without padding
    seen = sum(min(i + 1, c["window"] + c["sinks"]) for i in range(c["n"] - c["m"], c["n"]))
    return {"bytes": 4 * c["b"] * d * (c["h"] * c["m"] + c["hkv"] * c["n"]), "flops": 4 * c["b"] * c["h"] * d * seen}


def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "kv4_prompt": _exact_prompt, "kv4_step": _exact_kv4, "ring_step": _exact_ring,
            "window": _exact_window}[case["op"]](s)


def _exact_sample(s):
    return None


def _groups(x):
    """Every group of 32 of x, written anew from its scale, minimum and codes."""
    x = x.reshape(*x.shape[:-1], -1, 32)
    low, high = x.min(-1, keepdim=True).values.double(), x.max(-1, keepdim=True).values.double()
    step = ((high - low) / 15).half().double()
    step = torch.where(low + 15 * step >= 65520, step - 8, step)  # only the largest numbers: fp16 steps of 8 there
    code = ((x.double() - low) / step.clamp(min=1e-300)).round().clamp(0, 15)
    return torch.where(step > 0, low + step * code, low).reshape(*x.shape[:-2], -1)


def _exact_prompt(s):
    keys, values = [_groups(s[x]) for x in ("keys", "values")]
    if s["start"]:
        zeros = torch.zeros(s["b"], s["hkv"], s["start"], s["d"], dtype=torch.float64, device=DEV)
        keys, values = torch.cat([zeros, keys], 2), torch.cat([zeros, values], 2)
    return keys, values, None, None, None, None


def _turned(x, s):
    if s["cos"] is None:
        return x.double()
    out = torch.empty_like(x)
    half = x.shape[-1] // 2
    for b, p in enumerate(s["positions"].tolist()):
        c, n, a, z = s["cos"][p].double(), s["sin"][p].double(), x[b, :, :half].double(), x[b, :, half:].double()
        out[b, :, :half] = ((a * c[:half]).half().double() + (-z * n[:half]).half().double()).half()
        out[b, :, half:] = ((z * c[half:]).half().double() + (a * n[half:]).half().double()).half()
    return out.double()


def _each(s, rows):
    """Attention of each sequence and key/value head by itself; rows(b, j) gives its keys and values."""
    q = _turned(s["q"], s)
    out = torch.empty_like(q)
    g = s["h"] // s["hkv"]
    for b, p in enumerate(s["positions"].tolist()):
        held = min(p + 1, s["slots"])
        at = p if p < s["slots"] else s["sinks"] + (p - s["sinks"]) % (s["slots"] - s["sinks"])
        for j in range(s["hkv"]):
            k, v = rows(b, j, at)
            w = torch.softmax(k[:held] @ q[b, j * g:(j + 1) * g].T * s["scale"], dim=0)
            out[b, j * g:(j + 1) * g] = w.T @ v[:held]
    return out


def _exact_kv4(s):
    if s["b"] * s["hkv"] > 4096:
        return None
    k_new, v_new = _groups(_turned(s["k_new"], s).half()), _groups(s["v_new"])
    kc, kp, vc, vp = s["cache"]
    slot = torch.arange(kc.shape[2], device=DEV)
    t, r, i = slot % 32 // 16, slot % 16 // 4, slot % 4
    e = torch.arange(s["d"], device=DEV)
    # the byte and nibble of slot and element in a sequence's values
    byte = slot[:, None] // 32 * 16 * s["d"] + (e // 64 * 1024 + e % 16 * 16 + e % 64 // 16 * 4)[None] + (r * 256 + t * 2 + i // 2)[:, None]
    shift = (i % 2 * 4)[:, None]

    def rows(b, j, at):
        keys = torch.stack([kc[b, j] % 16, kc[b, j] // 16], -1).reshape(len(slot), -1).double()
        keys = keys * kp[b, j, :, :, 0].double().repeat_interleave(32, 1) + kp[b, j, :, :, 1].double().repeat_interleave(32, 1)
        codes = (vc[b, j].reshape(-1)[byte].int() >> shift & 15).double()
        par = vp[b, j][slot // 32, :, r, i].double()  # [slots, groups, 4]
        step, low = par[..., :2][torch.arange(len(slot), device=DEV), :, t], par[..., 2:][torch.arange(len(slot), device=DEV), :, t]
        values = codes * step.repeat_interleave(32, 1) + low.repeat_interleave(32, 1)
        keys[at], values[at] = k_new[b, j], v_new[b, j]
        return keys, values

    return _each(s, rows), None, None, None, None


def _exact_ring(s):
    k_new = _turned(s["k_new"], s)

    def rows(b, j, at):
        keys, values = s["k_cache"][b, j].double(), s["v_cache"][b, j].double()
        keys[at], values[at] = k_new[b, j], s["v_new"][b, j].double()
        return keys, values

    return _each(s, rows), None, None


def _exact_window(s):
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    b, h, m, d = q.shape
    n, g = k.shape[2], h // k.shape[1]
    out = torch.zeros(b, m, h, d, dtype=torch.float64, device=DEV)
    j = torch.arange(n, device=DEV)
    for r in range(b):
        first = 0 if s["starts"] is None else int(s["starts"][r])
        for lo in range(0, m, 1024):
            hi = min(m, lo + 1024)
            i = torch.arange(n - m + lo, n - m + hi, device=DEV)[:, None]
            sees = (j >= first) & (j <= i) & ((j > i - s["window"]) | (j < first + s["sinks"]))
            for a in range(h):
                w = (q[r, a, lo:hi] @ k[r, a // g].T * s["scale"]).masked_fill_(~sees, -math.inf)
                w = torch.softmax(w, dim=1).nan_to_num_(0.0)  # a query that sees nothing answers zero
                out[r, lo:hi, a] = w @ v[r, a // g]
    return out
