"""PrefillStep and DecodeStep over a KVCache: a prompt and the tokens after it through
a small MLX-4bit Llama, against the whole pipeline in numpy (rotary embedding and
causal attention included) on the same tokens; captured steps against eager ones;
a bounded cache."""
import numpy as np
import pytest

from oracle import q4_oracle as o
from test_gpu_decode import _bf16
from test_gpu_loader import CFG, _write_model

pytestmark = pytest.mark.gpu


def _ref_logits(src, tokens):
    """Logits after the last token, from the definition: every token, every layer."""
    c = CFG
    eps, g, D = c["rms_norm_eps"], 64, c["head_dim"]
    H, K = c["num_attention_heads"], c["num_key_value_heads"]
    lin = lambda x, p: o.matmul_q4_f64(x, src[p + ".weight"], src[p + ".scales"], src[p + ".biases"], g)
    e = "model.embed_tokens"
    S = len(tokens)
    h = o.embedding_q4_ref(src[e + ".weight"], src[e + ".scales"], src[e + ".biases"], tokens, g)
    angle = np.arange(S)[:, None] * c["rope_theta"] ** (-np.arange(0, D, 2) / D)[None]
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]

    def rotated(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1).astype(np.float16).astype(np.float64)

    for i in range(c["num_hidden_layers"]):
        p = f"model.layers.{i}"
        xn = o.rms_norm_ref(h, src[p + ".input_layernorm.weight"], eps)
        q, k, v = (lin(xn, f"{p}.self_attn.{x}_proj").astype(np.float16).astype(np.float64).reshape(S, -1, D)
                   for x in "qkv")
        q, k = rotated(q), rotated(k)
        attn = np.zeros((S, H, D))
        for n in range(H):
            x = q[:, n] @ k[:, n // (H // K)].T / np.sqrt(D)
            x = np.where(np.tri(S, dtype=bool), x, -np.inf)
            w = np.exp(x - x.max(1, keepdims=True))
            attn[:, n] = w / w.sum(1, keepdims=True) @ v[:, n // (H // K)]
        ov = lin(attn.reshape(S, -1).astype(np.float16), f"{p}.self_attn.o_proj")
        res, xn2 = o.residual_rms_norm_ref(h, ov.astype(np.float16),
                                           _bf16(src[p + ".post_attention_layernorm.weight"]), eps)
        act = o.silu_mul_f64(lin(xn2, f"{p}.mlp.gate_proj"), lin(xn2, f"{p}.mlp.up_proj"))
        h = o.residual_add_ref(res, lin(act.astype(np.float16), f"{p}.mlp.down_proj"))
    xn = o.rms_norm_ref(h[-1:], src["model.norm.weight"].astype(np.float32), eps)
    return lin(xn, e)[0]


def _cache(pkg, dev, capacity, **kw):
    return pkg.KVCache(CFG["num_hidden_layers"], 1, CFG["num_key_value_heads"], capacity, CFG["head_dim"], device=dev,
                       **kw)


def _close(logits, ref, what):
    err = np.max(np.abs(logits[0].float().cpu().numpy() - ref)) / np.max(np.abs(ref))
    assert err <= 1e-2, (what, err)       # the parity gate of the steps without a cache


@pytest.mark.parametrize("S,track", [(1, False), (9, True), (150, True), (150, False)])
def test_prompt_then_tokens(pkg, dev, tmp_path, S, track):
    import torch
    from swiftltx_amd.decode import DecodeStep
    from swiftltx_amd.prefill import PrefillStep
    from swiftltx_amd.weights import ModelWeights
    src = _write_model(tmp_path)
    mw = ModelWeights.from_directory(str(tmp_path), device=dev)
    tokens = np.random.default_rng(S).integers(0, CFG["vocab_size"], S).tolist()
    cache = _cache(pkg, dev, 200, track_weights=track)
    ps = PrefillStep(mw, S, cache=cache)
    ps.tokens.copy_(torch.tensor(tokens, dtype=torch.int32))
    _close(ps.forward(), _ref_logits(src, tokens), "prompt")
    assert cache.length.tolist() == [S] == cache.next_position.tolist()
    ds = DecodeStep(mw, cache=cache)
    for step in range(4):
        tok = (17 * step + 5) % CFG["vocab_size"]
        tokens.append(tok)
        ds.token.fill_(tok)
        ds.forward()
        _close(ds.logits, _ref_logits(src, tokens), step)
    assert cache.length.tolist() == [S + 4]
    if track:      # each of the last tokens gave each head the weight 1
        rows = min(S, 64) + 4
        per_group = CFG["num_attention_heads"] // CFG["num_key_value_heads"]
        total = cache.weight.double().sum(-1)
        assert (total - rows * per_group).abs().max() < 1e-3


def test_prompt_in_chunks(pkg, dev, tmp_path):
    """A prompt in two chunks leaves the cache and the logits of one, to rounding."""
    import torch
    from swiftltx_amd.prefill import PrefillStep
    from swiftltx_amd.weights import ModelWeights
    src = _write_model(tmp_path)
    mw = ModelWeights.from_directory(str(tmp_path), device=dev)
    tokens = np.random.default_rng(3).integers(0, CFG["vocab_size"], 120).tolist()
    cache = _cache(pkg, dev, 130)
    for part in (tokens[:70], tokens[70:]):
        ps = PrefillStep(mw, len(part), cache=cache)
        ps.tokens.copy_(torch.tensor(part, dtype=torch.int32))
        logits = ps.forward()
    _close(logits, _ref_logits(src, tokens), "chunks")


@pytest.mark.parametrize("budget", [None, 24])
def test_graphs_match_eager(pkg, dev, tmp_path, budget):
    """Greedy tokens after a prompt: each captured step over the growing (or bounded)
    cache gives the eager step's token, several replays long, with the program's own
    work between them."""
    import torch
    from swiftltx_amd.decode import DecodeStep
    from swiftltx_amd.prefill import PrefillStep
    from swiftltx_amd.weights import ModelWeights
    _write_model(tmp_path)
    mw = ModelWeights.from_directory(str(tmp_path), device=dev)
    prompt = torch.tensor(np.random.default_rng(5).integers(0, CFG["vocab_size"], 30), dtype=torch.int32, device=dev)
    opts = {} if budget is None else dict(budget=budget, sinks=2, recent=6)
    s = torch.cuda.Stream()

    def start():
        cache = _cache(pkg, dev, 64, track_weights=budget is not None)
        ps = PrefillStep(mw, 30, cache=cache, stream=s, **opts)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            ps.tokens.copy_(prompt)
            first = int(ps.forward().argmax())
        return cache, first

    cache, first = start()
    ds = DecodeStep(mw, cache=cache, stream=s, **opts)
    eager = []
    with torch.cuda.stream(s):
        ds.token.fill_(first)
        for _ in range(9):
            eager.append(int(ds.step().item()))
    cache, first2 = start()
    assert first2 == first
    ds = DecodeStep(mw, cache=cache, stream=s, **opts)
    with torch.cuda.stream(s):
        ds.token.fill_(first)
    ds.capture()                       # one eager step, which appends its token
    s.synchronize()
    got = [int(ds.token.item())]
    for _ in range(8):
        ds.replay()
        torch.cuda.synchronize()
        got.append(int(ds.token.item()))
        torch.zeros(1000, device=dev).add_(1)
    assert got == eager
    n = 39 if budget is None else budget
    assert cache.length.tolist() == [n] and cache.next_position.tolist() == [39]
    assert (cache.position[:, 0, :, :n] >= 33).sum(-1).eq(6).all() if budget else True


def test_wrong_caches(pkg, dev, tmp_path):
    import torch
    from swiftltx_amd.decode import DecodeStep
    from swiftltx_amd.prefill import PrefillStep
    from swiftltx_amd.weights import ModelWeights
    _write_model(tmp_path)
    mw = ModelWeights.from_directory(str(tmp_path), device=dev)
    for bad in (pkg.KVCache(1, 1, 2, 16, 64, device=dev), pkg.KVCache(2, 2, 2, 16, 64, device=dev),
                pkg.KVCache(2, 1, 4, 16, 64, device=dev), pkg.KVCache(2, 1, 2, 16, 128, device=dev),
                pkg.KVCache(2, 1, 2, 16, 64, dtype=torch.bfloat16, device=dev)):
        with pytest.raises(ValueError):
            DecodeStep(mw, cache=bad)
        with pytest.raises(ValueError):
            PrefillStep(mw, 4, cache=bad)
    cache = _cache(pkg, dev, 16)
    with pytest.raises(ValueError):
        DecodeStep(mw, cache=cache, attention=lambda layer, qkv: qkv)
    with pytest.raises(ValueError):
        DecodeStep(mw, cache=cache, budget=8)     # no weights tracked
    with pytest.raises(ValueError):
        DecodeStep(mw, budget=8)
