"""Attention of as many rows and heads as take blocks of 128 rows (attn_seq.hip: from
256 of them on, from 768 under a causal mask or documents), every mask, both types,
odd sizes: a sample of the heads against attention in 64 bits (attn_bounds.py)."""
import math

import pytest

import attn_bounds
import attn_ref as R

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def _inputs(dev, x, seed, B, Sq, Sk, Hq, Hk, D):
    import torch
    gen = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=gen, device=dev).to(_dt(x))
    return mk(B, Sq, Hq, D), mk(B, Sk, Hk, D), mk(B, Sk, Hk, D)


def _seen(b, Sq, Sk, dev, causal=False, prefix=None, q_docs=None, k_docs=None, q_lens=None, k_lens=None):
    """(seen [Sq, Sk], rows, keys, key - position [Sq, Sk]) of sequence b."""
    import torch
    m = Sq if q_lens is None else int(q_lens[b])
    n = Sk if k_lens is None else int(k_lens[b])
    i, j = torch.arange(Sq, device=dev)[:, None], torch.arange(Sk, device=dev)[None]
    far = j - (i + n - m)
    seen = (j < n).expand(Sq, Sk)
    if causal:
        seen = seen & ((far <= 0) | (j < (0 if prefix is None else int(prefix[b]))))
    if q_docs is not None:
        seen = seen & (q_docs[b][:, None] == k_docs[b][None]) & (q_docs[b][:, None] >= 0)
    return seen, m, n, far


def _check(pkg, dev, q, k, v, scale, *, softcap=0.0, bias=None, bias_zero=0, **masks):
    import torch
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1:3]
    blocks = B * Hq * -(-Sq // 128)
    assert blocks >= (768 if masks.get("causal") or "q_docs" in masks else 256)
    got = pkg.attention(q, k, v, scale, softcap=softcap, bias=bias, bias_zero=bias_zero, **masks)
    torch.cuda.synchronize()
    for b in sorted({0, B // 2, B - 1}):
        seen, m, n, far = _seen(b, Sq, Sk, dev, **masks)
        for h in sorted({0, Hq // 2 + 1, Hq - 1}):
            g = h // (Hq // Hk)
            add = None if bias is None else bias[h if bias.shape[0] > 1 else 0][(far + bias_zero).clamp(0, bias.shape[1] - 1)]
            _, ref, bound = attn_bounds.head(q[b, :m, h], k[b, :, g], v[b, :, g], scale, softcap,
                                             None if add is None else add[:m], seen[:m])
            R.check_out(got[b, :m, h], ref, bound, q.dtype, f"sequence {b} head {h}")
        if "q_lens" in masks:
            assert (got[b, m:] == 0).all()
    return got


DIMS = [64, 128, 40, 120]


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("cap", [0.0, 8.0, 1e5])
def test_bidirectional(pkg, dev, cap, biased, D, x):
    import torch
    q, k, v = _inputs(dev, x, D, 8, 191, 333, 32, 8, D)
    bias = torch.randn(32, 301, generator=torch.Generator(device=dev).manual_seed(D), device=dev) if biased else None
    _check(pkg, dev, q, k, v, 1.5 / math.sqrt(D), softcap=cap, bias=bias, bias_zero=150 if biased else 0)


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("kind", ["plain", "capped", "biased", "both", "prefix", "lengths"])
def test_causal(pkg, dev, kind, D, x):
    import torch
    B = 13
    q, k, v = _inputs(dev, x, D + 1, B, 129, 260, 32, 4, D)
    masks = dict(causal=True)
    if kind in ("biased", "both"):
        masks.update(bias=torch.randn(1, 77, generator=torch.Generator(device=dev).manual_seed(D), device=dev), bias_zero=70)
    if kind in ("capped", "both"):
        masks.update(softcap=12.0)
    if kind == "prefix":
        masks.update(prefix=torch.tensor([0, 1, 131, 200, 500] + [160 + b for b in range(B - 5)], dtype=torch.int32, device=dev))
    if kind == "lengths":
        masks.update(q_lens=torch.tensor([129, 100, 0, 1, 64] + [128] * (B - 6) + [33], dtype=torch.int32, device=dev),
                     k_lens=torch.tensor([3, 260, 260, 1, 65] + [200] * (B - 6) + [33], dtype=torch.int32, device=dev))
    _check(pkg, dev, q, k, v, 1.5 / math.sqrt(D), **masks)


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 72])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["plain", "capped", "biased", "both"])
def test_documents(pkg, dev, kind, causal, D, x):
    import torch
    B, S = 4, 769
    q, k, v = _inputs(dev, x, D + 2, B, S, S, 32, 8, D)
    docs = torch.zeros(B, S, dtype=torch.int32)
    docs[0] = torch.arange(S) // 61                       # packed, ends inside tiles
    docs[0, 700:] = -1                                    # padding sees nothing
    docs[1] = torch.arange(S) // 64
    docs[2] = torch.randint(0, 3, (S,), generator=torch.Generator().manual_seed(1))
    docs[3] = 7
    docs[3, ::5] = -5
    docs = docs.to(dev)
    more = {}
    if kind in ("biased", "both"):
        more.update(bias=torch.randn(32, 99, generator=torch.Generator(device=dev).manual_seed(D), device=dev), bias_zero=49)
    if kind in ("capped", "both"):
        more.update(softcap=12.0)
    got = _check(pkg, dev, q, k, v, 1.5 / math.sqrt(D), causal=causal, q_docs=docs, k_docs=docs, **more)
    assert (got[0, 700:] == 0).all() and (got[3, ::5] == 0).all()


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_unseen_values_do_not_matter(pkg, dev, D, x):
    """Infinities and NaN in keys that a row does not see: bit for bit the result of
    clean ones; what rows see of them comes through."""
    import torch
    B, S = 4, 400
    q, k, v = _inputs(dev, x, D + 3, B, S, S, 64, 8, D)
    docs = (torch.arange(S, device=dev) // 75).to(torch.int32).repeat(B, 1)
    lens = torch.tensor([400, 301, 220, 399], dtype=torch.int32, device=dev)
    for masks in (dict(causal=True), dict(causal=True, q_lens=lens, k_lens=lens), dict(q_docs=docs, k_docs=docs)):
        clean = pkg.attention(q, k, v, 0.1, **masks)
        for bad in (math.nan, math.inf, -math.inf):
            k2, v2 = k.clone(), v.clone()
            k2[:, 301:] = bad
            v2[:, 301:, :, ::3] = bad
            got = pkg.attention(q, k2, v2, 0.1, **masks)
            for b in range(B):
                seen, m, _, _ = _seen(b, S, S, dev, **masks)
                safe = ~seen[:, 301:].any(1)
                safe[m:] = False
                assert safe.any() and torch.equal(got[b][safe], clean[b][safe])
    v2 = v.clone()
    v2[:, 350, 0, 5], v2[:, 350, 0, 6], v2[:, 351, 0, 6] = math.inf, math.inf, -math.inf
    got, clean = (pkg.attention(q, k, t, 0.1, causal=True) for t in (v2, v))
    assert (got[:, 351:, :8, 5] == math.inf).all() and (got[:, 350, :8, 6] == math.inf).all()
    assert got[:, 351:, :8, 6].isnan().all()
    keep = torch.ones(B, S, 64, D, dtype=torch.bool, device=dev)
    keep[:, 350:, :8, 5:7] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_a_chunk_over_a_cache(pkg, dev, D, x):
    """Chunks of 521 tokens of 8 sequences, four query heads to a block's rows."""
    import torch
    B, T, Hq, Hk, lengths = 8, 521, 32, 8, [0, 1, 64, 100, 7, 127, 128, 79]
    gen = torch.Generator(device=dev).manual_seed(D)
    k, v = (torch.randn(1, B, Hk, 660, D, generator=gen, device=dev).to(_dt(x)) for _ in range(2))
    for b, n in enumerate(lengths):      # what nobody sees
        k[0, b, :, n + T:], v[0, b, :, n + T:] = math.nan, math.inf
    cache = pkg.KVCache.from_tensors(k, v, torch.tensor([lengths] * 2, dtype=torch.int32, device=dev))
    q = torch.randn(B, T, Hq, D, generator=gen, device=dev).to(_dt(x))
    for cap in (0.0, 20.0, 1e5):
        got = pkg.attention_cached(q, cache, 0, 1.5 / math.sqrt(D), softcap=cap)
        for b in (0, 3, 7):
            n = lengths[b]
            seen = torch.arange(n + T, device=dev)[None] <= n + torch.arange(T, device=dev)[:, None]
            for h in (0, 5, 31):
                _, ref, bound = attn_bounds.head(q[b, :, h], k[0, b, h // 4, :n + T], v[0, b, h // 4, :n + T],
                                                 1.5 / math.sqrt(D), cap, None, seen)
                R.check_out(got[b, :, h], ref, bound, q.dtype, f"sequence {b} head {h}")
