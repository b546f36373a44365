"""Attention under score caps up to the ends of fp32, whole sequences and over a cache,
against the bounds of attn_bounds.py."""
import pytest

import attn_bounds
import attn_ref as R

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def _qkv(dev, x, seed, q_shape, k_shape, spread=1.0):
    import torch
    gen = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda s: (torch.randn(*s, generator=gen, device=dev) * spread).to(_dt(x))
    return mk(q_shape), mk(k_shape), mk(k_shape)


def _check(got, q, k, v, scale, cap=0.0, bias=None, seen=None, heads=None, what=""):
    """Heads of got [B, S, Hq, D] against attention in 64 bits; bias [Hq, S, N]."""
    B, S, Hq, D = q.shape
    group = Hq // k.shape[2]
    for b in range(B):
        for h in heads or range(Hq):
            _, ref, bound = attn_bounds.head(q[b, :, h], k[b, :, h // group], v[b, :, h // group], scale, cap,
                                             None if bias is None else bias[h], seen)
            R.check_out(got[b, :, h], ref, bound, q.dtype, f"{what} sequence {b} head {h}")


CAPS = [30.0, 64.0, 65.0, 1e3, 1e4, 1e5, 1e6, 1e8, 1e30, 1e38]


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("cap", CAPS)
def test_caps(pkg, dev, cap, x):
    """Scores of spread 2 under caps that hardly bend them, with and without a bias."""
    import torch
    q, k, v = _qkv(dev, x, 1, (1, 100, 4, 64), (1, 150, 2, 64))
    j, i = torch.arange(150, device=dev)[None], torch.arange(100, device=dev)[:, None] + 50
    _check(pkg.attention(q, k, v, 0.25, softcap=cap, causal=True), q, k, v, 0.25, cap, seen=j <= i)
    bias = torch.randn(4, 61, generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    got = pkg.attention(q, k, v, 0.25, softcap=cap, bias=bias, bias_zero=30)
    _check(got, q, k, v, 0.25, cap, bias=bias[:, (j - i + 30).clamp(0, 60)])


@pytest.mark.parametrize("cap", [65.0, 1e3, 1e6])
def test_caps_that_bend(pkg, dev, cap):
    """Scores as large as the cap: rows whose largest weights are near 1, and equal ones."""
    import torch
    q, k, v = _qkv(dev, "f16", 3, (1, 70, 2, 64), (1, 200, 2, 64))
    k = k / k.float().norm(dim=-1, keepdim=True)
    q = q / q.float().norm(dim=-1, keepdim=True)
    q, k = (q * 4).half(), (k * 4).half()
    scale = min(cap, 2000.0) / 16
    _check(pkg.attention(q, k, v, scale, softcap=cap), q, k, v, scale, cap)


@pytest.mark.parametrize("cap", [1e-3, 1e36, 1e38])
@pytest.mark.parametrize("scale", [1e-6, 0.125])
def test_caps_and_scales_at_the_ends(pkg, dev, cap, scale):
    q, k, v = _qkv(dev, "f16", 4, (1, 40, 2, 64), (1, 90, 2, 64), spread=0.125 / scale ** 0.5 if scale < 0.1 else 1.0)
    assert q.isfinite().all() and k.isfinite().all()
    _check(pkg.attention(q, k, v, scale, softcap=cap), q, k, v, scale, cap)


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("T", [1, 20, 100])
@pytest.mark.parametrize("cap", CAPS[1:])
def test_caps_over_a_cache(pkg, dev, cap, T, x):
    """A token, a few (both in parts) and a chunk in one piece: the same scores."""
    import torch
    n, Hq, Hk, D = 200, 8, 2, 64
    gen = torch.Generator(device=dev).manual_seed(5)
    k, v = (torch.randn(1, 1, Hk, 320, D, generator=gen, device=dev).to(_dt(x)) for _ in range(2))
    cache = pkg.KVCache.from_tensors(k, v, torch.tensor([[n], [n]], dtype=torch.int32, device=dev))
    q = torch.randn(1, T, Hq, D, generator=gen, device=dev).to(_dt(x))
    got = pkg.attention_cached(q, cache, 0, 0.25, softcap=cap)
    seen = torch.arange(n + T, device=dev)[None] <= n + torch.arange(T, device=dev)[:, None]
    keys, values = (t[0, :, :, :n + T].transpose(1, 2) for t in (k, v))
    _check(got, q, keys, values, 0.25, cap, seen=seen)
