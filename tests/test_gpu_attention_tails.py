"""Attention whose weights differ widely: one key far above a long, flat tail, scores
that rise from key to key, against the bounds of attn_bounds.py."""
import math

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


def _tail(dev, x, n, at, drop, D=64):
    """n keys whose scores are `drop` below that of key `at`, whose value is 0, the others' 1."""
    import torch
    q = torch.zeros(1, 1, 1, D, device=dev)
    k, v = torch.zeros(1, n, 1, D, device=dev), torch.ones(1, n, 1, D, device=dev)
    q[..., 0] = 1.0
    k[0, at, 0, 0], v[0, at] = drop, 0.0
    return q.to(_dt(x)), k.to(_dt(x)), v.to(_dt(x))


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("drop", [12.0, 14.5, 15.4])
@pytest.mark.parametrize("at", [0, 10007, 19999])
def test_long_tails(pkg, dev, at, drop, x):
    q, k, v = _tail(dev, x, 20000, at, drop)
    got = pkg.attention(q, k, v, 1.0)
    _check(got, q, k, v, 1.0, what="attention")
    bias_got = pkg.attention(q, k, v, 1.0, bias=q.new_zeros(1, 1).float())
    _check(bias_got, q, k, v, 1.0, what="biased")


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("at", [0, 10007, 19999])
def test_long_tails_over_a_cache(pkg, dev, at, T, x):
    """The same in parts, with the weights that each key has: 2^-24 of the sums' terms and
    of the exponents (attn_bounds), the exponential's last place, 1 / l and its product."""
    import torch
    n, drop = 20000, 15.4
    q, k, v = _tail(dev, x, n, at, drop)
    kc, vc = (torch.zeros(1, 1, 1, n + 64, 64, dtype=_dt(x), device=dev) for _ in range(2))
    kc[0, 0, 0, :n], vc[0, 0, 0, :n] = k[0, :, 0], v[0, :, 0]
    weight = torch.zeros(1, 1, 1, n + 64, device=dev)
    cache = pkg.KVCache.from_tensors(kc, vc, torch.tensor([[n], [n]], dtype=torch.int32, device=dev), weight=weight,
                                     position=torch.zeros(1, 1, 1, n + 64, dtype=torch.int32, device=dev))
    qs = q.expand(1, T, 1, 64).contiguous()
    got = pkg.attention_cached(qs, cache, 0, 1.0, weight_rows=T)
    seen = torch.arange(n + T, device=dev)[None] <= n + torch.arange(T, device=dev)[:, None]
    p, ref, bound = attn_bounds.head(qs[0, :, 0], kc[0, 0, 0, :n + T], vc[0, 0, 0, :n + T], 1.0, seen=seen)
    R.check_out(got[0, :, 0], ref, bound, q.dtype)
    want = p.sum(0)
    # exponents up to 16: 2^-24 (68 * 16 + 10 * 16 + 64); the sum of n + T terms, each wave's by 32
    off = (math.expm1(2 * 2.0 ** -24 * (68 + 10 + 4) * 16) + ((n + T) / 32 + 64 + T) * 2.0 ** -23) * want
    assert ((weight[0, 0, 0, :n + T].double() - want).abs() <= off).all()


@pytest.mark.parametrize("x", ["f16", "bf16"])
def test_weights_of_equal_keys(pkg, dev, x):
    """As many equal weights as a row of tiles has, and one key that grows past them step
    by step: nothing overflows, and later maxima take over."""
    import torch
    q, k, v = _qkv(dev, x, 6, (1, 33, 1, 64), (1, 4000, 1, 64))
    _check(pkg.attention(torch.zeros_like(q), k, v, 1.0), torch.zeros_like(q), k, v, 1.0)
    q = torch.zeros_like(q)
    q[..., 0] = 1.0
    for step in (0.001, 0.004, 0.02):           # scores that rise from key to key
        k2 = torch.zeros_like(k)
        k2[0, :, 0, 0] = torch.arange(4000, device=dev) * step
        _check(pkg.attention(q, k2, v, 1.0), q, k2, v, 1.0, what=f"rising by {step}")
        _check(pkg.attention(q, k2.flip(1).contiguous(), v, 1.0), q, k2.flip(1).contiguous(), v, 1.0, what="falling")
