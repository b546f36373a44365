"""Masks written as a bias of -inf or of a type's lowest value, beside ordinary biases,
against the bounds of attn_bounds.py."""
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


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["-inf", "lowest", "lowest of fp16"])
def test_windows(pkg, dev, kind, x):
    """A window of distances, the rest masked by a bias: what is masked has no weight,
    beside ordinary biases too."""
    import torch
    q, k, v = _qkv(dev, x, 7, (1, 200, 2, 64), (1, 333, 1, 64))
    low = {"-inf": -math.inf, "lowest": torch.finfo(torch.float32).min, "lowest of fp16": -65504.0}[kind]
    bias = torch.randn(2, 81, generator=torch.Generator(device=dev).manual_seed(8), device=dev)
    bias[:, :20] = low
    bias[:, 60:] = low
    j, i = torch.arange(333, device=dev)[None], torch.arange(200, device=dev)[:, None] + 133
    at = (j - i + 40).clamp(0, 80)
    seen = torch.ones(200, 333, dtype=torch.bool, device=dev)
    for causal in (False, True):
        for cap in (0.0, 20.0):
            got = pkg.attention(q, k, v, 0.2, softcap=cap, bias=bias, bias_zero=40, causal=causal)
            _check(got, q, k, v, 0.2, cap, bias=bias[:, at], seen=seen & (j <= i) if causal else seen, what=kind)
    # every distance but one masked: a row is the value of one key
    one = torch.full((1, 5), low, device=dev)
    one[0, 2] = 0.0
    got = pkg.attention(q, k, v, 0.2, bias=one, bias_zero=2)
    assert torch.equal(got, v[:, 133:].expand(1, 200, 2, 64))
