"""The bound of attn_bounds.py on the CPU: it holds for the kernels' arithmetic done
in torch, and rejects results that ignore a mask, lose a long tail or form a
capped score with an error that grows with the cap."""
import math

import pytest

import attn_bounds
import attn_ref as R


def _normal(seed, *shape, dtype):
    import torch
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _plain(q, k, v, scale, cap=0.0, bias=None, seen=None, top_weight=2.0 ** 8, fast_cap=False):
    """fp32 scores, weights rounded to the type against the row's largest."""
    import torch
    x = scale * (q.float() @ k.float().T)
    if cap and fast_cap:
        x = cap - 2 * cap / (1 + torch.exp(x * (2 / cap)))
    elif cap:
        x = cap * torch.tanh(x / cap)
    if bias is not None:
        x = x + bias.float()
    if seen is not None:
        x = torch.where(seen, x, -math.inf)
    top = x.amax(1, keepdim=True)
    w = torch.exp(x - torch.where(top > -math.inf, top, 0.0)) * top_weight
    w = w.to(q.dtype).float()
    total = w.sum(1, keepdim=True)
    return (w @ v.float() / torch.where(total == 0, 1.0, total)).to(q.dtype)


def _ok(got, ref, bound, dtype):
    try:
        R.check_out(got, ref, bound, dtype)
        return True
    except AssertionError:
        return False


@pytest.mark.parametrize("x", ["float16", "bfloat16"])
@pytest.mark.parametrize("kind", ["-inf", "lowest"])
def test_masks_written_as_a_bias(x, kind):
    import torch
    dt = getattr(torch, x)
    q, k, v = (_normal(i, 150, 64, dtype=dt) for i in range(3))
    i, j = torch.arange(150)[:, None], torch.arange(150)[None]
    low = -math.inf if kind == "-inf" else torch.finfo(torch.float32).min
    bias = torch.where((j - i).abs() < 20, 0.0, low)
    _, ref, bound = attn_bounds.head(q, k, v, 0.2, bias=bias)
    assert _ok(_plain(q, k, v, 0.2, bias=bias), ref, bound, dt)
    assert (bound < 0.1).all()
    for wrong in (torch.zeros_like(q), _plain(q, k, v, 0.2), -ref.to(dt), ref.to(dt) * 3):
        assert not _ok(wrong, ref, bound, dt)


@pytest.mark.parametrize("cap", [30.0, 64.0, 1e3, 1e4, 1e6, 1e8])
@pytest.mark.parametrize("x", ["float16", "bfloat16"])
def test_caps(x, cap):
    import torch
    dt = getattr(torch, x)
    q, k, v = (_normal(3 + i, 64, 64, dtype=dt) for i in range(3))
    _, ref, bound = attn_bounds.head(q, k, v, 0.25, cap)
    assert _ok(_plain(q, k, v, 0.25, cap), ref, bound, dt)
    good = _ok(_plain(q, k, v, 0.25, cap, fast_cap=True), ref, bound, dt)
    assert good if cap <= attn_bounds.FAST_CAP else not good or cap <= 1e4
    assert not _ok(_plain(q, k, v, 0.25, 3.0), ref, bound, dt)


def test_long_tail():
    import torch
    n = 20000
    q = torch.zeros(1, 64, dtype=torch.float16)
    k, v = torch.zeros(n, 64, dtype=torch.float16), torch.ones(n, 64, dtype=torch.float16)
    q[0, 0], k[0, 0], v[0] = 1.0, 15.4, 0.0
    _, ref, bound = attn_bounds.head(q, k, v, 1.0)
    assert _ok(_plain(q, k, v, 1.0), ref, bound, torch.float16)
    assert not _ok(_plain(q, k, v, 1.0, top_weight=2.0 ** -3), ref, bound, torch.float16)


def test_rows_that_see_nothing():
    import torch
    q, k, v = (_normal(9 + i, 20, 64, dtype=torch.float16) for i in range(3))
    seen = torch.arange(20)[:, None] > torch.arange(20)[None]
    v[19], k[19] = math.nan, math.inf      # no row sees the last key
    _, ref, bound = attn_bounds.head(q, k, v, 0.2, seen=seen)
    assert (ref[0] == 0).all() and bound.isfinite().all()
    assert _ok(_plain(q, torch.where(k.isfinite(), k, 0.0), torch.where(v.isfinite(), v, 0.0), 0.2, seen=seen), ref, bound,
               torch.float16)
