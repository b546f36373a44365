"""Keys and values whose rows overlap in memory (a row stride below head_dim), up to the
end of their memory, with infinities and NaN in the last of them."""
import math

import pytest

import attn_bounds
import attn_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("stride", [8, 24])
@pytest.mark.parametrize("B,Hq", [(1, 2), (26, 32)], ids=["blocks of 64", "blocks of 128"])
def test_overlapping_rows(pkg, dev, B, Hq, stride, D, x):
    import torch
    dt, S = getattr(torch, x), 133
    gen = torch.Generator(device=dev).manual_seed(stride + D)
    base = torch.randn(2, (S - 1) * stride + D, generator=gen, device=dev).to(dt)
    view = lambda t: t.as_strided((B, S, 1, D), (0, stride, 0, 1), t.storage_offset())
    k, v = view(base[0].clone()), view(base[1].clone())
    q = torch.randn(B, S, Hq, D, generator=gen, device=dev).to(dt)
    clean = pkg.attention(q, k, v, 0.1, causal=True)
    seen = torch.ones(S, S, dtype=torch.bool, device=dev).tril()
    for b, h in ((0, 0), (B - 1, Hq - 1)):
        _, ref, bound = attn_bounds.head(q[b, :, h], k[b, :, 0], v[b, :, 0], 0.1, seen=seen)
        R.check_out(clean[b, :, h], ref, bound, dt)
    for bad in (math.inf, math.nan):
        flat = base[1].clone()
        flat[-4] = bad                     # of the last key's row only
        got = pkg.attention(q, k, view(flat), 0.1, causal=True)
        assert torch.equal(got[:, :-1], clean[:, :-1])
        hit = got[:, -1, :, D - 4]
        assert hit.isnan().all() if bad != bad else (hit == math.inf).all()
        keep = torch.arange(D, device=dev) != D - 4
        assert torch.equal(got[:, -1][..., keep], clean[:, -1][..., keep])
