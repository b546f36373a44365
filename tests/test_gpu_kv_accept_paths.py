"""Accepted paths that name a token more than once: every entry is a copy of it, and the
path ends at the capacity, whatever lies behind it in memory."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("D", [8, 72, 128])
def test_repeated_tokens(pkg, dev, D, weights):
    import torch
    L, Hk, C, lengths = 2, 2, 40, [30, 38, 39, 40, 0]
    B = len(lengths)
    gen = torch.Generator(device=dev).manual_seed(D)
    k, v = (torch.randn(L, B, Hk, C, D, generator=gen, device=dev).half() for _ in range(2))
    counts = torch.tensor([lengths, [n + 3 for n in lengths]], dtype=torch.int32, device=dev)
    more = {}
    if weights:
        more = dict(weight=torch.rand(L, B, Hk, C, generator=gen, device=dev),
                    position=torch.arange(C, dtype=torch.int32, device=dev).repeat(L, B, Hk, 1))
    cache = pkg.KVCache.from_tensors(k, v, counts, **more)
    path = torch.zeros(B, 64, dtype=torch.int32, device=dev)
    path[:, 1::3] = 1                        # 0 1 0 0 1 0 ...: 64 entries of two tokens
    path[4, 45:] = 63                        # past the capacity
    taken = [10, 2, 1, 0, 40]                # 39 + 1 and 40 + 0 have no slot
    tensors = (cache.k, cache.v) + tuple(more.values())
    before = [t.clone() for t in tensors]
    pkg.kv_accept(cache, 64, path=path)
    line = path.tolist()
    for old, new in zip(before, tensors):
        want = old.clone()
        for b, n in enumerate(lengths):
            want[:, b, :, n:n + taken[b]] = old[:, b, :, [n + t for t in line[b][:taken[b]]]]
        assert torch.equal(new, want)
    assert cache.length.tolist() == [n + m for n, m in zip(lengths, taken)]
    assert cache.next_position.tolist() == [n + 3 + m for n, m in zip(lengths, taken)]
