"""Calls of the attention operators with tensors of no elements, whose addresses torch
gives as null."""
import pytest

pytestmark = pytest.mark.gpu


def _cache(pkg, dev, B=2):
    import torch
    gen = torch.Generator(device=dev).manual_seed(0)
    k, v = (torch.randn(2, B, 2, 64, 64, generator=gen, device=dev).half() for _ in range(2))
    counts = torch.tensor([[10, 20], [12, 20]], dtype=torch.int32, device=dev)[:, :B].contiguous()
    return pkg.KVCache.from_tensors(k, v, counts)


def test_accept_of_an_empty_path(pkg, dev):
    """No token is on the path: none is accepted."""
    import torch
    cache = _cache(pkg, dev)
    before = [t.clone() for t in (cache.k, cache.v, cache.counts)]
    path = torch.zeros(2, 0, dtype=torch.int32, device=dev)
    pkg.kv_accept(cache, 5, path=path)
    pkg.kv_accept(cache, 5, path=path, count=torch.tensor([3, 1], dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    for t, old in zip((cache.k, cache.v, cache.counts), before):
        assert torch.equal(t, old)
    with pytest.raises(ValueError, match="shape"):
        pkg.kv_accept(cache, 5, path=path[:1])
    with pytest.raises(pkg.SltxError, match="drafted"):
        pkg.kv_accept(cache, -1, path=path)


@pytest.mark.parametrize("causal", [False, True])
def test_documents_of_no_keys(pkg, dev, causal):
    """No keys, with documents: every row sees nothing."""
    import torch
    q = torch.randn(2, 5, 4, 64, device=dev).half()
    k = torch.zeros(2, 0, 2, 64, dtype=torch.float16, device=dev)
    q_docs = torch.zeros(2, 5, dtype=torch.int32, device=dev)
    k_docs = torch.zeros(2, 0, dtype=torch.int32, device=dev)
    out = torch.full_like(q, 3.0)
    assert pkg.attention(q, k, k, 0.1, q_docs=q_docs, k_docs=k_docs, causal=causal, out=out) is out
    assert (out == 0).all()
    with pytest.raises(pkg.SltxError, match="go together"):
        pkg.attention(q, k, k, 0.1, k_docs=k_docs)
    with pytest.raises(pkg.SltxError, match="go together"):
        pkg.attention(q, k, k, 0.1, q_docs=q_docs)


@pytest.mark.parametrize("heads", [1, 4])
def test_bias_of_no_distances(pkg, dev, heads):
    import torch
    q = torch.randn(1, 5, 4, 64, device=dev).half()
    with pytest.raises(ValueError, match="bias"):
        pkg.attention(q, q, q, 0.1, bias=torch.zeros(heads, 0, device=dev))
