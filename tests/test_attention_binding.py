"""The native marshalling of the attention and cache calls: it declines whatever is
not the plain accepted call, and gives the ctypes route's results bit for bit."""
import ctypes

import pytest


@pytest.fixture
def native(pkg):
    if not pkg._native_tried:
        pkg._load_binding()
    assert pkg._native is not None, "lib/_q4_binding.*.so is not built"
    return pkg._native


def test_declines_host_tensors_and_wrong_arguments(pkg, native):
    import torch
    x = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    c = pkg.CKVCache(0, 0, 0, 0, 0, 0, 1, 1, 2, 64, 64, 0, 0, 0)
    h = (ctypes.addressof(c), 0)
    none = (None,) * 8
    assert native.attention(x, x, x, 1.0, 0.0, None, 0, False, *none[:7]) is None
    assert native.attention(None, x, x, 1.0, 0.0, None, 0, False, *none[:7]) is None
    assert native.attention(x, x) is None
    assert native.attention_cached(x, *h, 0, 0, 1.0, 0.0, None, 0, None, None) is None
    assert native.attention_cached(x, 0, 0, 0, 0, 1.0, 0.0, None, 0, None, None) is None
    assert native.kv_append(x, x, x, *h, 0, None, None, False, None, None) is None
    assert native.kv_accept("c", 0, 4, None, None, None) is None
    assert native.kv_evict(*h, 8, 1.0, 2, None) is None


def _run(pkg, dev, out):
    """Every call on fresh inputs; the results in order."""
    import torch
    gen = torch.Generator(device=dev).manual_seed(3)
    B, T, Hq, Hk, D = 2, 5, 4, 2, 64
    x = torch.randn(B, T, Hq + 2 * Hk, D, generator=gen, device=dev).half()
    q, k, v = x[:, :, :Hq], x[:, :, Hq:Hq + Hk], x[:, :, Hq + Hk:]
    lens = torch.tensor([5, 3], dtype=torch.int32, device=dev)
    docs = torch.tensor([[0, 0, 1, 1, 1], [2, 2, 2, -1, 2]], dtype=torch.int32, device=dev)
    bias = torch.randn(Hq, 9, generator=gen, device=dev)
    new = lambda: torch.zeros_like(q.contiguous()) if out else None
    got = [pkg.attention(q, k, v, 0.2, out=new()),
           pkg.attention(q, k, v, 0.2, softcap=9.0, bias=bias, bias_zero=4, causal=True, prefix=lens, q_docs=docs,
                         k_docs=docs, q_lens=lens, k_lens=lens, out=new())]
    kc, vc = (torch.randn(2, B, Hk, 40, D, generator=gen, device=dev).half() for _ in range(2))
    counts = torch.tensor([[20, 7], [30, 7]], dtype=torch.int32, device=dev)
    cache = pkg.KVCache.from_tensors(kc, vc, counts, weight=torch.rand(2, B, Hk, 40, generator=gen, device=dev),
                                     position=torch.arange(40, dtype=torch.int32, device=dev).repeat(2, B, Hk, 1))
    tree, depth = pkg.tree_masks([[-1, 0, 0, 1, 1]] * 2, device=dev)
    for layer in range(2):
        r = pkg.kv_append(q, k, v, cache, layer, pkg.rope_inv_freq(D, device=dev), depth=depth, q_out=new())
        got += [r, pkg.attention_cached(r, cache, layer, 0.2, tree=tree, weight_rows=2, out=new()),
                pkg.attention_cached(r, cache, layer, 0.2, softcap=4.0, out=new())]
    pkg.kv_accept(cache, 5, path=torch.tensor([[0, 2], [0, 1]], dtype=torch.int32, device=dev), count=lens - 3)
    got.append(counts.clone())
    pkg.kv_accept(cache, 1)
    pkg.kv_evict(cache, 16, sinks=1, recent=4)
    torch.cuda.synchronize()
    return got + [counts, kc, vc, cache.weight, cache.position]


@pytest.mark.gpu
@pytest.mark.parametrize("out", [False, True])
def test_same_results_as_ctypes(pkg, dev, native, out, monkeypatch):
    import torch
    made = dict.fromkeys(("attention", "attention_cached", "kv_append", "kv_accept", "kv_evict"), 0)

    class Counting:
        def __getattr__(self, name):
            def f(*a):
                r = getattr(native, name)(*a)
                made[name] += r is not None
                return r
            return f

    monkeypatch.setattr(pkg, "_native", Counting())
    got = _run(pkg, dev, out)
    assert all(made.values()), made
    monkeypatch.setattr(pkg, "_native", None)
    want = _run(pkg, dev, out)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_errors_are_the_librarys(pkg, dev, native):
    import torch
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16, device=dev)
    for kw in (dict(prefix=torch.zeros(1, dtype=torch.int32, device=dev)), dict(softcap=-1.0)):
        with pytest.raises(pkg.SltxError):
            pkg.attention(q, q, q, 1.0, **kw)
    with pytest.raises(pkg.SltxError):
        pkg.attention(q, q, q, 0.0)
    with pytest.raises(pkg.SltxError, match="overlaps"):
        pkg.attention(q, q, q, 1.0, out=q)
    with pytest.raises(ValueError, match="dtype"):
        pkg.attention(q, q.bfloat16(), q, 1.0)
    with pytest.raises(ValueError, match="shape"):
        pkg.attention(q, q[:, :3], q, 1.0)
    with pytest.raises(ValueError, match="device tensor"):
        pkg.attention(q, q, q, 1.0, q_docs=torch.zeros(1, 4, dtype=torch.int32))
    cache = pkg.KVCache(1, 1, 2, 16, 64, device=dev)
    with pytest.raises(pkg.SltxError, match="layer"):
        pkg.attention_cached(q, cache, 1, 1.0)
    with pytest.raises(pkg.SltxError, match="no weight"):
        pkg.attention_cached(q, cache, 0, 1.0, weight_rows=1)
    with pytest.raises(pkg.SltxError, match="no weight"):
        pkg.kv_evict(cache, 8)
    with pytest.raises(ValueError, match="shape"):
        pkg.kv_append(q, q[:, :, :1], q, cache, 0)
    with pytest.raises(pkg.SltxError, match="budget"):
        pkg.kv_evict(pkg.KVCache(1, 1, 2, 16, 64, track_weights=True, device=dev), 17)
    torch.cuda.synchronize()
