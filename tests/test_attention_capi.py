"""Refusals of the attention and cache entry points, checked on the CPU: argument
validation runs before any HIP call, with pointers that are never read."""
import ctypes

import pytest

A = 0x1000000          # aligned; never dereferenced
FAR = 0x4000000000


def _args(pkg, **kw):
    d = dict(q=A, k=A + 0x100000, v=A + 0x200000, out=FAR, dtype=0, batch=1, q_rows=4, k_rows=4, q_heads=4,
             kv_heads=2, head_dim=64, causal=0, scale=0.125, softcap=0.0)
    heads = kw.get("q_heads", 4)
    d.update(q_stride=(4 * heads * 64, heads * 64, 64), k_stride=(512, 128, 64), v_stride=(512, 128, 64),
             out_stride=(4 * heads * 64, heads * 64, 64))
    d.update(kw)
    a = pkg.CAttentionArgs()
    for n, x in d.items():
        setattr(a, n, (ctypes.c_int64 * 3)(*x) if n.endswith("_stride") and n != "bias_head_stride" else x)
    return a


@pytest.mark.parametrize("kw,code,frag", [
    (dict(dtype=2), -1, "dtype"),
    (dict(dtype=7), -1, "dtype"),
    (dict(q_heads=3), -1, "not a multiple"),
    (dict(q_heads=0), -1, "not a multiple"),
    (dict(kv_heads=0), -1, "not a multiple"),
    (dict(head_dim=0), -1, "head_dim"),
    (dict(head_dim=20), -1, "multiple of 8"),
    (dict(head_dim=136), -2, "above 128"),
    (dict(scale=0.0), -1, "scale"),
    (dict(scale=-1.0), -1, "scale"),
    (dict(scale=float("nan")), -1, "scale"),
    (dict(scale=float("inf")), -1, "scale"),
    (dict(softcap=-1.0), -1, "softcap"),
    (dict(softcap=float("nan")), -1, "softcap"),
    (dict(batch=-1), -1, "batch"),
    (dict(q_rows=-1), -1, "rows"),
    (dict(k_rows=-1), -1, "keys"),
    (dict(q_rows=(1 << 28) + 1), -2, "2^28"),
    (dict(q=0), -1, "q is null"),
    (dict(k=0), -1, "k is null"),
    (dict(v=0), -1, "v is null"),
    (dict(out=0), -1, "out is null"),
    (dict(q=A + 8), -1, "16-byte"),
    (dict(k=A + 2), -1, "16-byte"),
    (dict(out=FAR + 4), -1, "16-byte"),
    (dict(q_stride=(1024, 257, 64)), -1, "stride"),
    (dict(k_stride=(512, -128, 64)), -1, "stride"),
    (dict(k_stride=(512, 1 << 24, 64)), -2, "row stride"),
    (dict(out=A), -1, "overlaps"),
    (dict(out=A + 0x100000), -1, "overlaps"),
    (dict(out_stride=(1024, 256, 0)), -1, "overlap each other"),
    (dict(out_stride=(1024, 0, 64)), -1, "overlap each other"),
    (dict(out_stride=(1024, 64, 64)), -1, "overlap each other"),
    (dict(out_stride=(64, 256, 64), batch=2), -1, "overlap each other"),
    (dict(softcap=1e-38, scale=8.0), -2, "fp32's range"),
    (dict(softcap=2e38), -2, "fp32's range"),
    (dict(scale=3e38), -2, "fp32's range"),
    (dict(bias=FAR, bias_len=(1 << 30) + 1, bias_zero=0), -2, "distances"),
    (dict(bias=A, bias_len=0), -1, "bias"),
    (dict(bias=A, bias_len=5, bias_zero=5), -1, "bias"),
    (dict(bias=A, bias_len=5, bias_zero=-1), -1, "bias"),
    (dict(bias=A + 1, bias_len=5), -1, "misaligned"),
    (dict(prefix=A), -1, "prefix needs causal"),
    (dict(q_docs=A), -1, "go together"),
    (dict(k_docs=A), -1, "go together"),
    (dict(q_lens=A + 2), -1, "misaligned"),
])
def test_attention(pkg, kw, code, frag):
    a = _args(pkg, **kw)
    assert pkg.lib().sltx_attention(ctypes.byref(a), None) == code
    assert frag in pkg.last_error() and "sltx_attention" in pkg.last_error()


def test_attention_nothing_to_do(pkg):
    L = pkg.lib()
    assert L.sltx_attention(None, None) == -1
    for kw in (dict(batch=0), dict(q_rows=0)):
        a = _args(pkg, q=0, k=0, v=0, out=0, **kw)
        assert L.sltx_attention(ctypes.byref(a), None) == 0


def _cache(pkg, **kw):
    d = dict(k=A, v=A + 0x8000000, weight=A, position=A, length=A, next_position=A, layers=2, batch=3, kv_heads=2,
             capacity=256, head_dim=64, dtype=0, workspace=A, workspace_bytes=1 << 30)
    d.update(kw)
    c = pkg.CKVCache()
    for n, x in d.items():
        setattr(c, n, x)
    return c


S3 = (ctypes.c_int64 * 3)(4 * 256, 256, 64)

CACHES = [
    (dict(layers=0), -1, "layers"),
    (dict(batch=-1), -1, "batch"),
    (dict(capacity=0), -1, "capacity"),
    (dict(capacity=(1 << 28) + 1), -2, "slots"),
    (dict(layers=40, batch=900), -2, "layers"),
    (dict(kv_heads=0), -1, "heads"),
    (dict(head_dim=12), -1, "head_dim"),
    (dict(head_dim=256), -2, "head_dim"),
    (dict(dtype=2), -1, "dtype"),
    (dict(k=0), -1, "null"),
    (dict(length=0), -1, "null"),
    (dict(next_position=0), -1, "null"),
    (dict(v=A + 8), -1, "misaligned"),
    (dict(length=A + 2), -1, "misaligned"),
    (dict(workspace=A + 4), -1, "misaligned"),
    (dict(weight=0), -1, "go together"),
    (dict(position=0), -1, "go together"),
]


def _cached(pkg, c, q=FAR, stride=S3, layer=0, tokens=4, heads=4, scale=0.1, cap=0.0, tree=None, rows=0, out=FAR * 2,
            first=0):
    return pkg.lib().sltx_attention_cached(q, stride, ctypes.byref(c) if c else None, layer, first, tokens, heads,
                                           scale, cap, tree, rows, out, None)


def _append(pkg, c, q=FAR, k=FAR, v=FAR, stride=S3, layer=0, tokens=4, heads=4, freq=A, pairs=32, depth=None,
            out=FAR * 2):
    return pkg.lib().sltx_kv_append(q, stride, k, stride, v, stride, ctypes.byref(c) if c else None, layer, tokens,
                                    heads, freq, pairs, 0, depth, out, None)


def _accept(pkg, c, drafted=4, path=A, n=4, count=None):
    return pkg.lib().sltx_kv_accept(ctypes.byref(c) if c else None, drafted, path, n, count, None)


def _evict(pkg, c, budget=64, sinks=4, recent=8):
    return pkg.lib().sltx_kv_evict(ctypes.byref(c) if c else None, budget, sinks, recent, None)


@pytest.mark.parametrize("call", [_cached, _append, _accept, _evict])
@pytest.mark.parametrize("kw,code,frag", CACHES)
def test_bad_caches(pkg, call, kw, code, frag):
    assert call(pkg, _cache(pkg, **kw)) == code
    assert frag in pkg.last_error()


@pytest.mark.parametrize("call", [_cached, _append, _accept, _evict])
def test_no_cache_and_empty_cache(pkg, call):
    assert call(pkg, None) == -1 and "cache is null" in pkg.last_error()
    assert call(pkg, _cache(pkg, batch=0, k=0, v=0, weight=0, position=0, length=0, next_position=0)) == 0


@pytest.mark.parametrize("kw,code,frag", [
    (dict(layer=2), -1, "layer"),
    (dict(layer=-1), -1, "layer"),
    (dict(tokens=-1), -1, "tokens"),
    (dict(first=-1), -1, "first"),
    (dict(tokens=1 << 28), -2, "query heads for each"),
    (dict(heads=5), -1, "not a multiple"),
    (dict(scale=0.0), -1, "scale"),
    (dict(cap=-1.0), -1, "softcap"),
    (dict(cap=1e-38, scale=8.0), -2, "fp32's range"),
    (dict(tokens=65, tree=A), -1, "tree"),
    (dict(tree=A + 4), -1, "tree"),
    (dict(rows=5), -1, "weights"),
    (dict(rows=-1), -1, "weights"),
    (dict(tokens=65, rows=1), -2, "weights"),
    (dict(q=0), -1, "q is null"),
    (dict(q=FAR + 2), -1, "16-byte"),
    (dict(out=0), -1, "out is null"),
    (dict(out=FAR), -1, "overlaps"),
    (dict(out=A), -1, "overlaps"),
    (dict(stride=None), -1, "q_stride"),
    (dict(stride=(ctypes.c_int64 * 3)(1024, 256, 60)), -1, "stride"),
])
def test_attention_cached(pkg, kw, code, frag):
    assert _cached(pkg, _cache(pkg), **kw) == code
    assert frag in pkg.last_error()


def test_attention_cached_workspace(pkg):
    L = pkg.lib()
    c = _cache(pkg, workspace=0, workspace_bytes=1 << 30, capacity=4096)
    need = L.sltx_attention_cached_workspace(ctypes.byref(c), 1, 4, 0)
    assert need > 0
    assert _cached(pkg, c, tokens=1) == -1 and f"{need} needed" in pkg.last_error()
    c = _cache(pkg, workspace_bytes=need - 1, capacity=4096)
    assert _cached(pkg, c, tokens=1) == -1 and f"{need} needed" in pkg.last_error()
    assert _cached(pkg, _cache(pkg, weight=0, position=0), rows=1) == -1 and "no weight" in pkg.last_error()
    assert L.sltx_attention_cached_workspace(ctypes.byref(c), -1, 4, 0) == -1
    assert L.sltx_attention_cached_workspace(ctypes.byref(c), 1, 5, 0) == -1
    assert L.sltx_attention_cached_workspace(None, 1, 4, 0) == -1
    assert L.sltx_attention_cached_workspace(ctypes.byref(c), 0, 4, 0) == 0
    assert _cached(pkg, _cache(pkg), tokens=0, q=0, out=0) == 0


@pytest.mark.parametrize("kw,code,frag", [
    (dict(layer=2), -1, "layer"),
    (dict(tokens=-1), -1, "tokens"),
    (dict(heads=3), -1, "not a multiple"),
    (dict(pairs=33), -1, "pairs"),
    (dict(pairs=-1), -1, "pairs"),
    (dict(freq=0), -1, "inv_freq"),
    (dict(freq=A + 1), -1, "inv_freq"),
    (dict(depth=A + 2), -1, "depth"),
    (dict(q=0), -1, "q is null"),
    (dict(k=0), -1, "k is null"),
    (dict(v=FAR + 8), -1, "16-byte"),
    (dict(out=0), -1, "q_out is null"),
    (dict(out=FAR), -1, "overlaps"),
    (dict(out=A), -1, "overlaps the cache"),
    (dict(k=A), -1, "overlaps the cache"),
    (dict(stride=None), -1, "stride"),
])
def test_append(pkg, kw, code, frag):
    assert _append(pkg, _cache(pkg), **kw) == code
    assert frag in pkg.last_error()


def test_accept(pkg):
    c = _cache(pkg)
    for kw, frag in ((dict(drafted=-1), "drafted"), (dict(n=65), "path"), (dict(n=-1), "path"),
                     (dict(path=A + 2), "misaligned"), (dict(count=A + 1), "misaligned")):
        assert _accept(pkg, c, **kw) == -1 and frag in pkg.last_error()
    assert _accept(pkg, c, drafted=0) == 0 and _accept(pkg, c, n=0) == 0


def test_evict(pkg):
    L = pkg.lib()
    for kw, frag in ((dict(budget=0), "budget"), (dict(budget=257), "budget"), (dict(sinks=-1), "positions"),
                     (dict(recent=-1), "positions"), (dict(sinks=60, recent=5), "positions"),
                     (dict(sinks=1, recent=2**31 - 1), "positions")):
        assert _evict(pkg, _cache(pkg), **kw) == -1 and frag in pkg.last_error()
    assert _evict(pkg, _cache(pkg, weight=0, position=0)) == -1 and "no weight" in pkg.last_error()
    c = _cache(pkg, workspace_bytes=0)
    need = L.sltx_kv_evict_workspace(ctypes.byref(c), 64)
    assert need > 0
    assert _evict(pkg, c) == -1 and f"{need} needed" in pkg.last_error()
    assert L.sltx_kv_evict_workspace(ctypes.byref(c), 0) == -1
    assert L.sltx_kv_evict_workspace(None, 4) == -1


def test_python_checks(pkg):
    """Tensors that the kernels must never see are refused before the library is called."""
    torch = pytest.importorskip("torch")
    q = torch.zeros(1, 4, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensor"):
        pkg.attention(q, q, q, 1.0)
    with pytest.raises(ValueError, match="dtype"):
        pkg.attention(q.float(), q, q, 1.0)
    with pytest.raises(ValueError, match="batch, rows"):
        pkg.attention(q[0], q, q, 1.0)
    with pytest.raises(ValueError, match="device tensor"):
        pkg.KVCache.from_tensors(*(torch.zeros(1, 1, 2, 8, 64, dtype=torch.float16) for _ in range(2)),
                                 torch.zeros(2, 1, dtype=torch.int32))


def test_tree_masks(pkg):
    torch = pytest.importorskip("torch")
    tree, depth = pkg.tree_masks([[-1, 0, 0, 1, 3], [-1, -1, 1, 2, 0]], device="cpu")
    assert tree.tolist() == [[1, 3, 5, 11, 27], [1, 2, 6, 14, 17]]
    assert depth.tolist() == [[0, 1, 1, 2, 3], [0, 0, 1, 2, 1]] and depth.dtype == torch.int32
    long, _ = pkg.tree_masks([[t - 1 for t in range(64)]], device="cpu")
    assert [x % 2 ** 64 for x in long[0].tolist()] == [2 ** (t + 1) - 1 for t in range(64)]
    for bad in ([[0]], [[-1, 1]], [[-2]], [[-1] * 65]):
        with pytest.raises(ValueError):
            pkg.tree_masks(bad, device="cpu")


def test_rope_frequencies(pkg):
    torch = pytest.importorskip("torch")
    f = pkg.rope_inv_freq(128, theta=500000.0, device="cpu")
    assert f.shape == (64,) and f[0] == 1.0 and abs(f[32].item() * 500000.0 ** 0.5 - 1) < 1e-6
    scaling = dict(rope_type="llama3", factor=32.0, low_freq_factor=1.0, high_freq_factor=4.0,
                   original_max_position_embeddings=8192)
    g = pkg.rope_inv_freq(128, theta=500000.0, scaling=scaling, device="cpu")
    wave = 2 * torch.pi / f.double()
    assert torch.equal(g[wave < 2048], f[wave < 2048])                     # short waves as they are
    assert torch.allclose(g[wave > 8192], f[wave > 8192] / 32, rtol=1e-6)  # long ones stretched
    assert ((g <= f) & (g >= f / 32.01)).all()
    assert torch.allclose(pkg.rope_inv_freq(64, scaling=dict(type="linear", factor=4.0), device="cpu"),
                          pkg.rope_inv_freq(64, device="cpu") / 4)
    with pytest.raises(ValueError):
        pkg.rope_inv_freq(64, scaling=dict(rope_type="other"), device="cpu")
