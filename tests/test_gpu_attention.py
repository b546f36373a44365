"""sltx_attention against plain attention in 64 bits (attn_ref.py derives the
bounds): every mask, odd sizes around the tiles' edges, strides, masked places
that hold infinities and NaN, rows that see nothing, other streams, graphs."""
import math

import pytest

import attn_ref as R

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def _qkv(dev, B, Sq, Sk, Hq, Hk, D, x, seed=0, spread=1.0):
    import torch
    gen = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda *s: (torch.randn(*s, generator=gen, device=dev) * spread).to(_dt(x))
    return mk(B, Sq, Hq, D), mk(B, Sk, Hk, D), mk(B, Sk, Hk, D)


def _seen(b, Sq, Sk, dev, causal=False, prefix=None, q_docs=None, k_docs=None, q_lens=None, k_lens=None):
    import torch
    m = Sq if q_lens is None else min(max(int(q_lens[b]), 0), Sq)
    n = Sk if k_lens is None else min(max(int(k_lens[b]), 0), Sk)
    i, j = torch.arange(Sq, device=dev)[:, None], torch.arange(Sk, device=dev)[None]
    seen = (j < n).expand(Sq, Sk)
    if causal:
        near = j <= i + n - m
        if prefix is not None:
            near = near | (j < int(prefix[b]))
        seen = seen & near
    if q_docs is not None:
        seen = seen & (q_docs[b][:, None] == k_docs[b][None]) & (q_docs[b][:, None] >= 0)
    return seen, m, n


def _check(pkg, dev, q, k, v, scale, *, softcap=0.0, bias=None, bias_zero=0, out=None, stream=None, what="", **masks):
    import torch
    got = pkg.attention(q, k, v, scale, softcap=softcap, bias=bias, bias_zero=bias_zero, out=out, stream=stream, **masks)
    torch.cuda.synchronize()
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1:3]
    for b in range(B):
        seen, m, n = _seen(b, Sq, Sk, dev, **masks)
        if bias is not None:
            far = torch.arange(Sk, device=dev)[None] - (torch.arange(Sq, device=dev)[:, None] + n - m)
            at = (far + bias_zero).clamp(0, bias.shape[1] - 1)
        for h in range(Hq):
            g = h // (Hq // Hk)
            hb = None if bias is None else bias[h if bias.shape[0] > 1 else 0][at]
            _, ref, _, bound = R.head(q[b, :, h], k[b, :, g], v[b, :, g], scale, softcap, hb, seen)
            R.check_out(got[b, :m, h], ref[:m], bound[:m], q.dtype, f"{what} sequence {b} head {h}")
    return got


SIZES = [  # B, Sq, Sk, Hq, Hk, D
    (1, 1, 1, 1, 1, 64),
    (2, 1, 65, 4, 1, 128),
    (1, 31, 64, 2, 2, 8),
    (1, 33, 63, 3, 1, 40),
    (3, 127, 129, 2, 1, 64),
    (1, 129, 128, 6, 2, 128),
    (2, 200, 191, 4, 4, 72),
    (1, 257, 640, 2, 1, 80),
    (1, 5, 1000, 8, 1, 120),
]


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(pkg, dev, size, causal, x):
    q, k, v = _qkv(dev, *size, x, seed=sum(size))
    # fewer keys than rows under a causal mask: the first rows see nothing
    _check(pkg, dev, q, k, v, 1.5 / math.sqrt(size[-1]), causal=causal)


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("cap", [5.0, 50.0])
def test_softcap(pkg, dev, cap, x):
    q, k, v = _qkv(dev, 1, 100, 150, 4, 2, 64, x, seed=3, spread=3.0)
    _check(pkg, dev, q, k, v, 0.2, softcap=cap, causal=True)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("n,zero", [(1, 0), (9, 4), (65, 60), (401, 200)])
def test_distance_bias(pkg, dev, n, zero, shared):
    import torch
    q, k, v = _qkv(dev, 2, 90, 150, 4, 2, 64, "f16", seed=n)
    gen = torch.Generator(device=dev).manual_seed(n)
    bias = torch.randn(1 if shared else 4, n, generator=gen, device=dev) * 3
    lens = dict(q_lens=torch.tensor([90, 50], dtype=torch.int32, device=dev),
                k_lens=torch.tensor([150, 70], dtype=torch.int32, device=dev))
    _check(pkg, dev, q, k, v, 0.1, bias=bias, bias_zero=zero)
    _check(pkg, dev, q, k, v, 0.1, bias=bias, bias_zero=zero, causal=True, softcap=20.0, **lens)


def test_bias_of_minus_infinity_and_lowest(pkg, dev):
    """-inf masks a distance; the type's lowest value everywhere leaves equal weights."""
    import torch
    q, k, v = _qkv(dev, 1, 150, 150, 2, 1, 64, "f16", seed=8)
    window = torch.zeros(1, 41, device=dev)
    window[0, 0] = window[0, -1] = -math.inf              # keys within 19 of the row
    _check(pkg, dev, q, k, v, 0.2, bias=window, bias_zero=20)
    _check(pkg, dev, q, k, v, 0.2, bias=torch.full((1, 1), -math.inf, device=dev))   # nothing is left
    low = torch.full((1, 1), torch.finfo(torch.float32).min, device=dev)
    got = pkg.attention(q, k, v, 0.2, bias=low)
    ref = v.double().mean(1, keepdim=True).expand(1, 150, 1, 64).repeat_interleave(2, 2)
    R.check_out(got, ref, torch.full_like(ref, 150 * 2.0 ** -24 * 4), q.dtype)   # sums of exact weights 1
    # some distances at the lowest value, as masks are often written
    mask = torch.zeros(2, 301, device=dev)
    mask[:, :150] = torch.finfo(torch.float32).min
    _check(pkg, dev, q, k, v, 0.2, bias=mask, bias_zero=150)


@pytest.mark.parametrize("x", ["f16", "bf16"])
def test_prefix(pkg, dev, x):
    import torch
    q, k, v = _qkv(dev, 4, 150, 150, 2, 2, 64, x, seed=5)
    prefix = torch.tensor([0, 1, 100, 1000], dtype=torch.int32, device=dev)
    _check(pkg, dev, q, k, v, 0.2, causal=True, prefix=prefix)
    lens = torch.tensor([150, 0, 120, 3], dtype=torch.int32, device=dev)
    _check(pkg, dev, q, k, v, 0.2, causal=True, prefix=prefix, q_lens=lens, k_lens=lens)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_documents(pkg, dev, causal, D):
    import torch
    S = 700
    q, k, v = _qkv(dev, 3, S, S, 4, 2, D, "bf16", seed=6)
    docs = torch.zeros(3, S, dtype=torch.int32)
    docs[0] = torch.arange(S) // 130                      # packed, ends inside tiles
    docs[0, 690:] = -1                                    # padding sees nothing
    docs[1] = torch.randint(0, 3, (S,), generator=torch.Generator().manual_seed(1))   # mixed
    docs[2] = 7
    docs[2, ::2] = -5                                     # ids below 0 are of no document
    docs = docs.to(dev)
    got = _check(pkg, dev, q, k, v, 0.2, causal=causal, q_docs=docs, k_docs=docs, softcap=15.0)
    assert (got[0, 690:] == 0).all()


def test_rows_of_no_document(pkg, dev):
    """Rows without a document among rows that see whole tiles of keys."""
    import torch
    q, k, v = _qkv(dev, 1, 200, 320, 2, 1, 64, "f16", seed=16)
    q_docs = torch.full((1, 200), 3, dtype=torch.int32, device=dev)
    q_docs[0, [0, 40, 100, 199]] = -1
    k_docs = torch.full((1, 320), 3, dtype=torch.int32, device=dev)
    for causal in (False, True):
        got = _check(pkg, dev, q, k, v, 0.2, q_docs=q_docs, k_docs=k_docs, causal=causal)
        assert (got[0, [0, 40, 100, 199]] == 0).all()


def test_documents_of_other_keys(pkg, dev):
    """Rows and keys with ids of their own, over more than 64 tiles of keys."""
    import torch
    q, k, v = _qkv(dev, 1, 40, 9000, 2, 1, 64, "f16", seed=7)
    q_docs = (torch.arange(40, device=dev) // 8 * 3).to(torch.int32)[None]
    k_docs = (torch.arange(9000, device=dev) // 640).to(torch.int32)[None]
    _check(pkg, dev, q, k, v, 0.2, q_docs=q_docs, k_docs=k_docs)
    far = torch.full((1, 9000), 99, dtype=torch.int32, device=dev)
    assert (pkg.attention(q, k, v, 0.2, q_docs=q_docs, k_docs=far) == 0).all()


def test_lengths(pkg, dev):
    """Padded sequences: keys behind the length are not seen, rows behind it keep
    what `out` held; lengths beyond the tensors are cut, negative ones are 0."""
    import torch
    q, k, v = _qkv(dev, 5, 100, 170, 4, 2, 64, "f16", seed=9)
    q_lens = torch.tensor([100, 37, 0, 1, 5000], dtype=torch.int32, device=dev)
    k_lens = torch.tensor([170, 65, 10, 0, 9999], dtype=torch.int32, device=dev)
    for causal in (False, True):
        out = torch.full((5, 100, 4, 64), 7.0, dtype=torch.float16, device=dev)
        _check(pkg, dev, q, k, v, 0.2, causal=causal, q_lens=q_lens, k_lens=k_lens, out=out)
        for b, n in enumerate((100, 37, 0, 1, 100)):
            assert (out[b, n:] == 7.0).all()
    neg = torch.full((5,), -3, dtype=torch.int32, device=dev)
    assert (pkg.attention(q, k, v, 0.2, k_lens=neg, q_lens=q_lens)[0] == 0).all()
    assert (pkg.attention(q, k, v, 0.2, q_lens=neg) == 0).all()


@pytest.mark.parametrize("x", ["f16", "bf16"])
def test_unseen_values_do_not_matter(pkg, dev, x):
    """Infinities and NaN in k and v of keys that a row does not see: its result is
    that of clean ones, bit for bit; rows that see a NaN or an infinity have it."""
    import torch
    S = 300
    q, k, v = _qkv(dev, 2, S, S, 4, 2, 64, x, seed=10)
    lens = torch.tensor([S, 130], dtype=torch.int32, device=dev)
    docs = (torch.arange(S, device=dev) // 75).to(torch.int32).repeat(2, 1)
    for masks in (dict(causal=True, q_lens=lens, k_lens=lens), dict(q_docs=docs, k_docs=docs),
                  dict(causal=True, q_docs=docs, k_docs=docs)):
        clean = pkg.attention(q, k, v, 0.2, **masks)
        for bad in (math.nan, math.inf, -math.inf):
            k2, v2 = k.clone(), v.clone()
            k2[:, 200:] = bad
            v2[:, 200:, :, ::3] = bad
            k2[1, 130:] = math.nan
            v2[1, 130:] = math.nan
            got = pkg.attention(q, k2, v2, 0.2, **masks)
            for b in range(2):
                seen, m, _ = _seen(b, S, S, dev, **masks)
                safe = ~seen[:, 130 if b else 200:].any(1)     # what holds bad values
                safe[m:] = False
                assert safe.any()
                assert torch.equal(got[b][safe], clean[b][safe])
    # only v: what a row sees of it comes through
    v2 = v.clone()
    v2[:, 250, 0, 5], v2[:, 250, 0, 6], v2[:, 251, 0, 6], v2[:, 250, 0, 7] = math.inf, math.inf, -math.inf, math.nan
    got, clean = (pkg.attention(q, k, t, 0.2, causal=True) for t in (v2, v))
    assert (got[:, 251:, :2, 5] == math.inf).all() and (got[:, 250, :2, 6] == math.inf).all()
    assert got[:, 251:, :2, 6].isnan().all() and got[:, 250:, :2, 7].isnan().all()
    keep = torch.ones(2, S, 4, 64, dtype=torch.bool, device=dev)
    keep[:, 250:, :2, 5:8] = False
    assert torch.equal(got[keep], clean[keep])


def test_strides(pkg, dev):
    """Columns of one projection, broadcast heads and sequences, an output inside a
    larger tensor."""
    import torch
    gen = torch.Generator(device=dev).manual_seed(11)
    qkv = torch.randn(2, 130, 8 + 2 * 2, 72, generator=gen, device=dev).half()
    q, k, v = qkv[:, :, :8], qkv[:, :, 8:10], qkv[:, :, 10:]
    wide = torch.full((2, 130, 10, 80), 3.0, dtype=torch.float16, device=dev)
    _check(pkg, dev, q, k, v, 0.2, causal=True, out=wide[:, :, 1:9, :72])
    assert (wide[:, :, 0] == 3).all() and (wide[:, :, 9] == 3).all() and (wide[..., 72:] == 3).all()
    _check(pkg, dev, q, k[:1, :, :1].expand(2, 130, 8, 72), v[:, :, 1:].expand(2, 130, 8, 72), 0.2)
    heads_first = torch.randn(2, 8, 130, 72, generator=gen, device=dev).half().transpose(1, 2)
    _check(pkg, dev, heads_first, heads_first, heads_first, 0.2)
    one = k[:, 3:4].expand(2, 130, 2, 72)                 # one row of keys for all
    _check(pkg, dev, q, one, v, 0.2)


def test_far_offsets(pkg, dev):
    """Keys, values and rows 2^20 values apart: offsets past 2^32 bytes and 2^31 values."""
    import torch
    rows, gap, D = 2100, 1 << 20, 64
    base = torch.empty(rows * gap, dtype=torch.float16, device=dev)
    assert base.numel() > 2 ** 31
    q, k, v, out = (base.as_strided((1, rows, 2, D), (rows * gap, gap, D, 1), 256 * i) for i in range(4))
    gen = torch.Generator(device=dev).manual_seed(5)
    for x in (q, k, v):
        x.copy_(torch.randn(1, rows, 2, D, generator=gen, device=dev))
    with pytest.raises(pkg.SltxError):
        pkg.attention(q, k, v, 0.2, causal=True, out=out)     # its span holds q's
    _check(pkg, dev, q, k, v, 0.2, causal=True)


def test_large_and_equal_scores(pkg, dev):
    """A growing maximum (late keys dominate), and scores that are all equal."""
    import torch
    q, k, v = _qkv(dev, 1, 64, 640, 1, 1, 64, "f16", seed=12)
    k = (k * torch.linspace(0.1, 8.0, 640, device=dev)[None, :, None, None]).half()
    _check(pkg, dev, q, k, v, 1.0)
    _check(pkg, dev, q, k.flip(1).contiguous(), v, 1.0, causal=True)
    _check(pkg, dev, torch.zeros_like(q), k, v, 1.0)


def test_same_results_every_time(pkg, dev):
    import torch
    q, k, v = _qkv(dev, 1, 500, 500, 4, 1, 128, "bf16", seed=13)
    first = pkg.attention(q, k, v, 0.1, causal=True)
    for _ in range(5):
        assert torch.equal(pkg.attention(q, k, v, 0.1, causal=True), first)


def test_streams_and_graphs(pkg, dev):
    """On a stream other than the current one; captured, and replayed with new inputs."""
    import torch
    q, k, v = _qkv(dev, 2, 90, 90, 4, 2, 64, "f16", seed=14)
    want = pkg.attention(q, k, v, 0.2, causal=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        got = pkg.attention(q, k, v, 0.2, causal=True, stream=stream)
        s.synchronize()
        assert torch.equal(got, want)
    out = torch.empty_like(q)
    lens = torch.tensor([90, 60], dtype=torch.int32, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        pkg.attention(q, k, v, 0.2, causal=True, q_lens=lens, k_lens=lens, out=out, stream=s)
    for rep in range(3):
        q.copy_(torch.randn_like(q))
        lens[1] = 60 - 7 * rep
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, pkg.attention(q, k, v, 0.2, causal=True, q_lens=lens, k_lens=lens))


def test_empty_calls(pkg, dev):
    import torch
    q, k, v = _qkv(dev, 1, 4, 4, 2, 2, 64, "f16")
    assert pkg.attention(q[:0], k[:0], v[:0], 1.0).shape == (0, 4, 2, 64)
    assert pkg.attention(q[:, :0], k, v, 1.0).shape == (1, 0, 2, 64)
    assert (pkg.attention(q, k[:, :0], v[:, :0], 1.0) == 0).all()


def test_text_encoder_bias(pkg, dev):
    """distance_bias and attention as a text encoder's layer uses them: buckets of a
    relative-position table, scores unscaled."""
    import torch
    gen = torch.Generator(device=dev).manual_seed(15)
    table = torch.randn(32, 8, generator=gen, device=dev)
    bias, zero = pkg.distance_bias(table)
    q, k, v = _qkv(dev, 1, 200, 200, 8, 8, 64, "f16", seed=15, spread=0.5)
    _check(pkg, dev, q, k, v, 1.0, bias=bias, bias_zero=zero)
    # the buckets, from their definition: 16 for each direction, 8 of them exact
    for d in (-200, -128, -127, -91, -20, -8, -7, 0, 1, 7, 8, 15, 90, 128, 500):
        a = abs(d)
        n = a if a < 8 else min(15, 8 + int(math.log(a / 8) / math.log(128 / 8) * 8))
        assert torch.equal(bias[:, max(0, min(d + zero, bias.shape[1] - 1))], table[n + (16 if d > 0 else 0)])
