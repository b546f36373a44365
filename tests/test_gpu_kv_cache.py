"""The cache operators on the GPU: sltx_attention_cached, sltx_kv_append,
sltx_kv_accept and sltx_kv_evict against plain ones (attn_ref.py derives the
bounds of attention), alone, and together as a program decodes with them."""
import math

import pytest

import attn_ref as R

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def _cache(pkg, dev, L, lengths, Hk, cap, D, x="f16", weights=False, ahead=0, seed=0):
    """A cache with random entries in every slot (those behind the lengths too)."""
    import torch
    gen = torch.Generator(device=dev).manual_seed(seed)
    B = len(lengths)
    k, v = (torch.randn(L, B, Hk, cap, D, generator=gen, device=dev).to(_dt(x)) for _ in range(2))
    counts = torch.tensor([lengths, [n + ahead for n in lengths]], dtype=torch.int32, device=dev)
    more = {}
    if weights:
        more = dict(weight=torch.rand(L, B, Hk, cap, generator=gen, device=dev),
                    position=(torch.arange(cap, device=dev, dtype=torch.int32) + ahead).repeat(L, B, Hk, 1))
    return pkg.KVCache.from_tensors(k, v, counts, **more)


def _tree(T, seed, dev):
    import random
    rng = random.Random(seed)
    return [-1] + [rng.randrange(max(0, t - 5), t) for t in range(1, T)]


def _check_cached(pkg, dev, cache, layer, q, scale, cap=0.0, tree=None, weight_rows=0, stream=None):
    import torch
    B, T, Hq, D = q.shape
    Hk, C = cache.kv_heads, cache.capacity
    before = cache.weight.clone() if weight_rows else None
    got = pkg.attention_cached(q, cache, layer, scale, softcap=cap, tree=tree, weight_rows=weight_rows, stream=stream)
    torch.cuda.synchronize()
    want = before.double() if weight_rows else None
    off = torch.full_like(want, 2.0 ** -24) * want.abs() if weight_rows else None
    for b in range(B):
        old = min(max(int(cache.length[b]), 0), C)
        n = min(old + T, C)
        j, t = torch.arange(n, device=dev)[None] - old, torch.arange(T, device=dev)[:, None]
        if tree is None:
            seen = j <= t
        else:
            seen = (j < 0) | ((tree[b][:, None] >> j.clamp(0, 63)) & 1).bool()
        for h in range(Hq):
            g = h // (Hq // Hk)
            p, ref, wb, bound = R.head(q[b, :, h], cache.k[layer, b, g, :n], cache.v[layer, b, g, :n], scale, cap,
                                       None, seen)
            R.check_out(got[b, :, h], ref, bound, q.dtype, f"sequence {b} head {h}")
            if weight_rows:
                want[layer, b, g, :n] += p[:weight_rows].sum(0)
                # 8 more roundings: the product with 1 / l, the sum over rows, the addition
                off[layer, b, g, :n] += ((wb + 8 * 2.0 ** -24) * p)[:weight_rows].sum(0) * 1.01 + 2.0 ** -100
    if weight_rows:
        d = (cache.weight.double() - want).abs()
        sums = 2.0 ** -24 * weight_rows * (Hq // Hk) * want   # of the sum's order
        assert (d <= off + sums).all(), (d / (off + sums)).max().item()
    return got


CACHED = [  # lengths, T, Hq, Hk, D, capacity
    ([0], 1, 1, 1, 64, 1),
    ([5], 1, 3, 1, 128, 64),
    ([127, 128, 129], 1, 24, 8, 128, 256),
    ([4000], 1, 32, 8, 64, 4096),
    ([1000, 0, 31, 640], 1, 8, 2, 72, 1100),
    ([300], 7, 8, 4, 64, 400),
    ([300, 511], 23, 8, 2, 128, 700),
    ([2000], 64, 16, 4, 64, 2100),
    ([63, 1], 64, 3, 3, 40, 200),
    ([777], 130, 6, 2, 128, 1000),
    ([0, 100], 260, 4, 1, 64, 500),
]


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("case", CACHED, ids=str)
def test_chains(pkg, dev, case, cap, x):
    import torch
    lengths, T, Hq, Hk, D, C = case
    cache = _cache(pkg, dev, 2, lengths, Hk, C, D, x, seed=T)
    q = torch.randn(len(lengths), T, Hq, D, device=dev).to(_dt(x))
    _check_cached(pkg, dev, cache, 1, q, 2 / math.sqrt(D), cap)


@pytest.mark.parametrize("rows", ["one", "all"])
@pytest.mark.parametrize("case", [c for c in CACHED if c[1] <= 64], ids=str)
def test_weights(pkg, dev, case, rows):
    import torch
    lengths, T, Hq, Hk, D, C = case
    cache = _cache(pkg, dev, 2, lengths, Hk, C, D, "bf16", weights=True, seed=T)
    q = torch.randn(len(lengths), T, Hq, D, device=dev).bfloat16()
    _check_cached(pkg, dev, cache, 1, q, 2 / math.sqrt(D), 25.0 if T > 1 else 0.0, weight_rows=1 if rows == "one" else T)


@pytest.mark.parametrize("x", ["f16", "bf16"])
@pytest.mark.parametrize("case", [c for c in CACHED if 1 < c[1] <= 64], ids=str)
def test_trees(pkg, dev, case, x):
    import torch
    lengths, T, Hq, Hk, D, C = case
    cache = _cache(pkg, dev, 1, lengths, Hk, C, D, x, weights=True, seed=T)
    tree, depth = pkg.tree_masks([_tree(T, b, dev) for b in range(len(lengths))], device=dev)
    assert (depth[:, 0] == 0).all() and (depth >= 0).all()
    q = torch.randn(len(lengths), T, Hq, D, device=dev).to(_dt(x))
    _check_cached(pkg, dev, cache, 0, q, 2 / math.sqrt(D), 0.0, tree, weight_rows=T)


def test_empty_tree_rows_and_empty_cache(pkg, dev):
    """A token that sees nothing (no entries, no bit set) gives zeros."""
    import torch
    cache = _cache(pkg, dev, 1, [0, 3], 2, 64, 64, weights=True)
    tree = torch.tensor([[0, 2, 0], [0, 0, 4]], dtype=torch.int64, device=dev)
    q = torch.randn(2, 3, 4, 64, device=dev).half()
    got = _check_cached(pkg, dev, cache, 0, q, 0.2, 0.0, tree, weight_rows=3)
    assert (got[0, 0] == 0).all() and (got[0, 2] == 0).all() and (got[0, 1] != 0).any()
    many = torch.randn(2, 20, 8, 64, device=dev).half()                 # the many-row kernel
    got = _check_cached(pkg, dev, cache, 0, many, 0.2, 0.0, torch.zeros(2, 20, dtype=torch.int64, device=dev))
    assert (got[0] == 0).all() and (got[1] != 0).any()


@pytest.mark.parametrize("T", [1, 3, 40, 200])
@pytest.mark.parametrize("x", ["f16", "bf16"])
def test_unused_slots_do_not_matter(pkg, dev, x, T):
    """NaN in the slots behind the new tokens, and in new tokens that a row's branch
    does not have: bit for bit the result of clean ones."""
    import torch
    cache = _cache(pkg, dev, 1, [70, 0, 191], 2, 400, 64, x)
    q = torch.randn(3, T, 4, 64, device=dev).to(_dt(x))
    tree = None
    if 1 < T <= 64:   # the last token stands alone
        tree = torch.tensor([[1 << t for t in range(T)]] * 3, dtype=torch.int64, device=dev)
    clean = pkg.attention_cached(q, cache, 0, 0.2, tree=tree)
    for bad in (math.nan, math.inf):
        for b, n in enumerate((70, 0, 191)):
            cache.k[0, b, :, n + T:] = bad
            cache.v[0, b, :, n + T:] = bad
        assert torch.equal(pkg.attention_cached(q, cache, 0, 0.2, tree=tree), clean)
        if T > 1:      # the last new token too: only its own row sees it
            old = [(cache.k[0, b, :, n + T - 1].clone(), cache.v[0, b, :, n + T - 1].clone())
                   for b, n in enumerate((70, 0, 191))]
            for b, n in enumerate((70, 0, 191)):
                cache.k[0, b, :, n + T - 1] = bad
                cache.v[0, b, :, n + T - 1, ::2] = bad
            got = pkg.attention_cached(q, cache, 0, 0.2, tree=tree)
            assert torch.equal(got[:, :-1], clean[:, :-1])
            assert got[:, -1].isnan().any()
            for b, n in enumerate((70, 0, 191)):
                cache.k[0, b, :, n + T - 1], cache.v[0, b, :, n + T - 1] = old[b]


@pytest.mark.parametrize("T,n", [(70, 6), (200, 64), (300, 1)])
def test_chunk_in_two_calls(pkg, dev, T, n):
    """The last n of T appended tokens in a call of their own: the same rows as in one
    call, to the arithmetic's bounds, and their weights."""
    import torch
    cache = _cache(pkg, dev, 1, [37, 0], 2, 400, 64, weights=True)
    q = torch.randn(2, T, 6, 64, device=dev).half()
    whole = pkg.attention_cached(q, cache, 0, 0.2)
    before = cache.weight.clone()
    last = pkg.attention_cached(q[:, T - n:], cache, 0, 0.2, first=T - n, weight_rows=n)
    early = pkg.attention_cached(q[:, :T - n], cache, 0, 0.2)
    for b, old in enumerate((37, 0)):
        want = torch.zeros(2, old + T, dtype=torch.float64, device=dev)
        j, t = torch.arange(old + T, device=dev)[None] - old, torch.arange(T, device=dev)[:, None]
        for h in range(6):
            p, ref, _, bound = R.head(q[b, :, h], cache.k[0, b, h // 3, :old + T], cache.v[0, b, h // 3, :old + T], 0.2,
                                      0.0, None, j <= t)
            R.check_out(whole[b, :, h], ref, bound, q.dtype)
            R.check_out(last[b, :, h], ref[T - n:], bound[T - n:], q.dtype)
            R.check_out(early[b, :, h], ref[:T - n], bound[:T - n], q.dtype)
            want[h // 3] += p[T - n:].sum(0)
        d = (cache.weight[0, b, :, :old + T].double() - before[0, b, :, :old + T].double() - want).abs()
        assert (d <= 2.0 ** -22 * (1 + want) + 1e-5 * want).all()
    assert torch.equal(cache.weight[0, 0, :, 37 + T:], before[0, 0, :, 37 + T:])


@pytest.mark.parametrize("B,Hk,T,rows", [(2, 4, 1, 1), (5, 1, 1, 0), (70, 1, 1, 1), (130, 1, 3, 3), (3, 2, 23, 1),
                                         (70, 1, 23, 23), (4, 1, 40, 0)])
def test_unequal_lengths(pkg, dev, B, Hk, T, rows):
    """Parts are shared out by length: sequences from nothing to thousands of tokens in
    one call, every one against the plain attention."""
    import torch
    gen = torch.Generator().manual_seed(B)
    capacity = 6000 if B < 10 else 900
    lens = torch.randint(0, capacity // 8, (B,), generator=gen)
    lens[0], lens[-1] = 0, capacity - T       # one empty, one that fills the cache
    cache = _cache(pkg, dev, 1, lens.tolist(), Hk, capacity, 64, weights=True)
    before = cache.weight.clone()
    q = torch.randn(B, T, 4 * Hk, 64, device=dev).half()
    out = pkg.attention_cached(q, cache, 0, 0.25, weight_rows=rows)
    for b in range(B):
        n = int(lens[b])
        j, t = torch.arange(n + T, device=dev)[None] - n, torch.arange(T, device=dev)[:, None]
        for g in range(Hk):
            want = torch.zeros(n + T, dtype=torch.float64, device=dev)
            for h in range(4 * g, 4 * g + 4):
                p, ref, _, bound = R.head(q[b, :, h], cache.k[0, b, g, :n + T], cache.v[0, b, g, :n + T], 0.25, 0.0,
                                          None, j <= t)
                R.check_out(out[b, :, h], ref, bound, q.dtype, (b, h))
                want += p[:rows].sum(0)
            d = (cache.weight[0, b, g, :n + T].double() - before[0, b, g, :n + T].double() - want).abs()
            assert (d <= 2.0 ** -22 * (1 + want) + 1e-5 * want).all(), (b, g)
            assert torch.equal(cache.weight[0, b, g, n + T:], before[0, b, g, n + T:])


def test_full_cache(pkg, dev):
    """Tokens past the capacity are dropped: not written, not seen, not counted."""
    import torch
    cache = _cache(pkg, dev, 2, [60, 64, 10], 2, 64, 64, weights=True)
    k0, v0, w0, p0 = (t.clone() for t in (cache.k, cache.v, cache.weight, cache.position))
    new = torch.randn(3, 8, 4 + 2 + 2, 64, device=dev).half()
    freq = pkg.rope_inv_freq(64, device=dev)
    for layer in range(2):
        q = pkg.kv_append(new[:, :, :4], new[:, :, 4:6], new[:, :, 6:], cache, layer, freq)
    assert torch.equal(cache.k[:, 1], k0[:, 1]) and torch.equal(cache.v[:, 1], v0[:, 1])
    assert torch.equal(cache.k[:, 0, :, :60], k0[:, 0, :, :60]) and not torch.equal(cache.k[:, 0], k0[:, 0])
    assert torch.equal(cache.k[:, 2, :, 18:], k0[:, 2, :, 18:])
    assert torch.equal(cache.weight[:, 1], w0[:, 1]) and torch.equal(cache.position[:, 1], p0[:, 1])
    assert (cache.weight[:, 0, :, 60:] == 0).all()
    _check_cached(pkg, dev, cache, 1, q, 0.2)
    pkg.kv_accept(cache, 8)
    assert cache.length.tolist() == [64, 64, 18] and cache.next_position.tolist() == [64, 64, 18]


# ---- append ----

def _rotated(x, at, freq, interleaved):
    """x [T, heads, D] in 64 bits, at [T]."""
    import torch
    x, n = x.double().clone(), freq.numel()
    angle = (at.double()[:, None] * freq.double()[None])[:, None]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    ra, rb = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
    y = x.clone()
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = ra, rb
    else:
        y[..., :n], y[..., n:2 * n] = ra, rb
    return y


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,pairs", [(64, 32), (128, 64), (128, 16), (40, 20), (72, 5), (64, 0)])
@pytest.mark.parametrize("x", ["f16", "bf16"])
def test_append(pkg, dev, x, D, pairs, interleaved):
    """Rotation, slots, positions, at near and far places; q, k and v columns of one
    projection.  A value is off by half a step of its own, and 2^-21 of its pair
    (the angle's sine and cosine, two products and a sum in 32 bits)."""
    import torch
    lengths, starts = [0, 17, 90], [0, 4000, 2_000_000_011]
    cache = _cache(pkg, dev, 2, lengths, 2, 100, D, x, weights=True)
    cache.next_position.copy_(torch.tensor(starts, dtype=torch.int32))
    k0, v0 = cache.k.clone(), cache.v.clone()
    T = 6
    new = torch.randn(3, T, 4 + 2 + 2, D, device=dev).to(_dt(x))
    q, k, v = new[:, :, :4], new[:, :, 4:6], new[:, :, 6:]
    freq = (500000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))).float().to(dev)
    depth = torch.tensor([[0, 1, 1, 2, 2, 2]] * 3, dtype=torch.int32, device=dev)
    for tree in (False, True):
        got = pkg.kv_append(q, k, v, cache, 1, freq if pairs else None, depth=depth if tree else None,
                            interleaved=interleaved)
        torch.cuda.synchronize()
        for b in range(3):
            at = starts[b] + (depth[b] if tree else torch.arange(T, device=dev)).double()
            n = lengths[b]
            for y, src in ((got[b], q[b]), (cache.k[1, b, :, n:n + T].transpose(0, 1), k[b])):
                ref = _rotated(src, at, freq, interleaved)
                size = 2 * src.double().abs().amax()
                assert ((y.double() - ref).abs() <= R.half_step(y.dtype) * ref.abs() + 2.0 ** -21 * size + 2.0 ** -25).all()
            assert torch.equal(cache.v[1, b, :, n:n + T].transpose(0, 1), v[b])
            assert torch.equal(cache.position[1, b, :, n:n + T].double(), at[None].expand(2, T))
            assert (cache.weight[1, b, :, n:n + T] == 0).all()
            for y, y0 in ((cache.k, k0), (cache.v, v0)):     # nothing else changed
                assert torch.equal(y[0], y0[0]) and torch.equal(y[1, b, :, :n], y0[1, b, :, :n])
                assert torch.equal(y[1, b, :, n + T:], y0[1, b, :, n + T:])
    assert cache.length.tolist() == lengths                  # accepted later


# ---- accept ----

@pytest.mark.parametrize("D", [8, 64, 128])
@pytest.mark.parametrize("weights", [False, True])
def test_accept(pkg, dev, weights, D):
    """Paths in and out of order, counts that cut them, indices that end them."""
    import torch
    lengths = [0, 33, 100, 7, 120]
    cache = _cache(pkg, dev, 3, lengths, 2, 128, D, weights=weights, ahead=5)
    path = torch.tensor([[0, 2, 5, 9], [3, 1, 0, 2], [0, 1, 2, 3], [0, 30, 4, 5], [0, 3, 9, 5]],
                        dtype=torch.int32, device=dev)
    count = torch.tensor([4, 3, 9, 4, 4], dtype=torch.int32, device=dev)
    taken = [[0, 2, 5, 9], [3, 1, 0], [0, 1, 2, 3], [0], [0, 3]]   # 30 is no draft; slot 129 does not exist
    before = [t.clone() for t in (cache.k, cache.v) + ((cache.weight, cache.position) if weights else ())]
    pkg.kv_accept(cache, 12, path=path, count=count)
    after = (cache.k, cache.v) + ((cache.weight, cache.position) if weights else ())
    for old, new in zip(before, after):
        want = old.clone()
        for b, line in enumerate(taken):
            n = lengths[b]
            want[:, b, :, n:n + len(line)] = old[:, b, :, [n + t for t in line]]
        assert torch.equal(new, want)
    assert cache.length.tolist() == [n + len(t) for n, t in zip(lengths, taken)]
    assert cache.next_position.tolist() == [n + 5 + len(t) for n, t in zip(lengths, taken)]


def test_accept_counts(pkg, dev):
    import torch
    cache = _cache(pkg, dev, 1, [3, 3, 3, 3], 1, 16, 8)
    pkg.kv_accept(cache, 4, count=torch.tensor([-2, 0, 2, 9], dtype=torch.int32, device=dev))
    assert cache.length.tolist() == [3, 3, 5, 7] and cache.next_position.tolist() == [3, 3, 5, 7]
    pkg.kv_accept(cache, 12)
    assert cache.length.tolist() == [15, 15, 16, 16]
    pkg.kv_accept(cache, 4, path=torch.zeros(4, 2, dtype=torch.int32, device=dev),
                  count=torch.tensor([0, -1, 1, 2], dtype=torch.int32, device=dev))
    assert cache.length.tolist() == [15, 15, 16, 16]


def test_far_offsets(pkg, dev):
    """A cache of more than 2^31 values: its last layer and head, near the end of
    hundreds of thousands of slots, through all the operators."""
    import torch
    L, Hk, C, D, n, T = 4, 8, 600_064, 128, 600_000, 3
    k, v = (torch.empty(L, 1, Hk, C, D, dtype=torch.float16, device=dev) for _ in range(2))
    assert k.numel() > 2 ** 31
    gen = torch.Generator(device=dev).manual_seed(3)
    lay = L - 1
    for x in (k, v):
        x[lay].normal_(generator=gen)
    weight = torch.zeros(L, 1, Hk, C, device=dev)
    weight[lay] = torch.rand(1, Hk, C, generator=gen, device=dev)
    position = torch.arange(C, dtype=torch.int32, device=dev).repeat(L, 1, Hk, 1)
    counts = torch.tensor([[n], [n]], dtype=torch.int32, device=dev)
    cache = pkg.KVCache.from_tensors(k, v, counts, weight=weight, position=position)
    new = torch.randn(1, T, 3 * Hk, D, generator=gen, device=dev).half()
    q = pkg.kv_append(new[:, :, :Hk], new[:, :, Hk:2 * Hk], new[:, :, 2 * Hk:], cache, lay)
    assert torch.equal(k[lay, 0, :, n:n + T], new[0, :, Hk:2 * Hk].transpose(0, 1))
    assert torch.equal(v[lay, 0, :, n:n + T], new[0, :, 2 * Hk:].transpose(0, 1))
    out = pkg.attention_cached(q, cache, lay, 0.3)
    seen = torch.arange(n + T, device=dev)[None] <= n + torch.arange(T, device=dev)[:, None]
    for h in (0, Hk - 1):
        _, ref, _, bound = R.head(q[0, :, h], k[lay, 0, h, :n + T], v[lay, 0, h, :n + T], 0.3, 0.0, None, seen)
        R.check_out(out[0, :, h], ref, bound, q.dtype, h)
    want = k[lay, 0, :, n + 2].clone()
    pkg.kv_accept(cache, T, path=torch.tensor([[0, 2]], dtype=torch.int32, device=dev))
    assert cache.length.tolist() == [n + 2] and torch.equal(k[lay, 0, :, n + 1], want)
    budget, w = 500_000, weight[lay, 0, Hk - 1, :n + 2].clone()
    last = n + 2 - 8                       # protected: the first 4 and the last 8 positions
    w[:4] = w[last:] = 2.0
    keep = torch.zeros(n + 2, dtype=torch.bool, device=dev)
    keep[torch.sort(w, descending=True, stable=True).indices[:budget]] = True
    holes = torch.nonzero(~keep[:budget])[:, 0]
    comers = budget + torch.nonzero(keep[budget:])[:, 0]
    slots = torch.arange(budget, device=dev)
    slots[holes] = comers
    want, at = k[lay, 0, Hk - 1].index_select(0, slots), position[lay, 0, Hk - 1][slots]
    pkg.kv_evict(cache, budget, sinks=4, recent=8)
    assert cache.length.tolist() == [budget]
    assert torch.equal(position[lay, 0, Hk - 1, :budget], at)
    assert torch.equal(k[lay, 0, Hk - 1, :budget], want)


# ---- evict ----

def _evicted(w, p, n, after, budget, sinks, recent, C):
    """Slot each slot's entry comes from, by the rule."""
    source = list(range(C))
    if n <= budget:
        return source, n
    def rank(s):
        safe = p[s] < sinks or p[s] >= after - recent
        x = w[s]
        return (0 if safe else 1, 0 if safe else (0 if x == x else 1), 0 if safe or x != x else -x, s)
    keep = set(sorted(range(n), key=rank)[:budget])
    comers = sorted(s for s in keep if s >= budget)
    for hole, s in zip((s for s in range(budget) if s not in keep), comers):
        source[hole] = s
    return source, budget


EVICT = [  # capacity, lengths, budget, sinks, recent
    (64, [64], 16, 4, 4),
    (300, [300, 129, 128, 0], 128, 4, 32),
    (1500, [1025, 1500], 1024, 0, 0),
    (3000, [2999, 65, 1], 64, 10, 54),
    (200, [200], 199, 4, 100),
    (128, [128], 1, 0, 1),
    (5000, [4097], 2500, 0, 0),
    (2048, [2048, 1500], 700, 4, 50),
    (8192, [8192], 64, 4, 16),
    (12000, [12000, 9001], 5000, 0, 128),
    (17000, [17000], 16000, 1, 1),
]


@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
@pytest.mark.parametrize("case", EVICT, ids=str)
def test_evict(pkg, dev, case, kind):
    import torch
    C, lengths, budget, sinks, recent = case
    L, Hk = 2, 2
    cache = _cache(pkg, dev, L, lengths, Hk, C, 64, weights=True, ahead=3, seed=C)
    gen = torch.Generator(device=dev).manual_seed(budget)
    if kind == "ties":     # few values; zeros of both signs are equal
        cache.weight.copy_(torch.randint(-1, 2, cache.weight.shape, generator=gen, device=dev).float() * 0.0
                           + torch.randint(0, 3, cache.weight.shape, generator=gen, device=dev))
        cache.weight[cache.weight == 0] = -0.0
        cache.weight[..., ::7] = 0.0
    elif kind == "odd":    # infinities, NaN, negative and tiny values
        odd = torch.tensor([math.nan, math.inf, -math.inf, -1.0, 1e-45, 0.0, -1e-45, 3e38], device=dev)
        at = torch.randint(0, 24, cache.weight.shape, generator=gen, device=dev)
        cache.weight.copy_(torch.where(at < 8, odd[at.clamp(max=7)], cache.weight))
    # positions in another order than the slots, as after an earlier eviction
    perm = torch.stack([torch.randperm(C, generator=gen, device=dev) for _ in range(L * len(lengths) * Hk)])
    cache.position.copy_(perm.view(cache.position.shape))
    cache.next_position.fill_(C)
    before = [t.clone() for t in (cache.k, cache.v, cache.weight, cache.position)]
    w, p = cache.weight.tolist(), cache.position.tolist()
    pkg.kv_evict(cache, budget, sinks=sinks, recent=recent)
    torch.cuda.synchronize()
    for b, n in enumerate(lengths):
        for layer in range(L):
            for h in range(Hk):
                source, left = _evicted(w[layer][b][h], p[layer][b][h], n, C, budget, sinks, recent, C)
                for old, new in zip(before, (cache.k, cache.v, cache.weight, cache.position)):
                    want = old[layer, b, h][torch.tensor(source, device=dev)]
                    assert torch.equal(new[layer, b, h].nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0)), (b, layer, h)
        assert int(cache.length[b]) == min(n, budget)
    assert (cache.next_position == C).all()


def test_evict_more_protected_than_budget(pkg, dev):
    """Positions that occur twice can make more than the budget protected: the lowest
    slots of them stay."""
    import torch
    cache = _cache(pkg, dev, 1, [100], 1, 100, 8, weights=True)
    cache.position.zero_()
    before = cache.k.clone()
    pkg.kv_evict(cache, 10, sinks=1, recent=0)
    assert torch.equal(cache.k, before) and cache.length.tolist() == [10]


# ---- together ----

def test_streams_and_graphs(pkg, dev):
    """A decode step of two layers (append, attention with weights, accept, evict)
    captured once per cache on one stream and replayed in turns: each cache's
    results are those of the same steps run eagerly."""
    import torch
    T, Hq, Hk, D, C, steps = 1, 4, 2, 64, 200, 12
    s = torch.cuda.Stream()
    freq = pkg.rope_inv_freq(D, device=dev)
    gen = torch.Generator(device=dev).manual_seed(0)
    inputs = torch.randn(2, steps, 2, 3, T, Hq + 2 * Hk, D, generator=gen, device=dev).half()

    def step(cache, new, out, stream):
        for layer in range(2):
            q, k, v = new[layer][:, :, :Hq], new[layer][:, :, Hq:Hq + Hk], new[layer][:, :, Hq + Hk:]
            q = pkg.kv_append(q, k, v, cache, layer, freq, stream=stream)
            pkg.attention_cached(q, cache, layer, 0.2, weight_rows=1, out=out[layer], stream=stream)
        pkg.kv_accept(cache, 1, stream=stream)
        pkg.kv_evict(cache, 64, sinks=2, recent=8, stream=stream)

    def make(i):
        return _cache(pkg, dev, 2, [60, 5, 100], Hk, C, D, weights=True, seed=i)

    want = []
    for i in range(2):
        cache, out = make(i), torch.zeros(2, 3, T, Hq, D, dtype=torch.float16, device=dev)
        outs = []
        for n in range(steps):
            step(cache, inputs[i, n], out, None)
            outs.append(out.clone())
        want.append((outs, [t.clone() for t in (cache.k, cache.v, cache.counts, cache.weight, cache.position)]))
    torch.cuda.synchronize()
    caches, graphs, news, outs = [], [], [], []
    for i in range(2):
        cache, out = make(i), torch.zeros(2, 3, T, Hq, D, dtype=torch.float16, device=dev)
        new = inputs[i, 0].clone()
        saved = [t.clone() for t in (cache.k, cache.v, cache.counts, cache.weight, cache.position)]
        torch.cuda.synchronize()
        step(cache, new, out, s)          # sizes the scratch
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step(cache, new, out, s)
        for t, old in zip((cache.k, cache.v, cache.counts, cache.weight, cache.position), saved):
            t.copy_(old)
        caches.append(cache), graphs.append(g), news.append(new), outs.append(out)
    torch.cuda.synchronize()
    for n in range(steps):
        for i in range(2):
            news[i].copy_(inputs[i, n])
            torch.cuda.synchronize()
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i][0][n]), (i, n)
    for i in range(2):
        c = caches[i]
        for got, ref in zip((c.k, c.v, c.counts, c.weight, c.position), want[i][1]):
            assert torch.equal(got, ref)


@pytest.mark.parametrize("x", ["f16", "bf16"])
def test_prompt_draft_decode(pkg, dev, x):
    """A prompt in two chunks, a drafted tree of which a path is accepted, single
    tokens: each step's output is attention over the plain sequence of its tokens."""
    import torch
    Hq, Hk, D, scale = 6, 2, 128, 0.15
    gen = torch.Generator(device=dev).manual_seed(4)
    freq = pkg.rope_inv_freq(D, theta=500000.0, device=dev)
    cache = pkg.KVCache(1, 1, Hk, 400, D, dtype=_dt(x), track_weights=True, device=dev)
    keys, values = [], []                 # of the sequence, as stored

    def run(T, parents=None, accept=None):
        new = torch.randn(1, T, Hq + 2 * Hk, D, generator=gen, device=dev).to(_dt(x))
        tree = depth = None
        if parents:
            tree, depth = pkg.tree_masks([parents], device=dev)
        q = pkg.kv_append(new[:, :, :Hq], new[:, :, Hq:Hq + Hk], new[:, :, Hq + Hk:], cache, 0, freq, depth=depth)
        got = pkg.attention_cached(q, cache, 0, scale, tree=tree, weight_rows=T if T <= 64 else 0)
        n = len(keys)
        at = n + (depth[0] if parents else torch.arange(T, device=dev))
        k_new = _rotated(new[0, :, Hq:Hq + Hk], at, freq, False).to(_dt(x))
        for t in range(T):
            line, up = [], t
            while up >= 0:
                line.append(up)
                up = parents[up] if parents else up - 1
            line = line[::-1]
            k = torch.stack(keys + [k_new[u] for u in line])
            v = torch.stack(values + [new[0, u, Hq + Hk:] for u in line])
            if t in (0, T // 2, T - 1):
                for h in range(Hq):
                    # rotated keys may round to the other neighbour here and there
                    _, ref, _, bound = R.head(q[0, t:t + 1, h], k[:, h // 3], v[:, h // 3], scale)
                    R.check_out(got[0, t:t + 1, h], ref, bound * 1.5, q.dtype, f"token {n + t} head {h}")
        chosen = accept if accept is not None else list(range(T))
        if accept is None:
            pkg.kv_accept(cache, T)
        else:
            pkg.kv_accept(cache, T, path=torch.tensor([accept], dtype=torch.int32, device=dev))
        keys.extend(k_new[u] for u in chosen)
        values.extend(new[0, u, Hq + Hk:] for u in chosen)
        assert cache.length.tolist() == [len(keys)] == cache.next_position.tolist()

    run(150)
    run(64)
    run(9, parents=[-1, 0, 0, 1, 1, 2, 3, 5, 5], accept=[0, 2, 5, 8])
    for _ in range(3):
        run(1)
    run(17)
    # every row of the tracked calls gave the weight 1 in each group
    total = cache.weight[0, 0].double().sum(1)
    assert (total - 3 * (64 + 3 + 17)).abs().max() < 3 * 9 + 1e-2
