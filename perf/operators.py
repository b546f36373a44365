"""The attention operators that this library is judged on, in plain torch and through
its entry points: attention over whole sequences, attention over a key/value cache,
and what keeps such a cache: appending, accepting drafted tokens, evicting.

A case is a dict of plain values.  Its "work" names the operator:

    attention  softmax(cap(scale q.k) + bias[j - i]) v over B sequences of Sq rows and
               Sk keys; causal, with a prefix that every row sees, within documents,
               over padded rows
    cached     the same over a key/value cache: T tokens a sequence whose keys are
               already in the cache; a decoded token (T = 1), a tree of drafted tokens
               (each sees the cache and its ancestors), or a chunk of a prompt;
               adds the first rows' attention weights to the cache's sums
    append     rotary embedding of T tokens' q and k, and k and v written to the cache
    accept     drafted tokens kept: the accepted path's rows moved up in every layer,
               the sequence lengthened
    evict      every layer's and head's cache cut to a budget: first and recent
               positions and the highest attention sums stay

Heads and sizes are those of the decoder layers, the text encoder and the diffusion
transformer that the library's benchmark runs.
"""
import math
from types import SimpleNamespace

import torch

own = False

# (query heads, key/value heads, head dim): decoders of 3B, 1B and 8B, the text
# encoder, the diffusion transformer
HEADS = ((24, 8, 128), (32, 8, 64), (32, 8, 128), (64, 64, 64), (32, 32, 64))
# q.k products of the largest listed case: a drawn one has no more
MOST_PRODUCTS = 6144 * 6144 * 32 * 64
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # The text encoder of a video pipeline: a caption of 77 tokens padded to 128,
        # biased by distance alone, scores unscaled.
        dict(name="attn_text_m128", work="attention", heads=3, B=1, Sq=128, Sk=128, x="f16", bias=128,
             causal=False, prefix=0, docs=0, cap=0.0, pad=51),
        # Texts of odd lengths packed into one row of tokens, scored by a decoder whose
        # scores are capped.
        dict(name="attn_docs_m4095", work="attention", heads=1, B=1, Sq=4095, Sk=4095, x="bf16", bias=0,
             causal=True, prefix=0, docs=9, cap=30.0, pad=0),
        # One block of the video model at 16 x 16 x 24 latent patches: the largest product.
        dict(name="attn_video_m6144", work="attention", heads=4, B=1, Sq=6144, Sk=6144, x="bf16", bias=0,
             causal=False, prefix=0, docs=0, cap=0.0, pad=0),
        # One token of a chat near the end of the 4096 that a cache holds.
        dict(name="cached_m1_n4000", work="cached", heads=0, B=1, T=1, n=4000, kind="token", x="f16",
             weights=0, cap=0.0, ragged=False),
        # A tree of 23 drafted tokens for each of four long conversations of unequal
        # length, attention sums kept for eviction.
        dict(name="cached_tree23_b4", work="cached", heads=2, B=4, T=23, n=16301, kind="tree", x="bf16",
             weights=1, cap=0.0, ragged=True),
        # The benchmark's prompt of 750 tokens behind a system prompt that is cached.
        dict(name="cached_m750_n1300", work="cached", heads=0, B=1, T=750, n=1300, kind="chunk", x="f16",
             weights=0, cap=0.0, ragged=False),
        # Eight sequences decoded together: the smallest call.
        dict(name="append_m1_b8", work="append", heads=0, B=8, T=1, n=3000, kind="chain", x="f16", ragged=True),
        # The benchmark's prompt, far into a long conversation.
        dict(name="append_m750", work="append", heads=2, B=1, T=750, n=120001, kind="chain", x="bf16",
             ragged=False),
        # A verified draft: five of 23 tokens stay, in all 28 layers.
        dict(name="accept_5of23", work="accept", heads=0, layers=28, B=1, T=23, n=2000, depth=5, x="f16"),
        # Sixteen sequences with drafts of the largest tree.
        dict(name="accept_9of64_b16", work="accept", heads=1, layers=16, B=16, T=64, n=500, depth=9, x="bf16"),
        # A long prompt just read, cut to 1024 entries in every layer and head.
        dict(name="evict_n6001", work="evict", heads=1, layers=16, B=1, n=6001, budget=1024, sinks=4,
             recent=64, x="f16"),
        # One token past the budget, as in every step of a long generation of eight sequences.
        dict(name="evict_step_b8", work="evict", heads=0, layers=28, B=8, n=1025, budget=1024, sinks=4,
             recent=256, x="f16"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    work = rng.choice(("attention", "attention", "attention", "cached", "cached", "cached", "append",
                       "accept", "evict"))
    heads = rng.randrange(3)
    x = rng.choice(("f16", "bf16"))
    if work == "attention":
        heads = rng.randrange(len(HEADS))
        B, Sq = rng.choice((1, 1, 2, 3)), _log_int(rng, 1, 4096)
        kind = rng.choice(("plain", "bias", "causal", "prefix", "docs", "docs"))
        Sk = Sq + (_log_int(rng, 1, 2048) if kind in ("plain", "causal") and rng.random() < 0.3 else 0)
        Hq, _, D = HEADS[heads]
        if B * Sq * Sk * Hq * D > MOST_PRODUCTS:
            B, Sq, Sk = 1, Sq // 2, Sk // 2
        return dict(work=work, heads=heads, B=B, Sq=Sq, Sk=Sk, x=x,
                    bias=rng.choice((32, 128, 1000)) if kind == "bias" else 0,
                    causal=kind in ("causal", "prefix") or (kind == "docs" and rng.random() < 0.7),
                    prefix=rng.randint(1, Sk) if kind == "prefix" else 0,
                    docs=rng.randint(2, 12) if kind == "docs" else 0,
                    cap=rng.choice((0.0, 0.0, 30.0, 50.0)),
                    pad=rng.randint(0, Sq - 1) if rng.random() < 0.3 else 0)
    if work == "cached":
        kind = rng.choice(("token", "tree", "chunk"))
        T = 1 if kind == "token" else rng.randint(2, 64) if kind == "tree" else _log_int(rng, 65, 1024)
        B, n = _log_int(rng, 1, 8) if kind != "chunk" else rng.choice((1, 2)), _log_int(rng, 1, 16384)
        if B * T * (n + T) * HEADS[heads][0] * HEADS[heads][2] > MOST_PRODUCTS:
            B, n = 1, n // 2
        return dict(work=work, heads=heads, B=B, T=T, n=n, kind=kind, x=x,
                    weights=rng.choice((0, 1, T)) if kind != "chunk" else 0,
                    cap=rng.choice((0.0, 0.0, 50.0)), ragged=rng.random() < 0.5)
    if work == "append":
        T = rng.choice((1, _log_int(rng, 2, 64), _log_int(rng, 64, 2048)))
        return dict(work=work, heads=heads, B=_log_int(rng, 1, 16 if T <= 64 else 2), T=T,
                    n=_log_int(rng, 1, 200000), kind=rng.choice(("chain", "tree")) if 1 < T <= 64 else "chain",
                    x=x, ragged=rng.random() < 0.5)
    layers = rng.choice((2, 16, 28, 32))
    if work == "accept":
        T = rng.randint(2, 64)
        return dict(work=work, heads=heads, layers=layers, B=_log_int(rng, 1, 16), T=T,
                    n=_log_int(rng, 1, 2000), depth=rng.randint(1, min(T, 12)), x=x)
    B = _log_int(rng, 1, 8)
    n = _log_int(rng, 64, 8192 if layers * B <= 32 else 1500)
    budget = rng.randint(n // 2, n - 1) if rng.random() < 0.5 else _log_int(rng, 16, n - 1)
    return dict(work=work, heads=heads, layers=layers, B=B, n=n, budget=budget,
                sinks=rng.choice((0, 4)), recent=rng.randint(0, budget - 4), x=x)


# ---- inputs ----

def _normal(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _host(seed):
    """The generator of the choices that are made on the host (lengths, documents, trees)."""
    return torch.Generator().manual_seed(seed + 1)


def _randint(host, low, high):
    """A number from low to high, both included."""
    return int(torch.randint(low, high + 1, (1,), generator=host))


def _lengths(case, host, most):
    """Tokens that each sequence has in the cache."""
    if not case.get("ragged"):
        return [most] * case["B"]
    return [most] + [_randint(host, max(1, most // 2), most) for _ in range(case["B"] - 1)]


def _trees(case, host):
    """Drafted trees: each token but the first follows an earlier one (its parent); returns
    the parents, the depths, and for each token the set of tokens it sees as 64 bits."""
    parents, depths, masks = [], [], []
    for _ in range(case["B"]):
        p, d, m = [-1], [0], [1]
        for t in range(1, case["T"]):
            p.append(_randint(host, max(0, t - 6), t - 1))
            d.append(d[p[t]] + 1)
            m.append(m[p[t]] | 1 << t)
        parents.append(p)
        depths.append(d)
        masks.append([b - (1 << 64) if b >> 63 else b for b in m])
    return parents, depths, masks


def prepare(case, seed):
    """The tensors and the cache handle that a program has in hand before the call."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = _host(seed)
    s = SimpleNamespace(case=case)
    Hq, Hk, D = HEADS[case["heads"]]
    dt, B = DTYPES[case["x"]], case["B"]
    s.scale = 1.0 / math.sqrt(D)
    if case["work"] == "attention":
        Sq, Sk = case["Sq"], case["Sk"]
        # q, k and v are columns of one projection where a row has all three
        if Sq == Sk:
            qkv = _normal(gen, B, Sq, Hq + 2 * Hk, D, dtype=dt)
            s.q, s.k, s.v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
        else:
            s.q = _normal(gen, B, Sq, Hq, D, dtype=dt)
            s.k, s.v = (_normal(gen, B, Sk, Hk, D, dtype=dt) for _ in range(2))
        s.scale = 2.0 / math.sqrt(D)     # trained q.k spread wider than random ones
        s.bias = s.prefix = s.docs = s.q_lens = s.k_lens = None
        if case["bias"]:                 # one value for each distance, the same from `bias` on
            s.bias = torch.randn(Hq, 2 * case["bias"] + 1, generator=gen, device="cuda") * 2
        if case["prefix"]:
            s.prefix = _i32([case["prefix"]] + [_randint(host, 0, case["prefix"]) for _ in range(B - 1)])
        if case["docs"]:                 # lengths at random, the last tokens padding (no document)
            ids = torch.randint(0, Sq + 1, (B, case["docs"] - 1), generator=host)
            at = torch.arange(Sq)
            docs = (at[None, :, None] >= ids[:, None, :]).sum(2)
            docs[:, Sq - Sq // 50:] = -1
            s.docs = docs.to(torch.int32).cuda()
        if case["pad"]:
            pads = [case["pad"]] + [_randint(host, 0, case["pad"]) for _ in range(B - 1)]
            s.q_lens, s.k_lens = _i32([Sq - p for p in pads]), _i32([Sk - p for p in pads])
        s.out = torch.zeros(B, Sq, Hq, D, dtype=dt, device="cuda")
    else:
        L = case.get("layers", 1)
        T = case.get("T", 0)
        lengths = _lengths(case, host, case["n"])
        capacity = -(-(case["n"] + T + 1) // 128) * 128
        s.layer = 0
        s.k = _normal(gen, L, B, Hk, capacity, D, dtype=dt)
        s.v = _normal(gen, L, B, Hk, capacity, D, dtype=dt)
        # slots in use, and the position of the next token (later than that after evictions)
        ahead = 7 if case["work"] in ("append", "evict") else 0
        s.counts = _i32([lengths, [n + ahead for n in lengths]])
        # of each slot: its sum of attention weights, and its token's position
        s.book = torch.zeros(2, L, B, Hk, capacity, dtype=torch.int32, device="cuda")
        s.weight, s.position = s.book[0].view(torch.float32), s.book[1]
        s.position.copy_(torch.arange(capacity, device="cuda") + ahead)
        s.tracked = case["work"] in ("accept", "evict") or bool(case.get("weights"))
        if s.tracked:                    # few tokens get most of the attention
            s.weight.copy_(torch.empty_like(s.weight).exponential_(generator=gen).pow_(3).div_(case["n"]))
        if case["work"] == "cached":
            s.q = _normal(gen, B, T, Hq, D, dtype=dt)
            s.scale = 2.0 / math.sqrt(D)
            s.tree = torch.tensor(_trees(case, host)[2], device="cuda") if case["kind"] == "tree" else None
        elif case["work"] == "append":
            qkv = _normal(gen, B, T, Hq + 2 * Hk, D, dtype=dt)
            s.q, s.k_new, s.v_new = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
            s.inv_freq = (500000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
            s.depth = _i32(_trees(case, host)[1]) if case["kind"] == "tree" else None
        elif case["work"] == "accept":
            parents, depths, _ = _trees(case, host)
            path = [[0] * case["depth"] for _ in range(B)]
            count = []
            for b in range(B):           # the deepest branch, to the depth at most
                node = max(range(T), key=lambda t: depths[b][t])
                line = []
                while node >= 0:
                    line.append(node)
                    node = parents[b][node]
                line = line[::-1][:case["depth"]]
                path[b][:len(line)] = line
                count.append(len(line))
            s.path, s.count = _i32(path), _i32(count)
        s.counts0, s.book0 = s.counts.clone(), s.book.clone()
    if own:
        from __graft_entry__ import load_package
        s.pkg = load_package()
        if case["work"] != "attention":
            tracked = dict(weight=s.weight, position=s.position) if s.tracked else {}
            s.cache = s.pkg.KVCache.from_tensors(s.k, s.v, s.counts, **tracked)
    return s


# ---- one pass ----

def run(s):
    return {"attention": _attention, "cached": _cached, "append": _append, "accept": _accept,
            "evict": _evict}[s.case["work"]](s)


def _softmax_product(q, k, v, scale, cap, bias, seen):
    """q [B, Hk, G, S, D], k and v [B, Hk, N, D], bias and seen broadcast to the scores
    [B, Hk, G, S, N]: the weights and their product with v, in 32 bits."""
    B, Hk, G, S, D = q.shape
    scores = torch.matmul(q.float().reshape(B, Hk, G * S, D), k.float().transpose(2, 3).contiguous())
    scores = scores.view(B, Hk, G, S, -1).mul_(scale)
    if cap:
        scores = scores.div_(cap).tanh_().mul_(cap)
    if bias is not None:
        scores = scores + bias
    if seen is not None:
        scores = torch.where(seen, scores, scores.new_full((), -math.inf))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)      # a row that sees nothing
    p = scores.sub_(top).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30))
    return p, torch.matmul(p.view(B, Hk, G * S, -1), v.float()).view(B, Hk, G, S, D)


def _grouped(q, Hk):
    """[B, S, Hq, D] to [B, Hk, Hq / Hk, S, D]."""
    B, S, Hq, D = q.shape
    return q.reshape(B, S, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4)


def _attention(s):
    c = s.case
    if own:
        return s.pkg.attention(s.q, s.k, s.v, s.scale, softcap=c["cap"], bias=s.bias, bias_zero=c["bias"],
                               causal=c["causal"], prefix=s.prefix, q_docs=s.docs, k_docs=s.docs,
                               q_lens=s.q_lens, k_lens=s.k_lens, out=s.out)
    B, Sq, Hq, D = s.q.shape
    Sk, Hk = s.k.shape[1], s.k.shape[2]
    i, j = torch.arange(Sq, device="cuda"), torch.arange(Sk, device="cuda")
    # the last row stands at the last key
    shift = s.k_lens - s.q_lens if s.q_lens is not None else torch.full((B,), Sk - Sq, device="cuda")
    row = (i[None] + shift[:, None])[:, :, None]                    # [B, Sq, 1]
    seen = None
    if c["causal"]:
        seen = j <= row
        if s.prefix is not None:
            seen = seen | (j < s.prefix[:, None, None])
    if s.docs is not None:
        same = (s.docs[:, :, None] == s.docs[:, None, :]) & (s.docs[:, :, None] >= 0)
        seen = same if seen is None else seen & same
    if s.q_lens is not None:
        inside = j < s.k_lens[:, None, None]
        seen = inside if seen is None else seen & inside
    if seen is not None:
        seen = seen[:, None, None]
    bias = None
    if s.bias is not None:
        at = (j - row + c["bias"]).clamp(0, 2 * c["bias"])          # [B, Sq, Sk]
        bias = s.bias[:, at].permute(1, 0, 2, 3).reshape(B, Hk, Hq // Hk, Sq, Sk)
    _, o = _softmax_product(_grouped(s.q, Hk), s.k.transpose(1, 2), s.v.transpose(1, 2), s.scale, c["cap"],
                            bias, seen)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, Sq, Hq, D).to(s.out.dtype)
    if s.q_lens is None:
        s.out.copy_(o)
    else:
        s.out.copy_(torch.where((i < s.q_lens[:, None])[:, :, None, None], o, s.out))
    return s.out


def _cached(s):
    c = s.case
    if own:
        out = s.pkg.attention_cached(s.q, s.cache, s.layer, s.scale, softcap=c["cap"], tree=s.tree,
                                     weight_rows=c["weights"])
        return (out, s.weight) if c["weights"] else out
    B, T, Hq, D = s.q.shape
    k, v = s.k[s.layer], s.v[s.layer]
    Hk, N = k.shape[1], k.shape[2]
    j, t = torch.arange(N, device="cuda"), torch.arange(T, device="cuda")
    new = j - s.counts[0][:, None]                                  # [B, N]: which new token a slot holds
    if s.tree is None:
        seen = new[:, None, :] <= t[:, None]
    else:
        bit = (s.tree[:, :, None] >> new.clamp(0, 63)[:, None, :]) & 1
        seen = (new[:, None, :] < 0) | ((new[:, None, :] < T) & (bit != 0))
    p, o = _softmax_product(_grouped(s.q, Hk), k, v, s.scale, c["cap"], None, seen[:, None, None])
    out = o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(s.q.dtype)
    if not c["weights"]:
        return out
    s.weight[s.layer] += p[:, :, :, :c["weights"]].sum((2, 3))
    return out, s.weight


def _append(s):
    c = s.case
    if own:
        q = s.pkg.kv_append(s.q, s.k_new, s.v_new, s.cache, s.layer, s.inv_freq, depth=s.depth)
        return q, s.k, s.v
    B, T, D = s.q.shape[0], s.q.shape[1], s.q.shape[3]
    t = torch.arange(T, device="cuda")
    at = s.counts[1][:, None] + (t[None] if s.depth is None else s.depth)
    angle = (at[:, :, None].double() * s.inv_freq.double())[:, :, None]
    cos, sin = angle.cos().float(), angle.sin().float()

    def rotate(x):
        a, b = x[..., :D // 2].float(), x[..., D // 2:].float()
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(x.dtype)

    slot = (s.counts[0][:, None] + t[None]).long()
    b = torch.arange(B, device="cuda")[:, None]
    s.k[s.layer].transpose(1, 2)[b, slot] = rotate(s.k_new)
    s.v[s.layer].transpose(1, 2)[b, slot] = s.v_new
    return rotate(s.q), s.k, s.v


def _accept(s):
    s.counts.copy_(s.counts0)            # the next draft stands where this one stood
    if own:
        s.pkg.kv_accept(s.cache, s.case["T"], path=s.path, count=s.count)
        return s.k, s.v, s.counts, s.position, s.weight
    A = s.path.shape[1]
    i = torch.arange(A, device="cuda")
    start = s.counts[0][:, None]
    source = torch.where(i < s.count[:, None], start + s.path, start + i).long()   # [B, A]
    target = (start + i).long()
    b = torch.arange(s.counts.shape[1], device="cuda")[:, None]
    for x in (s.k, s.v, s.position, s.weight):
        x = x.movedim(1, 0).movedim(3, 1)                           # [B, capacity, L, Hk, ...]
        x[b, target] = x[b, source]
    s.counts += s.count
    return s.k, s.v, s.counts, s.position, s.weight


def _evict(s):
    c = s.case
    s.counts.copy_(s.counts0)            # as full as before the pass: what a step makes of it again
    s.book.copy_(s.book0)
    if own:
        s.pkg.kv_evict(s.cache, c["budget"], sinks=c["sinks"], recent=c["recent"])
        return s.k, s.v, s.counts, s.position, s.weight
    budget, D = c["budget"], s.k.shape[-1]
    N = s.k.shape[3]
    length, after = s.counts[0][None, :, None, None], s.counts[1][None, :, None, None]
    slot = torch.arange(N, device="cuda")
    live = slot < length
    safe = (s.position < c["sinks"]) | (s.position >= after - c["recent"])
    rank = torch.where(safe, math.inf, s.weight.double())
    rank = torch.where(live, rank, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    keep = torch.zeros(s.weight.shape, dtype=torch.bool, device="cuda").scatter_(-1, order, True) & live
    hole = (slot < budget) & ~keep & live
    comer = (slot >= budget) & keep
    comers = torch.where(comer, slot, N).sort(-1).values[..., :budget]
    nth = (hole.cumsum(-1) - 1).clamp(min=0)[..., :budget]
    source = torch.where(hole[..., :budget], comers.gather(-1, nth), slot[:budget])
    rows = source[..., None].expand(*source.shape, D)
    s.k[..., :budget, :] = s.k.gather(3, rows)
    s.v[..., :budget, :] = s.v.gather(3, rows)
    s.weight[..., :budget] = s.weight.gather(3, source)
    s.position[..., :budget] = s.position.gather(3, source)
    s.counts[0].clamp_(max=budget)
    return s.k, s.v, s.counts, s.position, s.weight


# ---- what a pass cannot do without ----

def work(case):
    Hq, Hk, D = HEADS[case["heads"]]
    B, T = case["B"], case.get("T", 0)
    if case["work"] == "attention":
        Sq, Sk = case["Sq"], case["Sk"]
        pad = case["pad"] if B == 1 else case["pad"] / 2            # the other sequences are padded less
        rows, keys = Sq - pad, Sk - pad
        if case["causal"]:
            # a row sees the keys up to its own, and the prefix
            pairs = rows * (keys - rows) + rows * (rows + 1) / 2
            behind = max(0.0, min(case["prefix"] / (1 if B == 1 else 2), keys) - (keys - rows))
            pairs += behind * (behind - 1) / 2
        else:
            pairs = rows * keys
        if case["docs"]:
            pairs *= 2 / (case["docs"] + 1)   # the mean of the squared shares of lengths cut at random
        return {"bytes": B * 2.0 * D * (2 * rows * Hq + 2 * keys * Hk) + 4.0 * Hq * (2 * case["bias"] + 1),
                "flops": 4.0 * B * Hq * D * pairs}
    if case["work"] == "cached":
        n = case["n"] * (1.0 if not case["ragged"] else (1 + 0.75 * (B - 1)) / B)
        pairs = T * n + (T * (T + 1) / 2 if case["kind"] != "tree" else 4 * T)
        return {"bytes": B * (2.0 * D * (2 * Hk * (n + T) + 2 * T * Hq) + (8.0 * Hk * n if case["weights"] else 0)),
                "flops": 4.0 * B * Hq * D * pairs}
    if case["work"] == "append":
        return {"bytes": 4.0 * B * T * D * (Hq + 2 * Hk), "flops": 3.0 * B * T * D * (Hq + Hk)}
    row = 4.0 * D + 8.0                  # k and v of a slot, its weight and its position
    if case["work"] == "accept":
        return {"bytes": 2 * row * case["layers"] * B * Hk * max(1, case["depth"] - 1), "flops": 0}
    moved = case["budget"] * (1 - case["budget"] / case["n"])
    return {"bytes": case["layers"] * B * Hk * (8.0 * case["n"] + 2 * row * moved), "flops": 0}


# ---- the same from the definitions, in 64 bits ----

def _row_by_row(q, k, v, scale, cap, bias, seen):
    """One head: q [S, D], k and v [N, D] in 64 bits."""
    x = scale * (q @ k.T)
    if cap:
        x = cap * torch.tanh(x / cap)
    if bias is not None:
        x = x + bias
    x = x.masked_fill(~seen, -math.inf)
    empty = ~seen.any(1, keepdim=True)
    p = torch.softmax(x.masked_fill(empty, 0.0), 1).masked_fill(empty, 0.0)
    return p, p @ v


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "cached": _exact_cached, "append": _exact_append,
            "accept": _exact_accept, "evict": _exact_evict}[case["work"]](s)


def _exact_attention(s):
    c = s.case
    B, Sq, Hq, D = s.q.shape
    Sk, Hk = s.k.shape[1], s.k.shape[2]
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        m = int(s.q_lens[b]) if s.q_lens is not None else Sq
        n = int(s.k_lens[b]) if s.k_lens is not None else Sk
        far = torch.arange(n, device="cuda")[None, :] - (torch.arange(m, device="cuda")[:, None] + (n - m))
        seen = torch.ones(m, n, dtype=torch.bool, device="cuda")
        if c["causal"]:
            seen = far <= 0
            if s.prefix is not None:
                seen[:, :int(s.prefix[b])] = True
        if s.docs is not None:
            d = s.docs[b]
            seen = seen & (d[:m, None] == d[None, :n]) & (d[:m, None] >= 0)
        for h in range(Hq):
            g = h // (Hq // Hk)
            bias = None
            if s.bias is not None:
                bias = s.bias[h].double()[far.clamp(-c["bias"], c["bias"]) + c["bias"]]
            out[b, :m, h] = _row_by_row(s.q[b, :m, h].double(), s.k[b, :n, g].double(), s.v[b, :n, g].double(),
                                        s.scale, c["cap"], bias, seen)[1]
    return out


def _exact_cached(s):
    c = s.case
    B, T, Hq, D = s.q.shape
    Hk = s.k.shape[2]
    G = Hq // Hk
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device="cuda")
    weight = s.weight.double()
    for b in range(B):
        n = int(s.counts[0, b])
        seen = torch.ones(T, n + T, dtype=torch.bool, device="cuda")
        if s.tree is None:
            seen = seen.tril(n)
        else:
            bits = [int(m) for m in s.tree[b].tolist()]
            seen[:, n:] = torch.tensor([[bool(m >> u & 1) for u in range(T)] for m in bits], device="cuda")
        for h in range(Hq):
            k, v = s.k[s.layer, b, h // G, :n + T].double(), s.v[s.layer, b, h // G, :n + T].double()
            p, out[b, :, h] = _row_by_row(s.q[b, :, h].double(), k, v, s.scale, c["cap"], None, seen)
            weight[s.layer, b, h // G, :n + T] += p[:c["weights"]].sum(0)
    return (out, weight) if c["weights"] else out


def _exact_append(s):
    B, T, Hq, D = s.q.shape
    k, v, half = s.k.double(), s.v.double(), D // 2
    q = s.q.double()
    freq = s.inv_freq.double()
    for b in range(B):
        n, start = int(s.counts[0, b]), int(s.counts[1, b])
        at = start + (torch.arange(T, device="cuda") if s.depth is None else s.depth[b]).double()
        turn = torch.polar(torch.ones(T, 1, half, dtype=torch.float64, device="cuda"),
                           (at[:, None] * freq[None])[:, None])

        def rotated(x):
            z = turn * torch.complex(x[..., :half].double(), x[..., half:].double())
            return torch.cat((z.real, z.imag), -1)

        q[b] = rotated(s.q[b])
        k[s.layer, b, :, n:n + T] = rotated(s.k_new[b]).transpose(0, 1)
        v[s.layer, b, :, n:n + T] = s.v_new[b].double().transpose(0, 1)
    return q, k, v


def _exact_accept(s):
    counts, position = s.counts.clone(), s.position.clone()
    k, v, weight = s.k.double(), s.v.double(), s.weight.double()
    for b, (line, m) in enumerate(zip(s.path.tolist(), s.count.tolist())):
        n = int(s.counts[0, b])
        from_ = [n + t for t in line[:m]]
        for x, y in ((k, s.k), (v, s.v), (position, s.position), (weight, s.weight)):
            x[:, b, :, n:n + m] = y[:, b, :, from_].to(x.dtype)
        counts[:, b] += m
    return k, v, counts, position, weight


def _exact_evict(s):
    c = s.case
    counts, position = s.counts.clone(), s.position.cpu()
    L, B, Hk, N, D = s.k.shape
    weights = s.weight.cpu()
    source = torch.arange(N).repeat(L, B, Hk, 1)
    for b in range(B):
        n, after = int(s.counts[0, b]), int(s.counts[1, b])
        if n <= c["budget"]:
            continue
        for layer in range(L):
            for h in range(Hk):
                p, w = position[layer, b, h, :n], weights[layer, b, h, :n]
                safe = (p < c["sinks"]) | (p >= after - c["recent"])
                rest = (~safe).nonzero()[:, 0]
                best = rest[torch.argsort(-w[rest].double(), stable=True)][:c["budget"] - int(safe.sum())]
                keep = safe.clone()
                keep[best] = True
                holes = (~keep[:c["budget"]]).nonzero()[:, 0]
                source[layer, b, h, holes] = keep[c["budget"]:].nonzero()[:, 0] + c["budget"]
        counts[0, b] = c["budget"]
    source = source.cuda()
    rows = source[..., None].expand(L, B, Hk, N, D)
    return (s.k.gather(3, rows).double(), s.v.gather(3, rows).double(), counts, s.position.gather(3, source),
            s.weight.gather(3, source).double())
