"""Attention and the key/value cache: Python mirror of include/swiftltx_attention.h.

    attention         whole sequences: score cap, distance bias, causal / prefix / document masks
    attention_cached  new tokens over a cache: decoding, trees of drafted tokens, prompt chunks
    kv_append         rotary embedding of q and k, k and v into the cache
    kv_accept         drafted tokens that were accepted become part of the sequences
    kv_evict          the cache cut to a budget by accumulated attention weight
    KVCache           the cache of all layers of a model, its lengths in device memory

What a decoder layer computes between its q|k|v projection and its output
projection (LlamaModel.swift:336-418, KVCache.swift:7-116), what a text encoder's
layer does with its relative-position bias (T5Encoder.swift:122-213, 360-421), and
a diffusion transformer's bidirectional attention (Ops.swift:2006-2058).

Tensors are fp16 or bf16 on the GPU, their last dimension contiguous; calls run
on `stream` (default: the current stream of the tensors' device), on the device
that the tensors are on.  Errors are SltxError and ValueError as elsewhere.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import sys

_P = sys.modules[__package__]


def _native():
    """The native binding of the plain calls (csrc/py/q4_binding.cpp), or None."""
    if not _P._native_tried:
        _P._load_binding()
    return _P._native


@contextlib.contextmanager
def _launch(t, stream):
    """The device of tensor t and the stream as current ones, for the call and what
    it allocates: yields the stream's handle."""
    import torch
    if stream is None:
        if torch.cuda.current_device() == t.device.index:
            yield torch.cuda.current_stream().cuda_stream
        else:
            with torch.cuda.device(t.device):
                yield torch.cuda.current_stream().cuda_stream
        return
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=t.device)
    if stream.device != t.device:
        raise ValueError(f"stream of {stream.device} for tensors on {t.device}")
    with torch.cuda.stream(stream):
        yield stream.cuda_stream


def _need(t, what, shape, dtypes, device=None, contiguous=True):
    """Checks a tensor handed to the library as a raw pointer."""
    if t is None:
        raise ValueError(f"{what} is None")
    if not getattr(t, "is_cuda", False):
        raise ValueError(f"{what} must be a device tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, the call on {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} has dtype {t.dtype}, expected one of {dtypes}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous (got strides {tuple(t.stride())})")
    if not contiguous and t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what} must be contiguous in its last dimension (got strides {tuple(t.stride())})")
    return t


def _rows(t, what, shape, dtype, device):
    """A [batch, rows, heads, head_dim] tensor of any strides."""
    return _need(t, what, shape, (dtype,), device, contiguous=False)


_I3 = ctypes.c_int64 * 3


def _strides(t):
    """Strides of the first three dimensions; those of dimensions of one are never
    stepped over and need no alignment."""
    return _I3(*(0 if n <= 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])))


def _halves():
    import torch
    return (torch.float16, torch.bfloat16)


def _opt(t, what, shape, dtype, device, empty=None):
    """The address of a tensor, or None.  One of no elements has no address; `empty`
    stands for it where no address would mean no tensor."""
    return None if t is None else _need(t, what, shape, (dtype,), device).data_ptr() or empty


def attention(q, k, v, scale, *, softcap=0.0, bias=None, bias_zero=0, causal=False, prefix=None,
              q_docs=None, k_docs=None, q_lens=None, k_lens=None, out=None, stream=None):
    """softmax(x) v with x = scale q.k, capped (softcap tanh(x / softcap)) and biased
    by distance (bias[h, clamp(j - pos + bias_zero, 0, n - 1)]).

    q [batch, rows, q_heads, head_dim]; k, v [batch, keys, kv_heads, head_dim], any
    strides (columns of one projection, say); bias fp32 [q_heads or 1, n]; the rest
    int32: prefix, q_lens, k_lens [batch], q_docs [batch, rows], k_docs [batch, keys].
    Row i stands at pos = i + k_len - q_len and sees key j < k_len if it is not
    causal or j <= pos or j < prefix, and both are of one document (negative ids:
    of none).  A row that sees nothing gives zeros; rows from q_len on are left as
    they are in `out` (default: a new tensor; with q_lens its last rows are zeros)."""
    native = _native()
    if native is not None:
        r = native.attention(q, k, v, scale, softcap, bias, bias_zero, causal, prefix, q_docs, k_docs, q_lens, k_lens,
                             out, stream)
        if r is not None:
            return r
    import torch
    if q is None or q.dim() != 4 or k is None or k.dim() != 4:
        raise ValueError("q and k are [batch, rows, heads, head_dim] tensors")
    if q.dtype not in _halves():
        raise ValueError(f"q has dtype {q.dtype}, expected one of {_halves()}")
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    dev = q.device
    _rows(q, "q", (B, Sq, Hq, D), q.dtype, None)
    _rows(k, "k", (B, Sk, Hk, D), q.dtype, dev)
    _rows(v, "v", (B, Sk, Hk, D), q.dtype, dev)
    a = _P.CAttentionArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_stride=_strides(q), k_stride=_strides(k),
                         v_stride=_strides(v), dtype=_P._dtype_code(q.dtype), batch=B, q_rows=Sq, k_rows=Sk,
                         q_heads=Hq, kv_heads=Hk, head_dim=D, causal=1 if causal else 0, scale=scale,
                         softcap=softcap)
    if bias is not None:
        if bias.dim() != 2 or bias.shape[0] not in (1, Hq) or bias.shape[1] == 0:
            raise ValueError(f"bias has shape {tuple(bias.shape)}, expected [{Hq} or 1, distances (at least one)]")
        _need(bias, "bias", bias.shape, (torch.float32,), dev)
        a.bias, a.bias_len, a.bias_zero = bias.data_ptr(), bias.shape[1], bias_zero
        a.bias_head_stride = 0 if bias.shape[0] == 1 else bias.shape[1]
    i32 = torch.int32
    a.prefix = _opt(prefix, "prefix", (B,), i32, dev)
    a.q_docs = _opt(q_docs, "q_docs", (B, Sq), i32, dev)
    a.k_docs = _opt(k_docs, "k_docs", (B, Sk), i32, dev, empty=q.data_ptr())   # of no keys
    a.q_lens = _opt(q_lens, "q_lens", (B,), i32, dev)
    a.k_lens = _opt(k_lens, "k_lens", (B,), i32, dev)
    with _launch(q, stream) as handle:
        if out is None:
            new = torch.zeros if q_lens is not None else torch.empty
            out = new(B, Sq, Hq, D, dtype=q.dtype, device=dev)
        _rows(out, "out", (B, Sq, Hq, D), q.dtype, dev)
        a.out, a.out_stride = out.data_ptr(), _strides(out)
        _P.check(_P.lib().sltx_attention(ctypes.byref(a), handle))
    return out


class KVCache:
    """sltx_kv_cache: keys and values of all layers for `batch` sequences, each of
    at most `capacity` entries, fp16 or bf16.

    length and next_position (int32 [batch] device tensors, the rows of `counts`)
    are a sequence's entries and the position of its next token.  track_weights
    keeps, per entry, its position and the attention weight that it has had
    (attention_cached(weight_rows=...)), which kv_evict goes by.

    Every tensor stays in place for the cache's life, so steps over it can be
    captured in a HIP graph; so does every scratch buffer that a call needed (they
    grow: make a captured call once eagerly first, so that its scratch does not
    come from the graph's own memory).  Calls over one cache share its scratch: they
    are ordered like any that write one tensor, on one stream or with events."""

    def __init__(self, layers, batch, kv_heads, capacity, head_dim, dtype=None, track_weights=False, device="cuda"):
        import torch
        dtype = dtype or torch.float16
        k, v = (torch.zeros(layers, batch, kv_heads, capacity, head_dim, dtype=dtype, device=device)
                for _ in range(2))
        weight = position = None
        if track_weights:
            weight = torch.zeros(layers, batch, kv_heads, capacity, dtype=torch.float32, device=device)
            position = torch.zeros(layers, batch, kv_heads, capacity, dtype=torch.int32, device=device)
        self._set(k, v, torch.zeros(2, batch, dtype=torch.int32, device=device), weight, position)
        torch.cuda.current_stream(k.device).synchronize()   # zeroed before other streams use it

    @classmethod
    def from_tensors(cls, k, v, counts, weight=None, position=None):
        """A cache over tensors that the caller keeps: k, v [layers, batch, kv_heads,
        capacity, head_dim], counts int32 [2, batch] (lengths, next positions), weight
        fp32 and position int32 [layers, batch, kv_heads, capacity] (both or neither)."""
        self = cls.__new__(cls)
        self._set(k, v, counts, weight, position)
        return self

    def _set(self, k, v, counts, weight, position):
        import torch
        if k.dim() != 5:
            raise ValueError("k is [layers, batch, kv_heads, capacity, head_dim]")
        _need(k, "k", k.shape, _halves())
        _need(v, "v", k.shape, (k.dtype,), k.device)
        self.layers, self.batch, self.kv_heads, self.capacity, self.head_dim = k.shape
        _need(counts, "counts", (2, self.batch), (torch.int32,), k.device)
        if (weight is None) != (position is None):
            raise ValueError("weight and position go together")
        if weight is not None:
            _need(weight, "weight", k.shape[:4], (torch.float32,), k.device)
            _need(position, "position", k.shape[:4], (torch.int32,), k.device)
        self.k, self.v, self.counts, self.weight, self.position = k, v, counts, weight, position
        self.length, self.next_position = counts[0], counts[1]
        self.dtype, self.device = k.dtype, k.device
        self._scratch = []        # the last one is in use; earlier ones a captured graph may name
        self._needs = {}          # bytes of scratch by call
        self.c = _P.CKVCache(k.data_ptr(), v.data_ptr(), _P._ptr(weight), _P._ptr(position), self.length.data_ptr(),
                            self.next_position.data_ptr(), *k.shape, _P._dtype_code(k.dtype), None, 0)
        self._ref = ctypes.byref(self.c)
        self._handle = (ctypes.addressof(self.c), self.device.index)

    def _workspace(self, name, *args):
        """Scratch for the call, of the size its query names (on the current stream)."""
        key = (name, *args)
        need = self._needs.get(key)
        if need is None:
            need = int(getattr(_P.lib(), name)(self._ref, *args))
            if need < 0:
                _P.check(need)
            self._needs[key] = need
        if need > self.c.workspace_bytes:
            import torch
            need = max(need, 2 * self.c.workspace_bytes)
            self._scratch.append(torch.empty(need, dtype=torch.uint8, device=self.device))
            self.c.workspace, self.c.workspace_bytes = self._scratch[-1].data_ptr(), need

    def reset(self):
        """Empties every sequence (on the current stream)."""
        self.counts.zero_()


def attention_cached(q, cache, layer, scale, *, softcap=0.0, tree=None, weight_rows=0, first=0, out=None,
                     stream=None):
    """Attention of T of the tokens appended to `layer` of the cache (from the first-th
    on): q [batch, T, q_heads, head_dim] -> the same shape, contiguous.  Token t sees the sequence's
    entries, the appended tokens before `first` and those of the call up to itself, or with `tree` (int64 [batch, T], T <=
    64) those whose bit is set in tree[b, t] (tree_masks).  weight_rows: adds the
    attention weights of the first so many tokens to cache.weight (T <= 64)."""
    native = _native()
    if native is not None:
        r = native.attention_cached(q, *cache._handle, layer, first, scale, softcap, tree, weight_rows, out, stream)
        if r is not None:
            return r
    import torch
    if q is None or q.dim() != 4:
        raise ValueError("q is a [batch, tokens, q_heads, head_dim] tensor")
    B, T, Hq, D = q.shape
    _rows(q, "q", (cache.batch, T, Hq, cache.head_dim), cache.dtype, cache.device)
    tree = _opt(tree, "tree", (B, T), torch.int64, cache.device)
    with _launch(q, stream) as handle:
        if out is None:
            out = torch.empty(B, T, Hq, D, dtype=q.dtype, device=q.device)
        _need(out, "out", q.shape, (q.dtype,), q.device)
        cache._workspace("sltx_attention_cached_workspace", T, Hq, weight_rows)
        _P.check(_P.lib().sltx_attention_cached(q.data_ptr(), _strides(q), cache._ref, layer, first, T, Hq, scale,
                                              softcap, tree, weight_rows, out.data_ptr(), handle))
    return out


def kv_append(q, k, v, cache, layer, inv_freq=None, *, depth=None, interleaved=False, q_out=None, stream=None):
    """T new tokens of each sequence into `layer` of the cache, behind its entries:
    q [batch, T, q_heads, head_dim] and k are rotated by (next_position + depth) *
    inv_freq (fp32 [pairs]; None: not rotated), depth int32 [batch, T] (default: 0,
    1, ...: a chain).  Returns the rotated q (contiguous).  Pairs of values are (i,
    i + pairs), or (2i, 2i + 1) if interleaved.  The tokens count once they are
    accepted (kv_accept), after every layer has them."""
    native = _native()
    if native is not None:
        r = native.kv_append(q, k, v, *cache._handle, layer, inv_freq, depth, interleaved, q_out, stream)
        if r is not None:
            return r
    import torch
    if q is None or q.dim() != 4:
        raise ValueError("q is a [batch, tokens, q_heads, head_dim] tensor")
    B, T, Hq, D = q.shape
    _rows(q, "q", (cache.batch, T, Hq, cache.head_dim), cache.dtype, cache.device)
    _rows(k, "k", (B, T, cache.kv_heads, D), cache.dtype, cache.device)
    _rows(v, "v", (B, T, cache.kv_heads, D), cache.dtype, cache.device)
    pairs = 0
    if inv_freq is not None:
        pairs = int(inv_freq.numel())
        inv_freq = _need(inv_freq, "inv_freq", (pairs,), (torch.float32,), cache.device).data_ptr()
    depth = _opt(depth, "depth", (B, T), torch.int32, cache.device)
    with _launch(q, stream) as handle:
        if q_out is None:
            q_out = torch.empty(B, T, Hq, D, dtype=q.dtype, device=q.device)
        _need(q_out, "q_out", q.shape, (q.dtype,), q.device)
        _P.check(_P.lib().sltx_kv_append(q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(),
                                       _strides(v), cache._ref, layer, T, Hq, inv_freq, pairs,
                                       1 if interleaved else 0, depth, q_out.data_ptr(), handle))
    return q_out


def kv_accept(cache, drafted, path=None, count=None, stream=None):
    """Of `drafted` tokens appended in every layer, those of `path` (int32 [batch, n],
    n <= 64: indices among the drafted, root first), the first count[b] of them
    (int32 [batch]; None: all), become the sequences' next entries, up to the
    capacity; without a path the first count[b] (None: all) drafted tokens."""
    native = _native()
    if native is not None and native.kv_accept(*cache._handle, drafted, path, count, stream):
        return
    import torch
    n = 0
    if path is not None:
        if path.dim() != 2:
            raise ValueError("path is an int32 [batch, n] tensor")
        n = int(path.shape[1])
        path = _opt(path, "path", (cache.batch, n), torch.int32, cache.device, empty=cache.length.data_ptr())
    count = _opt(count, "count", (cache.batch,), torch.int32, cache.device)
    with _launch(cache.k, stream) as handle:
        _P.check(_P.lib().sltx_kv_accept(cache._ref, drafted, path, n, count, handle))


def kv_evict(cache, budget, *, sinks=4, recent=32, stream=None):
    """Cuts every sequence to `budget` entries, in each layer and head on its own:
    the first `sinks` and the last `recent` positions stay, and of the rest those
    with the highest accumulated attention weight (ties: the lower slots).  Entries
    that stay move only into slots that became free."""
    native = _native()
    if native is not None and native.kv_evict(*cache._handle, budget, sinks, recent, stream):
        return
    with _launch(cache.k, stream) as handle:
        cache._workspace("sltx_kv_evict_workspace", budget)
        _P.check(_P.lib().sltx_kv_evict(cache._ref, budget, sinks, recent, handle))


class CachedAttention:
    """What DecodeStep and PrefillStep do between a layer's q|k|v projection and its
    output projection, over a KVCache of one sequence: rotary embedding, keys and
    values into the cache, causal attention over it; finish() then counts the tokens
    (and cuts the cache to `budget` entries).

    config: a ModelConfig (heads, head_dim, rope_theta, rope_scaling).  A cache that
    tracks weights gets those of each decoded token and of a prompt's last 64.
    softcap: the cap of the scores (0: none).  sinks, recent: as in kv_evict.  A
    budget is below the cache's capacity."""

    WINDOW = 64    # tokens of a prompt whose attention weights count

    def __init__(self, config, cache, stream=None, *, budget=None, sinks=4, recent=32, softcap=0.0):
        c = config
        want = (c.num_hidden_layers, 1, c.num_key_value_heads, c.head_dim)
        if (cache.layers, cache.batch, cache.kv_heads, cache.head_dim) != want:
            raise ValueError(f"a cache of {want[0]} layers, one sequence, {want[2]} heads of {want[3]} is needed, not "
                             f"{cache.layers}, {cache.batch}, {cache.kv_heads}, {cache.head_dim}")
        if cache.dtype != _halves()[0]:
            raise ValueError(f"the projections are fp16, the cache {cache.dtype}")
        if budget is not None:
            if cache.weight is None:
                raise ValueError("a budget needs a cache that tracks weights")
            if not 0 < budget < cache.capacity:
                raise ValueError(f"a budget of {budget} entries in a capacity of {cache.capacity}, which needs room for "
                                 "the next token beside them")
            if sinks < 0 or recent < 0 or sinks + recent > budget:
                raise ValueError(f"{sinks} first and {recent} recent positions in a budget of {budget}")
        self.cache, self.stream, self.softcap = cache, stream, float(softcap)
        self.heads, self.kv_heads, self.head_dim = c.num_attention_heads, c.num_key_value_heads, c.head_dim
        self.scale = 1.0 / math.sqrt(c.head_dim)
        self.inv_freq = rope_inv_freq(c.head_dim, c.rope_theta, c.rope_scaling, device=cache.device)
        self.budget, self.sinks, self.recent = budget, sinks, recent

    def __call__(self, layer, qkv):
        """[T, q+k+v] fp16 projections of the next T tokens -> [T, heads * head_dim]."""
        import torch
        T, H, K, s = qkv.shape[0], self.heads, self.kv_heads, self.stream
        x = qkv.view(1, T, H + 2 * K, self.head_dim)
        q = kv_append(x[:, :, :H], x[:, :, H:H + K], x[:, :, H + K:], self.cache, layer, self.inv_freq, stream=s)
        cap = self.softcap
        if self.cache.weight is None or T <= self.WINDOW:
            rows = 0 if self.cache.weight is None else T
            out = attention_cached(q, self.cache, layer, self.scale, softcap=cap, weight_rows=rows, stream=s)
        else:          # the last tokens in a call of their own, which adds their weights
            n = T - self.WINDOW
            out = torch.empty_like(q)
            attention_cached(q[:, :n], self.cache, layer, self.scale, softcap=cap, out=out[:, :n], stream=s)
            attention_cached(q[:, n:], self.cache, layer, self.scale, softcap=cap, weight_rows=self.WINDOW, first=n,
                             out=out[:, n:], stream=s)
        return out.view(T, H * self.head_dim)

    def finish(self, tokens):
        """After the last layer: the tokens become entries."""
        kv_accept(self.cache, tokens, stream=self.stream)
        if self.budget is not None:
            kv_evict(self.cache, self.budget, sinks=self.sinks, recent=self.recent, stream=self.stream)


# ---- what a program prepares once ----

def rope_inv_freq(head_dim, theta=10000.0, scaling=None, device="cuda"):
    """fp32 [head_dim / 2] rotary frequencies theta^(-2i / head_dim), and with a
    config.json `rope_scaling` of type "llama3" its interpolation of the long
    wavelengths ("linear": all of them)."""
    import torch
    f = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    if scaling:
        kind = scaling.get("rope_type", scaling.get("type"))
        factor = float(scaling.get("factor", 1.0))
        if kind == "linear":
            f = f / factor
        elif kind == "llama3":
            low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
            turns = f * float(scaling["original_max_position_embeddings"]) / (2 * math.pi)
            smooth = ((turns - low) / (high - low)).clamp(0, 1)
            f = f * (smooth + (1 - smooth) / factor)
        elif kind not in (None, "default"):
            raise ValueError(f"rope scaling {kind!r} is not known")
    return f.float().to(device)


def distance_bias(table, max_distance=128, bidirectional=True):
    """(bias fp32 [heads, n], bias_zero) of a text encoder's relative-position table
    [buckets, heads] (T5Encoder.swift:360-421): near distances have a bucket each,
    farther ones share buckets of equal log width up to max_distance, beyond which
    all share the last; the two directions have half the buckets each."""
    import torch
    buckets = table.shape[0]
    d = torch.arange(-max_distance, max_distance + 1)       # key - query
    half = buckets // 2 if bidirectional else buckets
    far = d.abs() if bidirectional else (-d).clamp(min=0)
    exact = half // 2
    log = exact + (torch.log(far.clamp(min=1).double() / exact) / math.log(max_distance / exact)
                   * (half - exact)).to(torch.int64)
    bucket = torch.where(far < exact, far, log.clamp(max=half - 1))
    if bidirectional:
        bucket = bucket + (d > 0) * half
    return table.float()[bucket.to(table.device)].t().contiguous(), max_distance


def tree_masks(parents, device="cuda"):
    """(tree int64 [batch, T], depth int32 [batch, T]) for attention_cached and
    kv_append, of host lists parents[b][t]: the drafted token that token t follows
    (-1: the sequence itself), always an earlier one."""
    import torch
    masks, depths = [], []
    for row in parents:
        m, d = [], []
        if len(row) > 64:
            raise ValueError(f"a tree of {len(row)} tokens (64 at most)")
        for t, up in enumerate(row):
            if not -1 <= up < t:
                raise ValueError(f"token {t} follows {up}, which is not an earlier one")
            m.append((m[up] if up >= 0 else 0) | 1 << t)
            d.append(d[up] + 1 if up >= 0 else 0)
        masks.append([x - (1 << 64) if x >> 63 else x for x in m])
        depths.append(d)
    return (torch.tensor(masks, dtype=torch.int64, device=device),
            torch.tensor(depths, dtype=torch.int32, device=device))
