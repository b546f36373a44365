// attn_capi.hip -- the C ABI of include/swiftltx_attention.h: argument
// validation, the choice of kernel, launches.  Validation runs before any HIP
// call.
#include <algorithm>
#include <array>
#include <cmath>
#include <utility>

#include "attn_launch.hpp"
#include "q4_common.hpp"
#include "q4_launch.hpp"
#include "swiftltx_attention.h"

namespace sltx {
namespace {

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int done(hipError_t e, const char* fn) {
    return e == hipSuccess ? kOk : set_error(kErrHip, "%s: %s", fn, hipGetErrorString(e));
}

constexpr int kMaxRows = 1 << 28;   // rows or keys of one sequence

// A [batch, rows, heads, head_dim] tensor of 16-bit elements.
struct Tensor {
    const char* name;
    const void* p;
    const int64_t* stride;
    int64_t batch, rows, heads, dim;
    // bytes from the first element to past the last
    size_t span() const {
        return 2 * (size_t)((batch - 1) * stride[0] + (rows - 1) * stride[1] + (heads - 1) * stride[2] + dim);
    }
};

int check_tensor(const char* fn, const Tensor& t) {
    if (!t.p) return set_error(kErrInvalid, "%s: %s is null", fn, t.name);
    if (!aligned(t.p, 16)) return set_error(kErrInvalid, "%s: %s must be 16-byte aligned", fn, t.name);
    for (int i = 0; i < 3; ++i)
        if (t.stride[i] < 0 || t.stride[i] % 8 != 0 || t.stride[i] > ((int64_t)1 << 40))
            return set_error(kErrInvalid, "%s: stride %lld of %s is not a multiple of 8 in [0, 2^40]", fn,
                             (long long)t.stride[i], t.name);
    return kOk;
}
// 64 rows within the 2 GB that a tile's buffer addresses
int check_rows_span(const char* fn, const Tensor& t) {
    if (t.stride[1] >= (1 << 24))
        return set_error(kErrUnsupported, "%s: row stride %lld of %s is above 2^24", fn, (long long)t.stride[1], t.name);
    return kOk;
}
bool overlap(const Tensor& a, const Tensor& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return x < y + b.span() && y < x + a.span();
}

// Whether rows of a tensor share memory: its dimensions, from the smallest stride on,
// have to step over all of those before.
bool rows_share(const Tensor& t) {
    std::array<std::pair<int64_t, int64_t>, 3> dims = {
        {{t.stride[0], t.batch}, {t.stride[1], t.rows}, {t.stride[2], t.heads}}};
    std::sort(dims.begin(), dims.end());
    int64_t span = t.dim;
    for (const auto& [stride, n] : dims) {
        if (n <= 1) continue;
        if (stride < span) return true;
        span += stride * (n - 1);
    }
    return false;
}

int check_heads(const char* fn, int dtype, int q_heads, int kv_heads, int head_dim) {
    if (dtype != SLTX_F16 && dtype != SLTX_BF16)
        return set_error(kErrInvalid, "%s: dtype %d must be SLTX_F16 or SLTX_BF16", fn, dtype);
    if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0)
        return set_error(kErrInvalid, "%s: %d query heads are not a multiple of %d key/value heads", fn, q_heads, kv_heads);
    if (head_dim <= 0 || head_dim % 8 != 0)
        return set_error(kErrInvalid, "%s: head_dim %d is not a positive multiple of 8", fn, head_dim);
    if (head_dim > 128) return set_error(kErrUnsupported, "%s: head_dim %d is above 128", fn, head_dim);
    return kOk;
}
int check_scores(const char* fn, float scale, float softcap) {
    if (!(scale > 0.0f) || !std::isfinite(scale))
        return set_error(kErrInvalid, "%s: scale must be positive and finite", fn);
    if (!(softcap >= 0.0f) || !std::isfinite(softcap))
        return set_error(kErrInvalid, "%s: softcap must be finite and not negative (0: none)", fn);
    // what the kernels form of them: 2 log2(e) scale / softcap, 2 log2(e) softcap
    if (!std::isfinite(3.0f * scale) || !std::isfinite(3.0f * softcap) ||
        (softcap > 0.0f && !std::isfinite(3.0f * scale / softcap)))
        return set_error(kErrUnsupported, "%s: scale %g with softcap %g leaves fp32's range", fn, scale, softcap);
    return kOk;
}

int check_cache(const char* fn, const sltx_kv_cache* c, bool pointers = true) {
    if (!c) return set_error(kErrInvalid, "%s: cache is null", fn);
    if (c->layers <= 0 || c->batch < 0 || c->capacity <= 0)
        return set_error(kErrInvalid, "%s: a cache of %d layers, batch %d and capacity %d", fn, c->layers, c->batch,
                         c->capacity);
    const int rc = check_heads(fn, c->dtype, c->kv_heads, c->kv_heads, c->head_dim);
    if (rc != kOk) return rc;
    if (c->capacity > kMaxRows || (int64_t)c->layers * c->batch * c->kv_heads > 65535)
        return set_error(kErrUnsupported, "%s: a cache of %d slots and %d layers x %d sequences x %d heads", fn,
                         c->capacity, c->layers, c->batch, c->kv_heads);
    if (!pointers || c->batch == 0) return kOk;
    if (!c->k || !c->v || !c->length || !c->next_position)
        return set_error(kErrInvalid, "%s: null pointer in the cache", fn);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->length, 4) || !aligned(c->next_position, 4) ||
        !aligned(c->weight, 4) || !aligned(c->position, 4) || !aligned(c->workspace, 16))
        return set_error(kErrInvalid, "%s: misaligned pointer in the cache", fn);
    if ((c->weight == nullptr) != (c->position == nullptr))
        return set_error(kErrInvalid, "%s: weight and position go together", fn);
    return kOk;
}
int check_layer(const char* fn, const sltx_kv_cache* c, int layer, int tokens) {
    if (layer < 0 || layer >= c->layers)
        return set_error(kErrInvalid, "%s: layer %d of %d", fn, layer, c->layers);
    if (tokens < 0) return set_error(kErrInvalid, "%s: %d tokens", fn, tokens);
    if (tokens > kMaxRows) return set_error(kErrUnsupported, "%s: %d tokens", fn, tokens);
    return kOk;
}
CacheParams cache_params(const sltx_kv_cache* c) {
    return {static_cast<uint16_t*>(c->k), static_cast<uint16_t*>(c->v), c->weight, c->position, c->length,
            c->next_position, c->layers, c->batch, c->kv_heads, c->capacity, c->head_dim};
}
int need_workspace(const char* fn, const sltx_kv_cache* c, size_t bytes) {
    if (bytes > 0 && (!c->workspace || c->workspace_bytes < bytes))
        return set_error(kErrInvalid, "%s: the cache's workspace holds %llu bytes, %llu needed", fn,
                         c->workspace ? (unsigned long long)c->workspace_bytes : 0ull, (unsigned long long)bytes);
    return kOk;
}

// How sltx_attention_cached runs: the kernel of few rows, or the one of many,
// and over how many ranges of keys.  The lengths are on the device, so the
// ranges go by the capacity.
struct CachedPlan {
    bool few, parts;
    int splits;
    int score_rows, score_pitch;   // scores kept for the weights' sums, or 0
    size_t part_bytes, row_bytes, shares, score, bytes;   // shares, score: where they start
};
CachedPlan cached_plan(const sltx_kv_cache* c, int tokens, int q_heads, int weight_rows) {
    CachedPlan p{};
    const int64_t pack = q_heads / c->kv_heads, rows = pack * tokens, heads = (int64_t)c->batch * c->kv_heads;
    p.few = rows <= kFewRows;
    int64_t splits;
    if (p.few) {
        // as many blocks as run at once: one on a CU at head_dim 128 (eight sequences of
        // 3000 keys 26.0 us, with twice as many blocks 31.2), two at 64
        splits = std::min<int64_t>({(c->head_dim > 64 ? 256 : 512) / heads, (c->capacity + kFewKeys - 1) / kFewKeys, kMostSplits});
    } else {
        // a tree's rows share blocks of 128 (or 64), in as many ranges of keys as fill
        // the GPU twice; more tokens only where even blocks of 64 rows leave CUs idle
        const int64_t blocks = heads * ((rows + kSeqTileRows - 1) / kSeqTileRows);
        splits = tokens <= 64 || 2 * blocks < kCUs ? std::min<int64_t>({512 / blocks, c->capacity / (4 * kTileKeys), 64}) : 1;
    }
    p.splits = (int)std::max<int64_t>(1, splits);
    // the kernel of many rows takes a tree (at most 64 tokens) only in parts
    p.parts = p.splits > 1 || weight_rows > 0 || (!p.few && tokens <= 64);
    if (p.parts) {
        const int64_t dt = c->head_dim > 64 ? 128 : 64;
        p.part_bytes = (size_t)(heads * rows * p.splits) * (size_t)(dt + 2) * sizeof(float);
        p.row_bytes = (size_t)(heads * rows + 1) / 2 * 2 * 2 * sizeof(float);   // a multiple of 16
        p.bytes = p.part_bytes = (p.part_bytes + 15) / 16 * 16;
        p.bytes += p.row_bytes;
        p.shares = p.bytes;
        p.bytes += ((size_t)c->batch * 2 * sizeof(int32_t) + 15) / 16 * 16;
        p.score = p.bytes;
        if (weight_rows > 0 && weight_rows * pack <= kScoreRows) {
            p.score_rows = (int)(weight_rows * pack);
            p.score_pitch = (c->capacity + kFewKeys - 1) / kFewKeys * kFewKeys;
            p.bytes += (size_t)heads * p.score_rows * p.score_pitch * sizeof(float);
        }
    }
    return p;
}

}  // namespace
}  // namespace sltx

using namespace sltx;

extern "C" {

int sltx_attention(const sltx_attention_args* a, void* stream) {
    const char* fn = "sltx_attention";
    if (!a) return set_error(kErrInvalid, "%s: args is null", fn);
    int rc = check_heads(fn, a->dtype, a->q_heads, a->kv_heads, a->head_dim);
    if (rc != kOk || (rc = check_scores(fn, a->scale, a->softcap)) != kOk) return rc;
    if (a->batch < 0 || a->q_rows < 0 || a->k_rows < 0)
        return set_error(kErrInvalid, "%s: batch %d, %d rows, %d keys", fn, a->batch, a->q_rows, a->k_rows);
    if (a->q_rows > kMaxRows || a->k_rows > kMaxRows || a->q_heads > 65535)
        return set_error(kErrUnsupported, "%s: more than 2^28 rows or keys or 65535 heads", fn);
    if (a->batch == 0 || a->q_rows == 0) return kOk;
    const Tensor q = {"q", a->q, a->q_stride, a->batch, a->q_rows, a->q_heads, a->head_dim};
    const Tensor k = {"k", a->k, a->k_stride, a->batch, a->k_rows, a->kv_heads, a->head_dim};
    const Tensor v = {"v", a->v, a->v_stride, a->batch, a->k_rows, a->kv_heads, a->head_dim};
    const Tensor out = {"out", a->out, a->out_stride, a->batch, a->q_rows, a->q_heads, a->head_dim};
    if ((rc = check_tensor(fn, q)) != kOk || (rc = check_tensor(fn, out)) != kOk) return rc;
    if (a->k_rows > 0 && ((rc = check_tensor(fn, k)) != kOk || (rc = check_tensor(fn, v)) != kOk ||
                          (rc = check_rows_span(fn, k)) != kOk || (rc = check_rows_span(fn, v)) != kOk))
        return rc;
    if (overlap(out, q) || (a->k_rows > 0 && (overlap(out, k) || overlap(out, v))))
        return set_error(kErrInvalid, "%s: out overlaps q, k or v", fn);
    if (rows_share(out)) return set_error(kErrInvalid, "%s: out's rows overlap each other", fn);
    if (a->bias && (a->bias_len <= 0 || a->bias_zero < 0 || a->bias_zero >= a->bias_len || a->bias_head_stride < 0))
        return set_error(kErrInvalid, "%s: bias of %d values with distance 0 at %d", fn, a->bias_len, a->bias_zero);
    if (a->bias && a->bias_len > (1 << 30))
        return set_error(kErrUnsupported, "%s: a bias of %d distances", fn, a->bias_len);
    if (a->prefix && !a->causal) return set_error(kErrInvalid, "%s: a prefix needs causal", fn);
    if ((a->q_docs == nullptr) != (a->k_docs == nullptr))
        return set_error(kErrInvalid, "%s: q_docs and k_docs go together", fn);
    for (const void* p : {(const void*)a->bias, (const void*)a->prefix, (const void*)a->q_docs, (const void*)a->k_docs,
                          (const void*)a->q_lens, (const void*)a->k_lens})
        if (!aligned(p, 4)) return set_error(kErrInvalid, "%s: misaligned pointer", fn);
    if ((rc = require_device()) != kOk) return rc;
    AttnParams p{};
    p.q = static_cast<const uint16_t*>(a->q);
    p.k = static_cast<const uint16_t*>(a->k);
    p.v = static_cast<const uint16_t*>(a->v);
    p.out = static_cast<uint16_t*>(a->out);
    p.qs = {a->q_stride[0], a->q_stride[1], a->q_stride[2]};
    p.ks = {a->k_stride[0], a->k_stride[1], a->k_stride[2]};
    p.vs = {a->v_stride[0], a->v_stride[1], a->v_stride[2]};
    p.os = {a->out_stride[0], a->out_stride[1], a->out_stride[2]};
    p.B = a->batch;
    p.Sq = a->q_rows;
    p.Sk = a->k_rows;
    p.Hq = a->q_heads;
    p.Hk = a->kv_heads;
    p.D = a->head_dim;
    p.bf16 = a->dtype == SLTX_BF16;
    p.scale = a->scale;
    p.cap = a->softcap;
    p.bias = a->bias;
    p.bias_h = a->bias_head_stride;
    p.bias_n = a->bias_len;
    p.bias_zero = a->bias_zero;
    p.causal = a->causal != 0;
    p.prefix = a->prefix;
    p.q_docs = a->q_docs;
    p.k_docs = a->k_docs;
    p.q_lens = a->q_lens;
    p.k_lens = a->k_lens;
    p.pack = 1;
    p.heads = a->q_heads;
    p.splits = 1;
    return done(launch_attn_seq(p, static_cast<hipStream_t>(stream)), fn);
}

int64_t sltx_attention_cached_workspace(const sltx_kv_cache* cache, int32_t tokens, int32_t q_heads,
                                        int32_t weight_rows) {
    const char* fn = "sltx_attention_cached_workspace";
    int rc = check_cache(fn, cache, false);
    if (rc != kOk || (rc = check_layer(fn, cache, 0, tokens)) != kOk ||
        (rc = check_heads(fn, cache->dtype, q_heads, cache->kv_heads, cache->head_dim)) != kOk)
        return rc;
    if (cache->batch == 0 || tokens == 0) return 0;
    return (int64_t)cached_plan(cache, tokens, q_heads, weight_rows).bytes;
}

int sltx_attention_cached(const void* q, const int64_t q_stride[3], const sltx_kv_cache* cache, int32_t layer,
                          int32_t first, int32_t tokens, int32_t q_heads, float scale, float softcap, const uint64_t* tree,
                          int32_t weight_rows, void* out, void* stream) {
    const char* fn = "sltx_attention_cached";
    int rc = check_cache(fn, cache);
    if (rc != kOk || (rc = check_layer(fn, cache, layer, tokens)) != kOk ||
        (rc = check_heads(fn, cache->dtype, q_heads, cache->kv_heads, cache->head_dim)) != kOk ||
        (rc = check_scores(fn, scale, softcap)) != kOk)
        return rc;
    if (first < 0 || first > kMaxRows) return set_error(kErrInvalid, "%s: first token %d", fn, first);
    if ((int64_t)tokens * (q_heads / cache->kv_heads) > kMaxRows)
        return set_error(kErrUnsupported, "%s: %d tokens of %d query heads for each key/value head", fn, tokens,
                         q_heads / cache->kv_heads);
    if (tree && tokens > 64) return set_error(kErrInvalid, "%s: a tree of %d tokens (64 at most)", fn, tokens);
    if (weight_rows < 0 || weight_rows > tokens)
        return set_error(kErrInvalid, "%s: weights of %d of %d tokens", fn, weight_rows, tokens);
    if (weight_rows > 0 && tokens > 64)
        return set_error(kErrUnsupported, "%s: weights of a call of %d tokens (64 at most)", fn, tokens);
    if (weight_rows > 0 && !cache->weight && cache->batch > 0)
        return set_error(kErrInvalid, "%s: the cache has no weight", fn);
    if (cache->batch == 0 || tokens == 0) return kOk;
    if (!q_stride) return set_error(kErrInvalid, "%s: q_stride is null", fn);
    const int D = cache->head_dim;
    const Tensor tq = {"q", q, q_stride, cache->batch, tokens, q_heads, D};
    const int64_t ostride[3] = {(int64_t)tokens * q_heads * D, (int64_t)q_heads * D, D};
    const Tensor to = {"out", out, ostride, cache->batch, tokens, q_heads, D};
    if ((rc = check_tensor(fn, tq)) != kOk || (rc = check_tensor(fn, to)) != kOk) return rc;
    const int64_t cstride[3] = {0, 0, 0};
    const int64_t total = (int64_t)cache->layers * cache->batch * cache->kv_heads * cache->capacity * D;
    const Tensor tk = {"k", cache->k, cstride, 1, 1, 1, total}, tv = {"v", cache->v, cstride, 1, 1, 1, total};
    if (overlap(to, tq) || overlap(to, tk) || overlap(to, tv))
        return set_error(kErrInvalid, "%s: out overlaps q or the cache", fn);
    if (!aligned(tree, 8)) return set_error(kErrInvalid, "%s: tree must be 8-byte aligned", fn);
    const CachedPlan plan = cached_plan(cache, tokens, q_heads, weight_rows);
    if ((rc = need_workspace(fn, cache, plan.bytes)) != kOk) return rc;
    if ((rc = require_device()) != kOk) return rc;
    AttnParams p{};
    const int64_t head = (int64_t)cache->capacity * D, seq = head * cache->kv_heads;
    p.q = static_cast<const uint16_t*>(q);
    p.k = static_cast<const uint16_t*>(cache->k) + layer * seq * cache->batch;
    p.v = static_cast<const uint16_t*>(cache->v) + layer * seq * cache->batch;
    p.out = static_cast<uint16_t*>(out);
    p.qs = {q_stride[0], q_stride[1], q_stride[2]};
    p.ks = p.vs = {seq, D, head};
    p.os = {ostride[0], ostride[1], ostride[2]};
    p.B = cache->batch;
    p.Sq = tokens;
    p.Sk = cache->capacity;
    p.Hq = q_heads;
    p.Hk = cache->kv_heads;
    p.D = D;
    p.bf16 = cache->dtype == SLTX_BF16;
    p.scale = scale;
    p.cap = softcap;
    p.causal = tree == nullptr;
    p.k_lens = cache->length;
    p.cached = 1;
    p.first = first;
    p.tree = tree;
    p.pack = q_heads / cache->kv_heads;
    p.heads = cache->kv_heads;
    p.splits = plan.splits;
    p.unit_bits = __builtin_ctz(plan.few ? kFewKeys : kTileKeys);
    if (plan.parts) {
        const int64_t rows = (int64_t)p.B * p.heads * tokens * p.pack;
        p.part_o = static_cast<float*>(cache->workspace);
        p.part_ml = p.part_o + rows * p.splits * (D > 64 ? 128 : 64);
        char* after = static_cast<char*>(cache->workspace) + plan.part_bytes;
        p.shares = reinterpret_cast<int32_t*>(static_cast<char*>(cache->workspace) + plan.shares);
        if (plan.score_rows > 0) {
            p.scores = reinterpret_cast<float*>(static_cast<char*>(cache->workspace) + plan.score);
            p.score_rows = plan.score_rows;
            p.score_pitch = plan.score_pitch;
        } else if (weight_rows > 0) {
            p.row_ml = reinterpret_cast<float*>(after);
        }
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* weight = weight_rows > 0 ? cache->weight + (int64_t)layer * p.B * p.heads * cache->capacity : nullptr;
    hipError_t e = plan.few ? launch_attn_few(p, st) : launch_attn_seq(p, st);
    if (e == hipSuccess && plan.parts) e = launch_attn_finish(p, weight, st);
    if (e == hipSuccess && p.row_ml) e = launch_attn_weights(p, weight, weight_rows, st);
    return done(e, fn);
}

int sltx_kv_append(const void* q, const int64_t q_stride[3], const void* k, const int64_t k_stride[3], const void* v,
                   const int64_t v_stride[3], const sltx_kv_cache* cache, int32_t layer, int32_t tokens,
                   int32_t q_heads, const float* inv_freq, int32_t pairs, int32_t interleaved, const int32_t* depth,
                   void* q_out, void* stream) {
    const char* fn = "sltx_kv_append";
    int rc = check_cache(fn, cache);
    if (rc != kOk || (rc = check_layer(fn, cache, layer, tokens)) != kOk ||
        (rc = check_heads(fn, cache->dtype, q_heads, cache->kv_heads, cache->head_dim)) != kOk)
        return rc;
    if (pairs < 0 || 2 * (int64_t)pairs > cache->head_dim)
        return set_error(kErrInvalid, "%s: %d rotated pairs in a head_dim of %d", fn, pairs, cache->head_dim);
    if (pairs > 0 && (!inv_freq || !aligned(inv_freq, 4)))
        return set_error(kErrInvalid, "%s: inv_freq is null or misaligned", fn);
    if (cache->batch == 0 || tokens == 0) return kOk;
    if (!q_stride || !k_stride || !v_stride) return set_error(kErrInvalid, "%s: a stride array is null", fn);
    const int D = cache->head_dim, B = cache->batch;
    const int64_t ostride[3] = {(int64_t)tokens * q_heads * D, (int64_t)q_heads * D, D}, cstride[3] = {0, 0, 0};
    const int64_t total = (int64_t)cache->layers * B * cache->kv_heads * cache->capacity * D;
    const Tensor in[3] = {{"q", q, q_stride, B, tokens, q_heads, D},
                          {"k", k, k_stride, B, tokens, cache->kv_heads, D},
                          {"v", v, v_stride, B, tokens, cache->kv_heads, D}};
    const Tensor to = {"q_out", q_out, ostride, B, tokens, q_heads, D};
    const Tensor tk = {"k", cache->k, cstride, 1, 1, 1, total}, tv = {"v", cache->v, cstride, 1, 1, 1, total};
    if ((rc = check_tensor(fn, to)) != kOk) return rc;
    for (const Tensor& t : in) {
        if ((rc = check_tensor(fn, t)) != kOk) return rc;
        if (overlap(to, t)) return set_error(kErrInvalid, "%s: q_out overlaps %s", fn, t.name);
        if (overlap(t, tk) || overlap(t, tv)) return set_error(kErrInvalid, "%s: %s overlaps the cache", fn, t.name);
    }
    if (overlap(to, tk) || overlap(to, tv)) return set_error(kErrInvalid, "%s: q_out overlaps the cache", fn);
    if (overlap(tk, tv)) return set_error(kErrInvalid, "%s: k and v of the cache overlap", fn);
    if (!aligned(depth, 4)) return set_error(kErrInvalid, "%s: misaligned depth", fn);
    if ((rc = require_device()) != kOk) return rc;
    AppendParams p{};
    p.c = cache_params(cache);
    p.layer = layer;
    p.q = static_cast<const uint16_t*>(q);
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.q_out = static_cast<uint16_t*>(q_out);
    p.qs = {q_stride[0], q_stride[1], q_stride[2]};
    p.ks = {k_stride[0], k_stride[1], k_stride[2]};
    p.vs = {v_stride[0], v_stride[1], v_stride[2]};
    p.T = tokens;
    p.Hq = q_heads;
    p.bf16 = cache->dtype == SLTX_BF16;
    p.inv_freq = inv_freq;
    p.pairs = pairs;
    p.interleaved = interleaved != 0;
    p.depth = depth;
    return done(launch_kv_append(p, static_cast<hipStream_t>(stream)), fn);
}

int sltx_kv_accept(const sltx_kv_cache* cache, int32_t drafted, const int32_t* path, int32_t path_len,
                   const int32_t* count, void* stream) {
    const char* fn = "sltx_kv_accept";
    int rc = check_cache(fn, cache);
    if (rc != kOk) return rc;
    if (drafted < 0) return set_error(kErrInvalid, "%s: %d drafted tokens", fn, drafted);
    if (path && (path_len < 0 || path_len > 64))
        return set_error(kErrInvalid, "%s: a path of %d tokens (64 at most)", fn, path_len);
    if (!aligned(path, 4) || !aligned(count, 4)) return set_error(kErrInvalid, "%s: misaligned pointer", fn);
    if (cache->batch == 0 || drafted == 0 || (path && path_len == 0)) return kOk;
    if ((rc = require_device()) != kOk) return rc;
    return done(launch_kv_accept(cache_params(cache), drafted, path, path_len, count, static_cast<hipStream_t>(stream)),
                fn);
}

static int check_evict(const char* fn, const sltx_kv_cache* cache, int budget) {
    if (budget <= 0 || budget > cache->capacity)
        return set_error(kErrInvalid, "%s: a budget of %d in a capacity of %d", fn, budget, cache->capacity);
    return kOk;
}

int64_t sltx_kv_evict_workspace(const sltx_kv_cache* cache, int32_t budget) {
    const char* fn = "sltx_kv_evict_workspace";
    int rc = check_cache(fn, cache, false);
    if (rc != kOk || (rc = check_evict(fn, cache, budget)) != kOk) return rc;
    return (int64_t)kv_evict_workspace_bytes(cache_params(cache), budget);
}

int sltx_kv_evict(const sltx_kv_cache* cache, int32_t budget, int32_t sinks, int32_t recent, void* stream) {
    const char* fn = "sltx_kv_evict";
    int rc = check_cache(fn, cache);
    if (rc != kOk || (rc = check_evict(fn, cache, budget)) != kOk) return rc;
    if (cache->batch > 0 && !cache->weight) return set_error(kErrInvalid, "%s: the cache has no weight", fn);
    if (sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
        return set_error(kErrInvalid, "%s: %d first and %d recent positions in a budget of %d", fn, sinks, recent, budget);
    if (cache->batch == 0) return kOk;
    const CacheParams c = cache_params(cache);
    if ((rc = need_workspace(fn, cache, kv_evict_workspace_bytes(c, budget))) != kOk) return rc;
    if ((rc = require_device()) != kOk) return rc;
    return done(launch_kv_evict(c, budget, sinks, recent, cache->workspace, static_cast<hipStream_t>(stream)), fn);
}

}  // extern "C"
