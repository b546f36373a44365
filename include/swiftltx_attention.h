/*
 * swiftltx_attention.h -- C ABI of attention and the key/value cache on MI355X
 * (gfx950): what a decoder layer, a text encoder layer or a diffusion
 * transformer block computes between its q|k|v and its output projection
 * (swiftltx_q4.h).  In the reference these are RoPE, KVCache.swift and a
 * metal-flash-attention kernel (LlamaModel.swift:336-418, T5Encoder.swift:360-421,
 * Ops.swift:2006-2058); the operators here also cover score capping, documents,
 * prefixes, drafted token trees and eviction, which the reference does not have.
 *
 * Conventions of swiftltx_q4.h hold (device pointers, status codes, streams,
 * nothing synchronises, validation before any launch), and:
 *   - Elements are SLTX_F16 or SLTX_BF16, of one type in a call.  Scores, softmax
 *     statistics and sums are fp32; softmax weights are rounded to the element
 *     type before they meet v, the output once more.  An fp16 weight keeps its 11
 *     binary digits down to 2^-22 of the row's largest, and counts as nothing below
 *     2^-33 of it.
 *   - head_dim is a multiple of 8, at most 128.  q_heads is a multiple of
 *     kv_heads; query head h reads key/value head h / (q_heads / kv_heads).
 *   - Strides are in elements, of dimensions batch, row and head; head_dim is
 *     contiguous.  Strides of inputs are multiples of 8, may be 0 (broadcast)
 *     and may interleave (columns of one q|k|v projection); data pointers are
 *     16-byte aligned; 64 rows of k or v span less than 2 GB.
 *   - Up to 2^28 rows or keys of a sequence (rows: tokens times the query heads of a
 *     key/value head, over a cache), 2^28 slots of a cache, 65535 query heads in
 *     sltx_attention and 65535 layers x sequences x heads of a cache; row strides of k and v below
 *     2^24.  More is SLTX_ERR_UNSUPPORTED.  A call of more than 2^23 blocks (of at least
 *     64 rows of a head, or one appended token) is refused by its launch.
 *   - A row that sees no key gives zeros.  A key that a row does not see does
 *     not touch it, whatever it holds (infinities and NaN included); a NaN that
 *     a row does see gives NaN.
 *   - The calls on a cache take their scratch from the cache's `workspace`
 *     (sizes: the *_workspace queries), never from the per-stream workspace, so
 *     graphs captured over different caches share nothing.  Calls on one cache
 *     must be ordered (one stream, or synchronization between streams).
 */
#ifndef SWIFTLTX_ATTENTION_H
#define SWIFTLTX_ATTENTION_H

#include "swiftltx_q4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Attention over whole sequences: for row i and key j of sequence b, with
 * pos = i + k_len - q_len (the last row stands at the last key),
 *   x = scale q_i.k_j;  softcap > 0: x = softcap tanh(x / softcap);
 *   bias: x += bias[h * bias_head_stride + clamp(j - pos + bias_zero, 0, bias_len - 1)]
 *   out_i = sum_j softmax_j(x) v_j over the keys that row i sees:
 *     j < k_len, and
 *     not causal, or j <= pos, or j < prefix[b], and
 *     no documents, or q_docs[b, i] == k_docs[b, j] >= 0.
 * Rows from q_len on are not written.  A bias of -inf masks its distance. */
typedef struct sltx_attention_args {
    const void* q;              /* [batch, q_rows, q_heads, head_dim] */
    const void* k;              /* [batch, k_rows, kv_heads, head_dim] */
    const void* v;              /* like k */
    void* out;                  /* like q; must not overlap q, k or v */
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];   /* batch, row, head */
    int32_t dtype, batch, q_rows, k_rows, q_heads, kv_heads, head_dim;
    int32_t causal;
    float scale;                /* > 0 */
    float softcap;              /* 0: none */
    const float* bias;          /* fp32, or NULL */
    int64_t bias_head_stride;   /* 0: the same for all heads */
    int32_t bias_len, bias_zero;
    const int32_t* prefix;      /* [batch], or NULL; needs causal */
    const int32_t* q_docs;      /* [batch, q_rows], or NULL */
    const int32_t* k_docs;      /* [batch, k_rows], with q_docs */
    const int32_t* q_lens;      /* [batch], or NULL: q_rows; cut to [0, q_rows] */
    const int32_t* k_lens;      /* [batch], or NULL: k_rows; cut to [0, k_rows] */
} sltx_attention_args;
int sltx_attention(const sltx_attention_args* args, void* stream);

/* A key/value cache of all layers of a model for `batch` sequences.  length[b]
 * slots of each layer and head hold sequence b's tokens; new tokens go to the
 * slots behind them and count only once accepted (sltx_kv_accept).
 * next_position[b] is the position that the next token has, for its rotary
 * angles: larger than length[b] once entries were evicted.  The lengths live in
 * device memory, so that a captured step can be replayed as they grow.
 * Calls over one cache share its workspace too: they run one after the other, on
 * one stream or ordered by events.
 * weight and position (both or neither) serve eviction: of each slot the
 * attention weight that its key has had so far, and its token's position. */
typedef struct sltx_kv_cache {
    void* k;                    /* [layers, batch, kv_heads, capacity, head_dim] */
    void* v;                    /* the same */
    float* weight;              /* [layers, batch, kv_heads, capacity] or NULL */
    int32_t* position;          /* the same, or NULL */
    int32_t* length;            /* [batch] */
    int32_t* next_position;     /* [batch] */
    int32_t layers, batch, kv_heads, capacity, head_dim, dtype;
    void* workspace;            /* 16-byte aligned scratch, or NULL where 0 bytes are asked for */
    uint64_t workspace_bytes;
} sltx_kv_cache;

/* `tokens` new tokens of each sequence go into one layer: q and k are rotated
 * (row t of sequence b by the angles (next_position[b] + d) * inv_freq[0..pairs),
 * d = depth[b, t], or t without depth; computed in 64 bits), q goes to q_out
 * [batch, tokens, q_heads, head_dim] (contiguous), k and v to the slots
 * length[b] + t, with weight 0 and the token's position.  Pairs of values are
 * (i, i + pairs), or with `interleaved` (2i, 2i + 1); values past 2 * pairs pass
 * unchanged (pairs may be 0, with inv_freq NULL).  Tokens past the capacity are
 * dropped.  The sequence's length stays: every layer appends at the same place.
 * The cache's k and v must not overlap. */
int sltx_kv_append(const void* q, const int64_t q_stride[3], const void* k, const int64_t k_stride[3],
                   const void* v, const int64_t v_stride[3], const sltx_kv_cache* cache, int32_t layer,
                   int32_t tokens, int32_t q_heads, const float* inv_freq, int32_t pairs,
                   int32_t interleaved, const int32_t* depth, void* q_out, void* stream);

/* Attention of `tokens` of the appended tokens over one layer of the cache, q from
 * sltx_kv_append: those from the first-th on (0 but where a chunk is taken in more
 * than one call).  Token t sees the slots below length[b] + first, and of the
 * tokens of the call those up to t, or with `tree` (uint64 [batch, tokens],
 * tokens <= 64) those u whose bit u is set in tree[b, t] (its ancestors and
 * itself).  x as in sltx_attention, without bias.  out [batch, tokens, q_heads, head_dim] is
 * contiguous.  weight_rows > 0 (at most tokens <= 64; the cache has weight)
 * adds to weight the softmax weights of the first weight_rows tokens, summed
 * over the query heads of each key/value head. */
int sltx_attention_cached(const void* q, const int64_t q_stride[3], const sltx_kv_cache* cache,
                          int32_t layer, int32_t first, int32_t tokens, int32_t q_heads, float scale,
                          float softcap, const uint64_t* tree, int32_t weight_rows, void* out, void* stream);
/* Bytes of cache->workspace that the call takes, or a negative sltx_status. */
int64_t sltx_attention_cached_workspace(const sltx_kv_cache* cache, int32_t tokens, int32_t q_heads,
                                        int32_t weight_rows);

/* Of `drafted` appended tokens, those that were accepted become part of the
 * sequences: path (int32 [batch, path_len], path_len <= 64) names them in order,
 * of which the first count[b] (NULL: all) count.  In every layer and head, slot
 * length[b] + i takes the entry of slot length[b] + path[b, i]; then length and
 * next_position grow by the number accepted.  A path ends before an index outside
 * [0, drafted), before a token that the capacity had no room for, and at the
 * capacity, which it can reach by naming a token more than once.  path NULL:
 * the first count[b] (NULL: all) tokens as they stand. */
int sltx_kv_accept(const sltx_kv_cache* cache, int32_t drafted, const int32_t* path, int32_t path_len,
                   const int32_t* count, void* stream);

/* Cuts every sequence longer than `budget` to that many entries, in each layer
 * and head on its own: positions below `sinks` and the last `recent` positions
 * (next_position[b] - recent and later) stay, and of the rest those with the
 * highest weight (NaN counts as the lowest; of equal ones those in lower slots).
 * sinks + recent <= budget <= capacity.  Entries that stay in slots below the
 * budget keep them; the others that stay move, in slot order, into the slots
 * below it that became free.  Entries behind the budget are left as they were. */
int sltx_kv_evict(const sltx_kv_cache* cache, int32_t budget, int32_t sinks, int32_t recent,
                  void* stream);
int64_t sltx_kv_evict_workspace(const sltx_kv_cache* cache, int32_t budget);

#ifdef __cplusplus
}
#endif

#endif /* SWIFTLTX_ATTENTION_H */
