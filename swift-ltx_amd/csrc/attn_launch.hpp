// attn_launch.hpp -- parameter blocks and host launchers of the attention and
// key/value cache kernels, shared with their C ABI (attn_capi.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace sltx {

// Strides of a [batch, row, head, head_dim] tensor in elements; head_dim is
// contiguous.
struct AttnStrides {
    int64_t b, r, h;
};

// One attention over B sequences; see attn_seq_kernel.hpp and attn_few.hip.  A block's
// rows are (query row i, head g of `pack`) pairs, i * pack + g: pack is 1, or
// the query heads that share a key/value head.
struct AttnParams {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    AttnStrides qs, ks, vs, os;
    int B, Sq, Sk, Hq, Hk, D;
    int bf16;
    float scale, cap;           // cap 0: none
    const float* bias;          // [Hq or 1][bias_n]: bias[clamp(distance + bias_zero)]
    int64_t bias_h;             // elements between heads (0: one row for all)
    int bias_n, bias_zero;
    int causal;
    const int32_t* prefix;      // [B] keys that every row sees, or null
    const int32_t *q_docs, *k_docs;   // [B, Sq], [B, Sk] or null
    const int32_t *q_lens, *k_lens;   // [B] or null
    // Over a cache: k_lens + first are the slots before the new tokens, Sk the
    // capacity, the keys k_lens[b] + first + Sq; row i stands at key k_lens[b] +
    // first + i.
    int cached, first;
    const uint64_t* tree;       // [B, Sq] new tokens that row i sees, or null
    // filled by the launchers
    int pack, heads, tiles, splits;
    int unit_bits;              // splits are whole units of 1 << unit_bits keys
    int by_xcd, long_first;     // order of the blocks
    int halves;                 // blocks of 64 rows
    float* part_o;              // [heads][B * splits][Sq * pack][DT] sums of a part (attn_tile.hpp)
    float* part_ml;             // [heads][B * splits][Sq * pack][2] (f m, l)
    int32_t* shares;            // [B][2]: a sequence's first part and how many it has (B > 1)
    float* row_ml;              // [B][heads][Sq * pack][2] (f m, 1 / l), or null
    // f x of the first score_rows rows, -inf where masked, for the weights' sums;
    // keys of tiles that a row does not see at all may be missing
    float* scores;              // [B][heads][score_rows][score_pitch], or null
    int score_rows, score_pitch;
};

// Keys and rows of sequence b.  Lengths come from device memory: out of range
// ones are cut to what the tensors hold.
struct SeqLens {
    int q, k;      // rows, keys
    int shift;     // row i stands at key i + shift
    int old;       // cached: keys that every row sees
};
__device__ __forceinline__ SeqLens seq_lens(const AttnParams& p, int b) {
    SeqLens s;
    s.q = p.q_lens ? min(max(p.q_lens[b], 0), p.Sq) : p.Sq;
    const int k = p.k_lens ? min(max(p.k_lens[b], 0), p.Sk) : p.Sk;
    s.old = p.cached ? min(k + p.first, p.Sk) : k;
    s.k = p.cached ? min(s.old + s.q, p.Sk) : k;
    s.shift = p.cached ? s.old : k - s.q;
    return s;
}

// Sums over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);   // from 1, 2, 4, 8 lanes below in a row of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // from the last lane of the row below
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // from lane 31
    return x;
}

constexpr int kSeqTileRows = 128;   // query rows of a block of attn_seq_kernel.hpp
constexpr int kTileKeys = 64;       // keys of its tiles
constexpr int kFewRows = 32;        // most rows of a block of attn_few.hip
constexpr int kFewKeys = 128;       // keys that its four waves take at a time

hipError_t launch_attn_seq(AttnParams p, hipStream_t st);
hipError_t launch_attn_seq_d128(const AttnParams& p, dim3 g, hipStream_t st);
hipError_t launch_attn_few(AttnParams p, hipStream_t st);
// out = sum of the splits' parts; row_ml where asked for; with scores, also
// weight[b, head, key] += the weights of the first score_rows rows.
hipError_t launch_attn_finish(const AttnParams& p, float* weight, hipStream_t st);
// weight[b, head, key] += the weights of the first `rows` query rows, recomputed
// from row_ml.
hipError_t launch_attn_weights(const AttnParams& p, float* weight, int rows, hipStream_t st);
constexpr int kMostSplits = 256;   // parts of one sequence
constexpr int kScoreRows = 16;   // most rows whose scores are kept

// ---- cache ----
struct CacheParams {
    uint16_t *k, *v;            // [layers, B, heads, capacity, D]
    float* weight;              // [layers, B, heads, capacity] or null
    int32_t* position;          // the same, or null
    int32_t *length, *next;     // [B]
    int layers, B, heads, capacity, D;
};
struct AppendParams {
    CacheParams c;
    int layer;
    const uint16_t *q, *k, *v;
    uint16_t* q_out;            // [B, T, Hq, D]
    AttnStrides qs, ks, vs;
    int T, Hq, bf16;
    const float* inv_freq;      // [pairs]
    int pairs, interleaved;
    const int32_t* depth;       // [B, T] or null
};
hipError_t launch_kv_append(const AppendParams& p, hipStream_t st);
hipError_t launch_kv_accept(const CacheParams& c, int drafted, const int32_t* path, int path_len,
                            const int32_t* count, hipStream_t st);
size_t kv_evict_workspace_bytes(const CacheParams& c, int budget);
hipError_t launch_kv_evict(const CacheParams& c, int budget, int sinks, int recent, void* ws,
                           hipStream_t st);

}  // namespace sltx
