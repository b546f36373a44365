// attn_few.hip -- attention of few query rows over a key/value cache (a decoded
// token, a small tree of drafted tokens), the parts of split attentions joined,
// and attention weights added up per key.
//
// At most 32 rows, those of all query heads that share a key/value head, against
// thousands of keys: bound by reading the cache once.  A block takes one range
// of the keys of one head; its four waves take 32 keys each at a time, every
// wave with its own two stages of LDS, so nothing waits for another wave until
// the waves' sums are added at the end.
//
// One token of 24 heads over 8 of 128, fp16: 4000 keys (16 MB) 8.1 us and 3.9 to join
// the parts, most of both launch and trips to memory; 60000 keys 45 us in all, 5.5
// TB/s; eight sequences of 3000 26 us, 3.8 TB/s.  The kernel of many rows, made to take
// the same calls, has fewer waves at work on few keys: 12.8 us instead of 11.2 for 4000
// keys (head_dim 64: 10.6 instead of 9.6), but is up to a tenth faster at head_dim 128
// over many (eight sequences of 3000 23.9 us).  Which of the two it is goes by the
// lengths, which are on the device: calls of at most 32 rows take this one.
#include "attn_tile.hpp"

namespace sltx {

enum : int { kCap = 1, kSplit = 2 };
constexpr int kWaveKeys = kFewKeys / 4;   // keys of a wave's tile

template <int D, bool BF, int MODE>
__global__ __launch_bounds__(256, 1) void attn_few_kernel(AttnParams p) {
    constexpr bool CAP = MODE & kCap, SPLIT = MODE & kSplit;
    constexpr int TILE = kWaveKeys * D;      // values of a tile
    constexpr int QT = D / 16, DB = D / 32;
    constexpr int INSTR = TILE * 2 / 1024;   // copies of a tile
    constexpr int PITCH = D + 4;             // of the waves' sums in LDS
    constexpr int STAGES = 4 * 2 * 2 * TILE * 2, SUMS = 4 * kFewRows * PITCH * 4;
    __shared__ __attribute__((aligned(1024))) char lds[STAGES > SUMS ? STAGES : SUMS];
    __shared__ float mls[4][kFewRows][2];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    int hb = blockIdx.x % p.heads, b = blockIdx.x / p.heads, split = 0, each = 0;
    if constexpr (SPLIT) {
        const int parts = p.B * p.splits;
        hb = blockIdx.x / parts;
        const Shares shares(p, lane);
        if (p.B > 1 && blockIdx.x == 0 && wave == 0) shares.leave(p, lane);
        if (!shares.find(p, blockIdx.x % parts, b, split)) return;
        each = shares.each;
    }
    const int bh = b * p.heads + hb;
    const SeqLens len = seq_lens(p, b);
    const int rows = p.Sq * p.pack;

    const bool has_row = n < rows;
    const int qi = has_row ? n / p.pack : 0;
    const int head = hb * p.pack + (has_row ? n % p.pack : 0);
    const int units = (len.k + kFewKeys - 1) / kFewKeys;
    int first = 0, last = units;
    if (SPLIT) {
        first = min(units, split * each);
        last = min(units, first + each);
    }
    const int kstride = (int)p.ks.r * 2, vstride = (int)p.vs.r * 2, head_bytes = p.D * 2;
    const uint16_t* kbase = p.k + b * p.ks.b + hb * p.ks.h;
    const uint16_t* vbase = p.v + b * p.vs.b + hb * p.vs.h;
    TileCopy<D, false, INSTR> kc;
    TileCopy<D, true, INSTR> vc;
    kc.init(0, lane, kstride, head_bytes);
    vc.init(0, lane, vstride, head_bytes);
    // this wave's stages: K, V, K, V
    const uint32_t mine = lds_offset(lds) + wave * (4 * TILE * 2);
    // the wave's tile of unit u; a tile past the last key is not copied
    auto copy = [&](int u, int stage) {
        const int j0 = u * kFewKeys + wave * kWaveKeys;
        const int left = min(kWaveKeys, len.k - j0);
        if (left <= 0) return;
        const u32x4 kr = tile_rsrc(kbase + j0 * p.ks.r, left, kstride, head_bytes);
        const u32x4 vr = tile_rsrc(vbase + j0 * p.vs.r, left, vstride, head_bytes);
        const uint32_t at = mine + stage * (2 * TILE * 2);
#pragma unroll
        for (int i = 0; i < INSTR; ++i) copy_1k(kr, kc.off[i], at + i * 1024);
#pragma unroll
        for (int i = 0; i < INSTR; ++i) copy_1k(vr, vc.off[i], at + TILE * 2 + i * 1024);
    };
    if (first < last) copy(first, 0);
    if (first + 1 < last) copy(first + 1, 1);

    u32x4 qf[QT];
    {
        const uint16_t* q = p.q + b * p.qs.b + (int64_t)qi * p.qs.r + (int64_t)head * p.qs.h;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int c = 16 * t + 8 * h;
            qf[t] = has_row && c < p.D ? *reinterpret_cast<const u32x4*>(q + c) : u32x4{};
        }
    }
    // the row sees the keys below lim, but for the tree
    const int lim = p.tree ? len.k : min(len.k, len.old + qi + 1);
    const uint64_t tree = p.tree && has_row ? p.tree[b * (int64_t)p.Sq + qi] : 0;
    auto in_tree = [&](int j) { return j < len.old || (tree >> ((j - len.old) & 63) & 1); };

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x16{};
    RowState<BF> st;
    const float f = CAP ? kLog2e : p.scale * kLog2e;
    const float yscale = CAP ? p.scale / p.cap : 0.0f;
    const uint32_t kfrag = k_frag_base<D>(lane), vfrag = v_frag_base<D>(lane);
    float* score_row = nullptr;
    if (SPLIT && p.scores && has_row && n < p.score_rows)
        score_row = p.scores + ((int64_t)bh * p.score_rows + n) * p.score_pitch;
    int stage = 0;
    for (int u = first; u < last; ++u, stage ^= 1) {
        const int j0 = u * kFewKeys + wave * kWaveKeys;
        if (j0 >= len.k) break;   // only in the last unit
        // the next tile's copies may stay in flight
        // (and the 4 stores of the tile before's scores, issued ahead of them)
        if (!(u + 1 < last && j0 + kFewKeys < len.k)) copies_wait<0>();
        else if (SPLIT && p.scores && u > first) copies_wait<2 * INSTR + 4>();
        else copies_wait<2 * INSTR>();
        const uint32_t kt = mine + stage * (2 * TILE * 2), vt = kt + TILE * 2;
        const bool all = j0 + kWaveKeys <= len.old;
        uint32_t bad = 0;   // keys whose V rows are not finite
        if (!all) {
#pragma unroll
            for (int i = 0; i < TILE / 8 / 64; ++i) {
                constexpr int P = D / 8;
                const uint64_t m = __ballot(clear_piece<BF>(vt + (i * 64 + lane) * 16));
#pragma unroll
                for (int k = 0; k < 64 / P; ++k)
                    bad |= (m >> (k * P) & ((1u << P) - 1)) ? 1u << (i * (64 / P) + k) : 0;
            }
        }
        f32x16 s = {};
#pragma unroll
        for (int t = 0; t < QT; ++t) s = mfma32<BF>(k_frag<D>(kt, kfrag, 0, t), qf[t], s);
        if constexpr (CAP) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = capped(s[i], yscale, p.scale, p.cap);
        }
        if (!all) {
            const int d = lim - j0 - 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 8 * (i / 4) + i % 4 < d ? s[i] : -kInf;
            if (p.tree) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[i] = in_tree(j0 + 8 * (i / 4) + 4 * h + i % 4) ? s[i] : -kInf;
            }
        }
        if constexpr (SPLIT) {
            if (score_row) keep_scores(score_row, j0, h, f, s);
        }
        u32x4 pf[2];
        st.template take<false, SPLIT, DB>(s, f, pf, o);
        weigh_values<D, BF, 2>(o, pf, vt, vfrag);
        while (bad) {
            const int j = j0 + __builtin_ctz(bad);
            bad &= bad - 1;
            const bool mine = has_row && j < lim && (!p.tree || in_tree(j));
            add_values<D, BF>(o, vbase + j * p.vs.r, p.D, h, mine);
        }
        // the stage is free once every read of it has returned
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (u + 2 < last) copy(u + 2, stage);
    }

    // ---- the waves' sums ----
    const float l = half_sum(st.l);
    __syncthreads();   // no wave reads its stages any more
    float* sums = reinterpret_cast<float*>(lds);
    if (has_row) {
        float* po = sums + (wave * kFewRows + n) * PITCH;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(po + 32 * db + 8 * i + 4 * h) =
                    f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
        if (h == 0) mls[wave][n][0] = st.mf, mls[wave][n][1] = l;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * (D / 4); e += 256) {
        const int r = e / (D / 4), c = e % (D / 4) * 4;
        float m = -kInf;
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, mls[w][r][0]);
        f32x4 x = {};
        float lsum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float a = __builtin_amdgcn_exp2f(mls[w][r][0] - m);
            lsum += a * mls[w][r][1];
            const f32x4 y = *reinterpret_cast<const f32x4*>(sums + (w * kFewRows + r) * PITCH + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] += a * y[i];
        }
        if constexpr (SPLIT) {
            const int64_t at = (int64_t)blockIdx.x * rows + r;
            *reinterpret_cast<f32x4*>(p.part_o + at * D + c) = x;
            if (c == 0) *reinterpret_cast<f32x2*>(p.part_ml + at * 2) = f32x2{m, lsum};
        } else if (c < p.D) {
            const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
            uint16_t* out = p.out + b * p.os.b + (int64_t)(r / p.pack) * p.os.r +
                            (int64_t)(hb * p.pack + r % p.pack) * p.os.h;
            *reinterpret_cast<u32x2*>(out + c) =
                u32x2{pack2<BF>(x[0] * inv, x[1] * inv), pack2<BF>(x[2] * inv, x[3] * inv)};
        }
    }
}

// The end of a split attention.  A block for each row: out = sum over the splits of
// exp2(m_s - m) part_s, divided by the same sum of their l; four waves take every
// fourth split.  Or a wave for each row, ROWS = 4 to a block, where those are
// enough.  Blocks ahead of them take 1024 keys of a head each, and add the
// weights of the rows whose scores were kept, exp2(f x - m) / l summed over the
// rows.  What a block reads does not depend on what it computes, so all of it is on
// its way at once: the launch is a trip or two to memory long: 24 rows in 32 parts of head_dim 128 3.9 us, 2944
// rows in 15 parts and the weights of 47000 keys from 4 rows each for 8 heads 10.3 us
// for 33 MB.
constexpr int kFinishKeys = 1024;
constexpr int kAhead = 8;   // parts that a wave reads at a time

// (m, l) of a row over all splits, `every` lanes holding every `every`-th split: the
// lane's own first, in x, then all of them.
template <int EVERY, int MOST>
__device__ __forceinline__ f32x2 whole_row(const f32x2 (&x)[MOST / EVERY]) {
    float m = -kInf, l = 0.0f;
#pragma unroll
    for (int i = 0; i < MOST / EVERY; ++i) m = fmaxf(m, x[i][0]);
#pragma unroll
    for (int o = 1; o < EVERY; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
#pragma unroll
    for (int i = 0; i < MOST / EVERY; ++i) l += x[i][1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x[i][0] - m) * x[i][1];
#pragma unroll
    for (int o = 1; o < EVERY; o <<= 1) l += __shfl_xor(l, o, 64);
    return f32x2{m, l};
}

template <int D, bool BF, int ROWS>
__global__ __launch_bounds__(256) void attn_finish_kernel(AttnParams p, float* weight) {
    constexpr int PER = D / 64;
    __shared__ __attribute__((aligned(8))) float sums[ROWS == 1 ? 4 : 1][D];
    __shared__ f32x2 ml[kScoreRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rows = p.Sq * p.pack;
    const int chunks = p.scores ? (p.Sk + kFinishKeys - 1) / kFinishKeys : 0;
    if ((int)blockIdx.x < p.B * p.heads * chunks) {
        const int bh = blockIdx.x / chunks, j = blockIdx.x % chunks * kFinishKeys + threadIdx.x * 4;
        const int b = bh / p.heads;
        // the (m, l) of the rows: 16 lanes for each
        const int row = threadIdx.x >> 4, l16 = threadIdx.x & 15;
        const int start = p.B > 1 ? p.shares[2 * b] : 0, splits = p.B > 1 ? p.shares[2 * b + 1] : p.splits;
        const f32x2* part = reinterpret_cast<const f32x2*>(p.part_ml) +
                            ((int64_t)(bh % p.heads) * (p.B * p.splits) + start) * rows + min(row, rows - 1);
        f32x2 parts[kMostSplits / 16];
#pragma unroll
        for (int i = 0; i < kMostSplits / 16; ++i) {
            parts[i] = f32x2{-kInf, 0.0f};
            if (i * 16 < splits && i * 16 + l16 < splits) parts[i] = part[(int64_t)(i * 16 + l16) * rows];
        }
        const SeqLens len = seq_lens(p, b);
        if (blockIdx.x % chunks * kFinishKeys >= len.k) return;
        const float* scores = p.scores + (int64_t)bh * p.score_rows * p.score_pitch + j;
        float* w = weight + (int64_t)bh * p.Sk + j;
        f32x4 x[4], sum = {};
        auto read = [&](int r0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r0 + i < p.score_rows && j < len.k)
                    x[i] = *reinterpret_cast<const f32x4*>(scores + (int64_t)(r0 + i) * p.score_pitch);
        };
        read(0);
        float old[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) old[e] = j + e < len.k ? w[e] : 0.0f;
        const f32x2 r = whole_row<16, kMostSplits>(parts);
        if (l16 == 0) ml[row] = f32x2{r[0], r[1] == 0.0f ? 0.0f : 1.0f / r[1]};
        __syncthreads();
        if (j >= len.k) return;
        for (int r0 = 0; r0 < p.score_rows; r0 += 4) {
            if (r0 > 0) read(r0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (r0 + i >= p.score_rows) break;
                const f32x2 c = ml[r0 + i];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // keys before the new tokens are seen by every row
                    const bool sees = j + e < len.old || cached_sees(p, len, b, (r0 + i) / p.pack, j + e);
                    sum[e] += sees ? __builtin_amdgcn_exp2f(x[i][e] - c[0]) * c[1] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < len.k) w[e] = old[e] + sum[e];
        return;
    }
    // the wave's row, and its parts: every fourth one, or all
    const int block = blockIdx.x - p.B * p.heads * chunks, index = ROWS == 1 ? block : block * ROWS + wave;
    constexpr int STEP = 4 / ROWS;
    const int first = ROWS == 1 ? wave : 0;
    if (index >= p.B * p.heads * rows) return;
    const int row = index % rows, bh = index / rows;
    const int hb = bh % p.heads, b = bh / p.heads;
    const int start = p.B > 1 ? p.shares[2 * b] : 0, splits = p.B > 1 ? p.shares[2 * b + 1] : p.splits;
    const int64_t at = ((int64_t)hb * (p.B * p.splits) + start) * rows + row;   // of the first part
    const f32x2* part_ml = reinterpret_cast<const f32x2*>(p.part_ml) + at;
    typedef float vec __attribute__((ext_vector_type(PER)));   // columns PER lane ..
    const vec* part_o = reinterpret_cast<const vec*>(p.part_o + at * D) + lane;
    f32x2 parts[kMostSplits / 64];
#pragma unroll
    for (int i = 0; i < kMostSplits / 64; ++i) {
        parts[i] = f32x2{-kInf, 0.0f};
        if (i * 64 < splits && i * 64 + lane < splits) parts[i] = part_ml[(int64_t)(i * 64 + lane) * rows];
    }
    // kAhead of the wave's parts, and their m
    vec y[kAhead];
    float ms[kAhead];
    auto read = [&](int s0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int s = s0 + STEP * i;
            if (s >= splits) break;
            ms[i] = part_ml[(int64_t)s * rows][0];
            y[i] = part_o[(int64_t)s * rows * 64];
        }
    };
    read(first);
    const f32x2 whole = whole_row<64, kMostSplits>(parts);
    const float m = whole[0], l = whole[1];
    vec x = {};
    for (int s0 = first; s0 < splits; s0 += STEP * kAhead) {
        if (s0 > first) read(s0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (s0 + STEP * i >= splits) break;
            x += __builtin_amdgcn_exp2f(ms[i] - m) * y[i];
        }
    }
    if constexpr (ROWS == 1) {
        reinterpret_cast<vec*>(sums[wave])[lane] = x;
        __syncthreads();
        if (wave > 0) return;
        x = vec{};
#pragma unroll
        for (int w = 0; w < 4; ++w) x += reinterpret_cast<const vec*>(sums[w])[lane];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (p.row_ml && lane == 0)
        *reinterpret_cast<f32x2*>(p.row_ml + (int64_t)index * 2) = f32x2{l == 0.0f ? 0.0f : m, inv};
    if (lane * PER < p.D) {
        uint16_t* out = p.out + b * p.os.b + (int64_t)(row / p.pack) * p.os.r +
                        (int64_t)(hb * p.pack + row % p.pack) * p.os.h + lane * PER;
        if constexpr (PER == 2) *reinterpret_cast<uint32_t*>(out) = pack2<BF>(x[0] * inv, x[1] * inv);
        else *out = (uint16_t)pack2<BF>(x[0] * inv, 0.0f);
    }
}

// The same for more rows, whose scores are formed again (to keep them would write
// and read 8 bytes for each; reading K again is 2 head_dim for all of them):
// weight[key] += sum over rows r < wrows of exp2(f x_r - mf_r) / l_r.  S = Q K^T
// this way round, so that a lane holds 16 rows of one key: the sum over rows is
// its own.  A wave takes kWeightTiles times 32 keys, for which it reads 32 rows of
// Q and their statistics once; all fragments come straight from memory.  92 rows and
// 47000 keys of 8 heads of 128: 63 us (86 with one tile), 141 TFLOP/s of products and
// 550 weights a ns; 20 rows 33.  To keep the scores of 16 rows costs 12: hence
// kScoreRows.
constexpr int kWeightTiles = 2;
template <int D, bool BF, bool CAP>
__global__ __launch_bounds__(256) void attn_weights_kernel(AttnParams p, float* weight, int wrows) {
    constexpr int QT = D / 16, KEYS = 32 * kWeightTiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int bh = blockIdx.y, hb = bh % p.heads, b = bh / p.heads;
    const SeqLens len = seq_lens(p, b);
    const int rows = p.Sq * p.pack;
    const float f = CAP ? kLog2e : p.scale * kLog2e;
    const float yscale = CAP ? p.scale / p.cap : 0.0f;
    const f32x2* row_ml = reinterpret_cast<const f32x2*>(p.row_ml) + (int64_t)bh * rows;
    for (int j0 = (blockIdx.x * 4 + wave) * KEYS; j0 < len.k; j0 += gridDim.x * 4 * KEYS) {
        const bool all = j0 + KEYS <= len.old;   // every row sees every key
        u32x4 kf[kWeightTiles][QT];
#pragma unroll
        for (int kt = 0; kt < kWeightTiles; ++kt) {
            const uint16_t* k = p.k + b * p.ks.b + hb * p.ks.h + min(j0 + 32 * kt + n, len.k - 1) * p.ks.r;
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const int c = 16 * t + 8 * h;
                kf[kt][t] = c < p.D ? *reinterpret_cast<const u32x4*>(k + c) : u32x4{};
            }
        }
        float sum[kWeightTiles] = {};
        for (int r0 = 0; r0 < wrows; r0 += 32) {
            const int r = min(r0 + n, wrows - 1);
            const uint16_t* q = p.q + b * p.qs.b + (int64_t)(r / p.pack) * p.qs.r +
                                (int64_t)(hb * p.pack + r % p.pack) * p.qs.h;
            u32x4 qf[QT];
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const int c = 16 * t + 8 * h;
                qf[t] = c < p.D ? *reinterpret_cast<const u32x4*>(q + c) : u32x4{};
            }
            f32x2 ml[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = r0 + 8 * (i / 4) + 4 * h + i % 4;
                ml[i] = row_ml[min(row, wrows - 1)];
                if (row >= wrows) ml[i][1] = 0.0f;
            }
#pragma unroll
            for (int kt = 0; kt < kWeightTiles; ++kt) {
                f32x16 s = {};
#pragma unroll
                for (int t = 0; t < QT; ++t) s = mfma32<BF>(qf[t], kf[kt][t], s);
                const int j = j0 + 32 * kt + n;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x = CAP ? capped(s[i], yscale, p.scale, p.cap) : s[i];
                    const int row = min(r0 + 8 * (i / 4) + 4 * h + i % 4, wrows - 1);
                    const bool sees = (all || (j < len.k && cached_sees(p, len, b, row / p.pack, j))) && ml[i][1] != 0.0f;
                    sum[kt] += sees ? __builtin_amdgcn_exp2f(x * f - ml[i][0]) * ml[i][1] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int kt = 0; kt < kWeightTiles; ++kt) {
            const int j = j0 + 32 * kt + n;
            const float w = half_sum(sum[kt]);
            if (j < len.k && h == 0) weight[(int64_t)bh * p.Sk + j] += w;
        }
    }
}

template <int D, bool BF>
static hipError_t launch_few(const AttnParams& p, hipStream_t st) {
    const dim3 g(p.B * p.heads * p.splits), t(256);
    const bool split = p.part_o != nullptr;
    if (p.cap > 0.0f) {
        if (split) hipLaunchKernelGGL((attn_few_kernel<D, BF, kCap | kSplit>), g, t, 0, st, p);
        else hipLaunchKernelGGL((attn_few_kernel<D, BF, kCap>), g, t, 0, st, p);
    } else {
        if (split) hipLaunchKernelGGL((attn_few_kernel<D, BF, kSplit>), g, t, 0, st, p);
        else hipLaunchKernelGGL((attn_few_kernel<D, BF, 0>), g, t, 0, st, p);
    }
    return hipGetLastError();
}

hipError_t launch_attn_few(AttnParams p, hipStream_t st) {
    if (p.D > 64) return p.bf16 ? launch_few<128, true>(p, st) : launch_few<128, false>(p, st);
    return p.bf16 ? launch_few<64, true>(p, st) : launch_few<64, false>(p, st);
}

template <int D, bool BF>
static hipError_t launch_finish(const AttnParams& p, float* weight, hipStream_t st) {
    const int chunks = p.scores ? (p.Sk + kFinishKeys - 1) / kFinishKeys : 0;
    const int64_t heads = (int64_t)p.B * p.heads, rows = heads * p.Sq * p.pack;
    // A wave for each row from four blocks of them for each CU on.  Measured (one wave /
    // four, us of the whole call): 40 rows for 4 sequences of 12000 keys and 24 heads of
    // 128 50.0 / 52.4; 16 rows for 8 sequences of 3000 28.5 / 30.7; fewer rows leave CUs idle.
    const bool many = rows >= 4 * kCUs;
    const int64_t blocks = heads * chunks + (many ? (rows + 3) / 4 : rows);
    if (blocks > 0x7fffff00 / 256) return hipErrorInvalidValue;
    const dim3 g((unsigned)blocks), t(256);
    if (many) hipLaunchKernelGGL((attn_finish_kernel<D, BF, 4>), g, t, 0, st, p, weight);
    else hipLaunchKernelGGL((attn_finish_kernel<D, BF, 1>), g, t, 0, st, p, weight);
    return hipGetLastError();
}

hipError_t launch_attn_finish(const AttnParams& p, float* weight, hipStream_t st) {
    if (p.D > 64) return p.bf16 ? launch_finish<128, true>(p, weight, st) : launch_finish<128, false>(p, weight, st);
    return p.bf16 ? launch_finish<64, true>(p, weight, st) : launch_finish<64, false>(p, weight, st);
}

template <int D, bool BF>
static hipError_t launch_weights(const AttnParams& p, float* weight, int wrows, hipStream_t st) {
    const dim3 g(std::min(64, (p.Sk + 128 * kWeightTiles - 1) / (128 * kWeightTiles)), p.B * p.heads), t(256);
    if (p.cap > 0.0f) hipLaunchKernelGGL((attn_weights_kernel<D, BF, true>), g, t, 0, st, p, weight, wrows);
    else hipLaunchKernelGGL((attn_weights_kernel<D, BF, false>), g, t, 0, st, p, weight, wrows);
    return hipGetLastError();
}

hipError_t launch_attn_weights(const AttnParams& p, float* weight, int rows, hipStream_t st) {
    const int w = rows * p.pack;
    if (p.D > 64) return p.bf16 ? launch_weights<128, true>(p, weight, w, st) : launch_weights<128, false>(p, weight, w, st);
    return p.bf16 ? launch_weights<64, true>(p, weight, w, st) : launch_weights<64, false>(p, weight, w, st);
}

}  // namespace sltx
