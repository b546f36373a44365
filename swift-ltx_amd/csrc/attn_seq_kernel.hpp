// attn_seq_kernel.hpp -- attention of many query rows: o = softmax(x) v with
// x = cap tanh(scale q.k / cap) + bias[j - pos(i)], over the keys that a row
// sees (causal, prefix, documents, lengths, a tree of drafted tokens).
//
// A block of 4 waves takes 128 query rows (32 a wave, Q in registers), or where
// those blocks would be few 64 rows, its waves two and two on the halves of each
// tile's keys (WK = 2), over all keys or over one of `splits` ranges of them.
// Tiles of 64 keys pass through LDS, copied while the tiles before are computed.
// One pass over the keys with a running maximum and sum; nothing but the output
// is written.
//
// 4 head_dim operations a score on the matrix units and about 4 vector instructions,
// one of them an exponential at a quarter of the others' rate.  At head_dim 64 the
// scores cost more than the products: 6144 rows and keys of 32 heads, bf16, 340 to
// 382 us, 810 to 908 TFLOP/s, where a large product reaches 1190 to 1245.  Counters
// (about 1.9 GHz): the matrix units are busy in 40% of a SIMD's cycles, vector
// instructions are at work in 53%.  Head_dim 128 halves the scores: 8192
// causal rows of 32 heads, two sequences, 1057 to 1096 us, 1003 to 1040 TFLOP/s;
// 4096 rows of one 152 us, 900.  A tile takes 1.0 us for 64 rows and 64 keys of
// head_dim 128, mostly the chain of its steps, so that few rows (750 behind 1300
// cached keys, 24 heads: 45 us, 340 TFLOP/s) are bound by the tiles in a row.
#pragma once

#include "attn_tile.hpp"

namespace sltx {

// Variants.  Documents, and the parts that a cached attention is split into (the
// only ones with a tree), have kernels of their own: their state costs registers.
// So have caps above kShortCap (kClose, with kCap).
enum : int { kCap = 1, kBias = 2, kSplit = 4, kDocs = 8, kClose = 16 };
constexpr float kShortCap = 64.0f;   // models' caps are 30 and 50

// Documents of a run of 64 tiles (one lane each): the smallest and largest id
// of a tile's keys, ids below 0 (padding) left out, and whether all are equal.
struct DocTiles {
    int lo[64], hi[64], same[64];
};

template <int D, bool BF, int MODE, int WK>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_seq_kernel(AttnParams p) {
    constexpr bool CAP = MODE & kCap, BIAS = MODE & kBias, SPLIT = MODE & kSplit, DOCS = MODE & kDocs;
    constexpr bool CLOSE = CAP && (SPLIT || MODE & kClose);
    constexpr int TILE = kTileKeys * D;          // values of a tile
    constexpr int QT = D / 16, DB = D / 32, KB = 2 / WK;   // KB blocks of 32 keys a wave and tile
    constexpr int INSTR = TILE * 2 / 1024 / 4;   // copies of a wave into a tile
    // Two stages.  A third changed nothing (6144 rows of 32 heads of 64: 350 us with
    // three, 347 with two; 4095 rows of documents 62 and 61): other blocks of the CU
    // compute while one waits.
    constexpr int STAGES = 2;
    __shared__ __attribute__((aligned(1024))) uint16_t ks[STAGES][TILE], vs[STAGES][TILE];
    __shared__ DocTiles docs;
    __shared__ __attribute__((aligned(8))) float half_ml[WK == 2 ? 2 : 1][32][2];   // (m, l) of the second half's rows
    __shared__ __attribute__((aligned(16))) int tile_docs[STAGES][kTileKeys];   // [stage]: documents of a tile's keys
    __shared__ uint32_t bad_keys[STAGES][2];   // [stage]: its keys whose V rows are not finite

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int wave_row = WK == 1 ? wave : wave & 1, wave_key = WK == 1 ? 0 : wave >> 1;   // its rows, its half of a tile's keys

    // Blocks go round the 8 XCDs in turn: each XCD gets a run of the heads (with
    // their parts), so that the blocks that share keys share an L2.  Under a causal
    // mask or documents the last tiles of all of the XCD's heads come first: they
    // see the most keys, and a long one that starts late is waited for at the end.
    // Else a head's tiles are next to each other.
    int hs, tile;   // (sequence, head) or (head, part), and the tile of rows
    {
        const int all = p.B * p.heads * p.splits, each = all / 8;
        const int i = blockIdx.x >> 3, x = blockIdx.x & 7;
        if (p.by_xcd) {
            hs = x * each + (p.long_first ? i % each : i / p.tiles);
            tile = p.long_first ? i / each : i % p.tiles;
        } else {
            hs = blockIdx.x % all;
            tile = blockIdx.x / all;
        }
        tile = p.tiles - 1 - tile;
    }
    int hb = hs % p.heads, b = hs / p.heads, split = 0, each = 0;
    if constexpr (SPLIT) {   // hs: (head, part)
        const int parts = p.B * p.splits;
        hb = hs / parts;
        const Shares shares(p, lane);
        if (p.B > 1 && blockIdx.x == 0 && wave == 0) shares.leave(p, lane);
        if (!shares.find(p, hs % parts, b, split)) return;
        each = shares.each;
    }
    const SeqLens len = seq_lens(p, b);
    const int rows = len.q * p.pack;
    const int row0 = tile * (kSeqTileRows / WK);
    if (row0 >= rows) return;

    // this lane's query row
    const int row = row0 + wave_row * 32 + n;
    const bool has_row = row < rows;
    const int qi = has_row ? row / p.pack : 0;
    const int head = p.pack == 1 ? hb : hb * p.pack + (has_row ? row % p.pack : 0);
    const int kvh = p.pack == 1 ? hb / (p.Hq / p.Hk) : hb;
    u32x4 qf[QT];
    {
        const uint16_t* q = p.q + b * p.qs.b + (int64_t)qi * p.qs.r + (int64_t)head * p.qs.h;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int c = 16 * t + 8 * h;
            qf[t] = has_row && c < p.D ? *reinterpret_cast<const u32x4*>(q + c) : u32x4{};
        }
    }
    // rows of this wave and of the block: first and last position
    const int wrow0 = row0 + wave_row * 32;
    const bool wave_rows = wrow0 < rows;
    const int wpos0 = wrow0 / p.pack + len.shift;
    const int wpos1 = (min(wrow0 + 31, rows - 1)) / p.pack + len.shift;
    const int bpos0 = row0 / p.pack + len.shift;
    const int bpos1 = (min(row0 + (kSeqTileRows / WK), rows) - 1) / p.pack + len.shift;
    const int pos = qi + len.shift;
    const int prefix = p.prefix ? p.prefix[b] : 0;
    const int kend = p.causal ? min(len.k, max(bpos1 + 1, prefix)) : len.k;
    int first = 0, last = (kend + kTileKeys - 1) / kTileKeys;   // tiles
    if (SPLIT) {
        first = min(last, split * each);
        last = min(last, first + each);
    }

    // documents of the rows: the smallest and largest of a wave's and of the
    // block's, and the one that all of them are of (-2: none, as where a row is of
    // no document)
    int qdoc = -1, wdoc0 = 0x7fffffff, wdoc1 = -1, wdoc = -2, bdoc0 = 0, bdoc1 = 0, bdoc = -2;
    const int32_t* kdocs = nullptr;
    if constexpr (DOCS) {
        kdocs = p.k_docs + b * (int64_t)p.Sk;
        qdoc = has_row ? p.q_docs[b * (int64_t)p.Sq + qi] : -1;
        wdoc0 = qdoc >= 0 ? qdoc : 0x7fffffff;
        wdoc1 = qdoc;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            wdoc0 = min(wdoc0, __shfl_xor(wdoc0, o, 64));
            wdoc1 = max(wdoc1, __shfl_xor(wdoc1, o, 64));
        }
        wdoc0 = __builtin_amdgcn_readfirstlane(wdoc0);
        wdoc1 = __builtin_amdgcn_readfirstlane(wdoc1);
        if (wdoc0 == wdoc1 && !__any(has_row && qdoc < 0)) wdoc = wdoc0;
        if (lane == 0) docs.lo[wave] = wdoc0, docs.hi[wave] = wdoc1, docs.same[wave] = wave_rows ? wdoc : -3;
        __syncthreads();
        bdoc0 = min(min(docs.lo[0], docs.lo[1]), min(docs.lo[2], docs.lo[3]));
        bdoc1 = max(max(docs.hi[0], docs.hi[1]), max(docs.hi[2], docs.hi[3]));
        bdoc = docs.same[0];   // the first wave has rows
#pragma unroll
        for (int i = 1; i < 4; ++i)
            if (docs.same[i] != -3 && docs.same[i] != bdoc) bdoc = -2;
        __syncthreads();
    }
    const uint64_t tree = SPLIT && p.tree && has_row ? p.tree[b * (int64_t)p.Sq + qi] : 0;

    // ---- copies ----
    const int head_bytes = p.D * 2;
    const uint16_t* kbase = uniform(p.k + b * p.ks.b + kvh * p.ks.h);
    const uint16_t* vbase = uniform(p.v + b * p.vs.b + kvh * p.vs.h);
    TileCopy<D, false, INSTR> kc;
    TileCopy<D, true, INSTR> vc;
    kc.init(wave * INSTR, lane, (int)p.ks.r * 2, head_bytes);
    vc.init(wave * INSTR, lane, (int)p.vs.r * 2, head_bytes);
    const uint32_t klds = lds_offset(&ks[0][0]), vlds = lds_offset(&vs[0][0]);
    const uint32_t dlds = DOCS ? lds_offset(&tile_docs[0][0]) : 0;
    auto copy = [&](int t, int stage) __attribute__((always_inline)) {
        const int64_t j0 = (int64_t)t * kTileKeys;
        const int left = min(kTileKeys, len.k - (int)j0);
        const u32x4 kr = tile_rsrc(kbase + j0 * p.ks.r, left, (int)p.ks.r * 2, head_bytes);
        const u32x4 vr = tile_rsrc(vbase + j0 * p.vs.r, left, (int)p.vs.r * 2, head_bytes);
        const uint32_t at = stage * (TILE * 2) + wave * (INSTR * 1024);
#pragma unroll
        for (int i = 0; i < INSTR; ++i) copy_1k(kr, kc.off[i], klds + at + i * 1024);
#pragma unroll
        for (int i = 0; i < INSTR; ++i) copy_1k(vr, vc.off[i], vlds + at + i * 1024);
        if (DOCS && wave == 0)   // keys past the last are masked by it, whatever this gives
            copy_256(tile_rsrc(reinterpret_cast<const uint16_t*>(kdocs + j0), 1, 0, left * 4), lane * 4, dlds + stage * (kTileKeys * 4));
    };

    // ---- which tiles ----
    // The tiles of [first, last) that some row of the block may see, in order.
    // With documents, runs of 64 tiles are looked through at a time: `live` has
    // a bit for each.
    uint64_t live = 0, one_b = 0, one_w = 0, seen_w = 0;
    int run = first - 64, next_t = first;
    auto look = [&](int at) __attribute__((always_inline)) {   // all threads: fills docs for tiles at .. at + 63
        const int t = threadIdx.x >> 2, j = (at + t) * kTileKeys + (threadIdx.x & 3) * 16;
        int lo = 0x7fffffff, hi = -1, low = 0x7fffffff;
        auto take = [&](int d) __attribute__((always_inline)) {
            lo = min(lo, d < 0 ? 0x7fffffff : d);
            low = min(low, d);
            hi = max(hi, d);
        };
        // four ids a load (4-byte aligned); the last ones are read again rather than past the end
        typedef int ids __attribute__((ext_vector_type(4), aligned(4)));
        if (kend >= 4) {
            ids d[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) d[g] = *reinterpret_cast<const ids*>(kdocs + min(j + 4 * g, kend - 4));
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) take(min(j + 4 * g, kend - 4) + e >= j + 4 * g ? d[g][e] : -1);
        } else {
            for (int e = 0; e < 16; ++e) take(j + e < kend ? kdocs[j + e] : -1);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            lo = min(lo, __shfl_xor(lo, o, 64));
            low = min(low, __shfl_xor(low, o, 64));
            hi = max(hi, __shfl_xor(hi, o, 64));
        }
        __syncthreads();
        if ((threadIdx.x & 3) == 0) docs.lo[t] = lo, docs.hi[t] = hi, docs.same[t] = low == hi;
        __syncthreads();
        const int lo1 = docs.lo[lane], hi1 = docs.hi[lane], one = docs.same[lane] ? lo1 : -4;
        live = __ballot(at + lane < last && hi1 >= bdoc0 && lo1 <= bdoc1);
        one_b = __ballot(one == bdoc);
        one_w = __ballot(one == wdoc);
        seen_w = __ballot(hi1 >= wdoc0 && lo1 <= wdoc1);
    };
    struct Tile {
        int t;
        bool one_b, one_w, seen_w;   // of the one document of the block's or the wave's rows; seen by the wave
    };
    auto advance = [&]() __attribute__((always_inline)) -> Tile {
        if constexpr (!DOCS) return Tile{next_t++, true, true, true};
        while (live == 0) {
            run += 64;
            if (run >= last) return Tile{last, false, false, false};
            look(run);
        }
        const int i = __builtin_ctzll(live);
        live &= live - 1;
        return Tile{run + i, (one_b >> i & 1) != 0, (one_w >> i & 1) != 0, (seen_w >> i & 1) != 0};
    };

    const bool keeps = SPLIT && p.scores && wave_rows && wrow0 < p.score_rows;   // this wave keeps scores
    float* score_row = nullptr;
    if (keeps && has_row && row < p.score_rows)
        score_row = p.scores + ((int64_t)(b * p.heads + hb) * p.score_rows + row) * p.score_pitch;
    // this lane's row sees the keys below lim, but for documents and trees
    const int lim = p.causal ? min(len.k, max(pos + 1, prefix)) : len.k;
    auto in_tree = [&](int j) __attribute__((always_inline)) { return j < len.old || (tree >> ((j - len.old) & 63) & 1); };

    // ---- loop ----
    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x16{};
    RowState<BF> st;
    // Weights are exp2(f x).  A capped score is cap tanh(y) = cap - 2 cap t, with
    // t = 1 / (1 + e^(2 y)): x = -t, the constant drops out of the softmax (with a
    // bias the score itself is formed).  Off by 9 * 2^-24 cap, at the largest cap that
    // takes this form a fourteenth of what rounding to fp16 costs a weight.  Larger
    // caps, and parts, which may serve fp32 weights, take the form that is as close at
    // any cap (capped).  4096 causal rows of 32 heads, head_dim 64 / 128: 91 / 147 us
    // without a cap, 120 / 183 in the short form, 160 / 219 in the other.
    const float f = BIAS || CLOSE ? kLog2e : CAP ? 2.0f * p.cap * kLog2e : p.scale * kLog2e;
    const float capscale = !CAP ? 0.0f : CLOSE ? p.scale / p.cap : 2.0f * kLog2e * p.scale / p.cap;
    const float* bias = BIAS ? p.bias + head * p.bias_h : nullptr;
    const uint32_t kfrag = klds + k_frag_base<D>(lane), vfrag = vlds + v_frag_base<D>(lane);

    // The tiles are gone through again where that gave an infinity or NaN: then with
    // care for those in V that only some rows see.
    for (int careful = 0; careful < 2; ++careful) {
    bool partly = false;   // some row did not see some key
    bool stored = false;   // the wave kept scores of the tile before
    Tile cur = advance(), nxt = cur;
    if (cur.t < last) {
        copy(cur.t, 0);
        nxt = advance();
    }
    for (int stage = 0; cur.t < last; stage ^= 1) {
        const int j0 = cur.t * kTileKeys, j1 = j0 + kTileKeys - 1;
        // does every row of the block see every key of the tile?
        const bool some = !(j1 < len.k && (!p.causal || j1 <= bpos0 || j1 < prefix) &&
                            cur.one_b && (!(SPLIT && p.tree) || j1 < len.old));
        partly |= some;
        if (careful && threadIdx.x < 2) bad_keys[stage][threadIdx.x] = 0;
        // This tile is in LDS, and the stage of the one before is free.  The tile
        // before's scores, 8 stores (4 with WK = 2) and the last that the wave issued,
        // need not have arrived.
        if (SPLIT && stored) copies_wait<4 * KB>();
        else copies_wait<0>();
        if constexpr (SPLIT) stored = false;
        __syncthreads();
        if (nxt.t < last) copy(nxt.t, stage ^ 1);
        if (careful && some) {
#pragma unroll
            for (int i = 0; i < TILE / 8 / 256; ++i) {
                const int piece = i * 256 + threadIdx.x, key = piece / (D / 8);
                if (clear_piece<BF>(vlds + stage * (TILE * 2) + piece * 16))
                    atomicOr(&bad_keys[stage][key >> 5], 1u << (key & 31));
            }
            __syncthreads();
        }
        const bool sees = wave_rows && (!p.causal || j0 <= wpos1 || j0 < prefix) &&
                          cur.seen_w;
        if (sees) {
            if constexpr (SPLIT) stored = keeps;
            const bool all = j1 < len.k && (!p.causal || j1 <= wpos0 || j1 < prefix) &&
                             cur.one_w && (!(SPLIT && p.tree) || j1 < len.old);
            uint32_t ka[QT], va[DB];   // lane addresses of the tile's fragments
#pragma unroll
            for (int t = 0; t < QT; ++t) ka[t] = opaque((kfrag ^ (t << 5)) + stage * (TILE * 2) + wave_key * (64 * D));
#pragma unroll
            for (int db = 0; db < DB; ++db) va[db] = opaque((vfrag ^ (db << 6)) + stage * (TILE * 2) + wave_key * (64 * D));
            f32x16 s[KB] = {};
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int t = 0; t < QT; ++t) s[kb] = mfma32<BF>(lds_16(ka[t] + kb * (64 * D)), qf[t], s[kb]);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int jb = j0 + (wave_key + kb) * 32;   // its first key
                u32x4 pf[2], vf[2][DB];
                // V's fragments (at head_dim 128 the first half of them, for registers)
                // are on their way while the weights are formed
                constexpr int AHEAD = D == 64 && !SPLIT ? 2 : 1;
                auto values = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const uint32_t a = va[db] + (kb * 2 + ks) * (32 * D);
                        const u32x2 x = lds_tr8(a), y = lds_tr8(a + 16 * D);
                        vf[ks][db] = u32x4{x[0], x[1], y[0], y[1]};
                    }
                };
#pragma unroll
                for (int ks = 0; ks < AHEAD; ++ks) values(ks);
                if constexpr (CAP || BIAS) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float x = s[kb][i];
                        if constexpr (CLOSE) x = capped(x, capscale, p.scale, p.cap);
                        else if constexpr (CAP) x = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(x * capscale));
                        if constexpr (BIAS) {
                            const int j = jb + 8 * (i / 4) + 4 * h + i % 4;
                            x = (CLOSE ? x : CAP ? p.cap + 2.0f * p.cap * x : x * p.scale) +
                                bias[min(max(j - pos + p.bias_zero, 0), p.bias_n - 1)];
                        }
                        s[kb][i] = x;
                    }
                }
                if (!all) {
                    const int d = lim - jb - 4 * h;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[kb][i] = 8 * (i / 4) + i % 4 < d ? s[kb][i] : -kInf;
                    if constexpr (DOCS) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int4 e = *reinterpret_cast<const int4*>(&tile_docs[stage][(wave_key + kb) * 32 + 8 * i + 4 * h]);
                            s[kb][4 * i] = e.x == qdoc ? s[kb][4 * i] : -kInf;
                            s[kb][4 * i + 1] = e.y == qdoc ? s[kb][4 * i + 1] : -kInf;
                            s[kb][4 * i + 2] = e.z == qdoc ? s[kb][4 * i + 2] : -kInf;
                            s[kb][4 * i + 3] = e.w == qdoc ? s[kb][4 * i + 3] : -kInf;
                        }
                        if (qdoc < 0) s[kb] = f32x16{} - kInf;   // of no document
                    }
                    if (SPLIT && p.tree) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            s[kb][i] = in_tree(jb + 8 * (i / 4) + 4 * h + i % 4) ? s[kb][i] : -kInf;
                    }
                }
                if constexpr (SPLIT) {
                    if (keeps && score_row) keep_scores(score_row, jb, h, f, s[kb]);
                }
                st.template take<BIAS, SPLIT, DB>(s[kb], f, pf, o);
#pragma unroll
                for (int ks = AHEAD; ks < 2; ++ks) values(ks);
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int db = 0; db < DB; ++db) o[db] = mfma32<BF>(vf[ks][db], pf[ks], o[db]);
            }
            if (careful && some) {   // keys with infinities or NaN in their V rows
                uint64_t bad = (uint64_t)bad_keys[stage][1] << 32 | bad_keys[stage][0];
                // Rows that overlap (a stride below head_dim) put values of the last keys
                // into the places of keys past the end, which have no row to read.
                if (j1 >= len.k) bad &= (1ull << (len.k - j0)) - 1;
                while (bad) {
                    const int j = j0 + __builtin_ctzll(bad);
                    bad &= bad - 1;
                    const bool mine = has_row && (WK == 1 || (j - j0) / 32 == wave_key) && j < lim && (!DOCS || (qdoc >= 0 && tile_docs[stage][j - j0] == qdoc)) &&
                                      (!(SPLIT && p.tree) || in_tree(j));
                    const late_params_t e = late_params();
                    add_values<D, BF>(o, vbase + j * e->vs.r, e->D, h, mine);
                }
            }
        }
        cur = nxt;
        if (nxt.t < last) nxt = advance();
    }
    if (careful || !partly) break;
    float any = 0.0f * st.l;   // NaN where a sum is infinite or NaN
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) any = fmaf(o[i][e], 0.0f, any);
    if (!__syncthreads_or(has_row && any != any)) break;
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x16{};
    st = RowState<BF>();
    live = 0;
    run = first - 64;
    next_t = first;
    }

    // ---- the two halves of the keys ----
    float l = half_sum(st.l);
    if constexpr (WK == 2) {
        // 32 rows of D sums for each of the waves of the second half, in pieces of 4
        // that are permuted by the row; the tiles are not read any more
        constexpr int P = D / 4;
        float* sums = reinterpret_cast<float*>(&ks[0][0]) + wave_row * (32 * D);
        static_assert(2 * 32 * D * sizeof(float) <= sizeof(ks), "the sums fit");
        __syncthreads();
        if (wave_key == 1) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4*>(sums + n * D + ((8 * db + 2 * i + h) ^ (n & (P - 1))) * 4) =
                        f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
            if (h == 0) *reinterpret_cast<f32x2*>(half_ml[wave_row][n]) = f32x2{BIAS ? st.m : st.mf, l};
        }
        __syncthreads();
        if (wave_key == 1) return;
        const f32x2 other = *reinterpret_cast<const f32x2*>(half_ml[wave_row][n]);
        const float m0 = BIAS ? st.m : st.mf, m = fmaxf(m0, other[0]);
        const float a0 = __builtin_amdgcn_exp2f(BIAS ? (m0 - m) * f : m0 - m);
        const float a1 = __builtin_amdgcn_exp2f(BIAS ? (other[0] - m) * f : other[0] - m);
        st.mf = m;   // only parts need it, and they have no bias
        l = a0 * l + a1 * other[1];
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 y = *reinterpret_cast<const f32x4*>(sums + n * D + ((8 * db + 2 * i + h) ^ (n & (P - 1))) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[db][4 * i + e] = a0 * o[db][4 * i + e] + a1 * y[e];
            }
    }

    // ---- output ----
    if (!has_row) return;
    const late_params_t e = late_params();
    if constexpr (SPLIT) {
        const int64_t at = (int64_t)hs * ((int64_t)e->Sq * e->pack) + row;
        float* po = e->part_o + at * D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(po + 32 * db + 8 * i + 4 * h) =
                    f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
        if (h == 0) *reinterpret_cast<f32x2*>(e->part_ml + at * 2) = f32x2{st.mf, l};
    } else {
        // a row that sees nothing is 0
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* out = e->out + b * e->os.b + (int64_t)qi * e->os.r + (int64_t)head * e->os.h;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 32 * db + 8 * i + 4 * h;
                if (c < e->D)
                    *reinterpret_cast<u32x2*>(out + c) = u32x2{pack2<BF>(o[db][4 * i] * inv, o[db][4 * i + 1] * inv),
                                                              pack2<BF>(o[db][4 * i + 2] * inv, o[db][4 * i + 3] * inv)};
            }
    }
}

template <int D, bool BF, int MODE, int WK>
static hipError_t launch_one(const AttnParams& p, dim3 g, hipStream_t st) {
    hipLaunchKernelGGL((attn_seq_kernel<D, BF, MODE, WK>), g, dim3(256), 0, st, p);
    return hipGetLastError();
}
template <int D, bool BF, int WK>
static hipError_t launch_mode(const AttnParams& p, dim3 g, hipStream_t st) {
    const int mode = (p.cap > 0.0f ? kCap : 0) | (p.cap > kShortCap && !p.part_o ? kClose : 0) | (p.bias ? kBias : 0) |
                     (p.part_o ? kSplit : 0) | (p.q_docs ? kDocs : 0);
    switch (mode) {
        case 0: return launch_one<D, BF, 0, WK>(p, g, st);
        case kCap: return launch_one<D, BF, kCap, WK>(p, g, st);
        case kBias: return launch_one<D, BF, kBias, WK>(p, g, st);
        case kCap | kBias: return launch_one<D, BF, kCap | kBias, WK>(p, g, st);
        case kDocs: return launch_one<D, BF, kDocs, WK>(p, g, st);
        case kDocs | kCap: return launch_one<D, BF, kDocs | kCap, WK>(p, g, st);
        case kDocs | kBias: return launch_one<D, BF, kDocs | kBias, WK>(p, g, st);
        case kDocs | kCap | kBias: return launch_one<D, BF, kDocs | kCap | kBias, WK>(p, g, st);
        case kClose | kCap: return launch_one<D, BF, kClose | kCap, WK>(p, g, st);
        case kClose | kCap | kBias: return launch_one<D, BF, kClose | kCap | kBias, WK>(p, g, st);
        case kClose | kDocs | kCap: return launch_one<D, BF, kClose | kDocs | kCap, WK>(p, g, st);
        case kClose | kDocs | kCap | kBias: return launch_one<D, BF, kClose | kDocs | kCap | kBias, WK>(p, g, st);
        case kSplit: return launch_one<D, BF, kSplit, WK>(p, g, st);
        case kSplit | kCap: return launch_one<D, BF, kSplit | kCap, WK>(p, g, st);
        default: return hipErrorInvalidValue;   // parts have neither documents nor a bias
    }
}

template <int D>
static hipError_t launch_dim(const AttnParams& p, dim3 g, hipStream_t st) {
    if (p.halves) return p.bf16 ? launch_mode<D, true, 2>(p, g, st) : launch_mode<D, false, 2>(p, g, st);
    return p.bf16 ? launch_mode<D, true, 1>(p, g, st) : launch_mode<D, false, 1>(p, g, st);
}

}  // namespace sltx
