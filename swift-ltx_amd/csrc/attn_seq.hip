// attn_seq.hip -- attention of many query rows: o = softmax(x) v with
// x = cap tanh(scale q.k / cap) + bias[j - pos(i)], over the keys that a row
// sees (causal, prefix, documents, lengths, a tree of drafted tokens).
//
// A block of 4 waves takes 128 query rows (32 a wave, Q in registers) over all
// keys, or over one of `splits` ranges of them.  Tiles of 64 keys pass through
// two stages of LDS, copied while the tiles before are computed.  One pass over the keys with a running maximum and sum; nothing but
// the output is written.
#include "attn_tile.hpp"

namespace sltx {

// Variants.  Documents, and the parts that a cached attention is split into (the
// only ones with a tree), have kernels of their own: their state costs registers.
enum : int { kCap = 1, kBias = 2, kSplit = 4, kDocs = 8 };

// Documents of a run of 64 tiles (one lane each): the smallest and largest id
// of a tile's keys, ids below 0 (padding) left out, and whether all are equal.
struct DocTiles {
    int lo[64], hi[64], same[64];
};

template <int D, bool BF, int MODE>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_seq_kernel(AttnParams p) {
    constexpr bool CAP = MODE & kCap, BIAS = MODE & kBias, SPLIT = MODE & kSplit, DOCS = MODE & kDocs;
    constexpr int TILE = kTileKeys * D;          // values of a tile
    constexpr int QT = D / 16, DB = D / 32;
    constexpr int INSTR = TILE * 2 / 1024 / 4;   // copies of a wave into a tile
    __shared__ __attribute__((aligned(1024))) uint16_t ks[2][TILE], vs[2][TILE];
    __shared__ DocTiles docs;
    __shared__ __attribute__((aligned(16))) int tile_docs[kTileKeys];   // documents of a tile's keys
    __shared__ uint32_t bad_keys[2][2];   // [stage]: its keys whose V rows are not finite

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;

    // Blocks go round the 8 XCDs in turn: each XCD gets a contiguous run of the
    // (sequence, head, tile, split) order, so that the blocks that share keys
    // share an L2.  The last tiles, which see the most keys under a causal mask,
    // come first.
    const int total = p.B * p.heads * p.tiles * p.splits;
    const int per = (total + 7) / 8;
    int w = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (w >= min(total, ((int)(blockIdx.x & 7) + 1) * per)) return;
    const int split = SPLIT ? w % p.splits : 0;
    if (SPLIT) w /= p.splits;
    const int tile = p.tiles - 1 - w % p.tiles;
    w /= p.tiles;
    const int hb = w % p.heads, b = w / p.heads;
    const SeqLens len = seq_lens(p, b);
    const int rows = len.q * p.pack;
    const int row0 = tile * kSeqTileRows;
    if (row0 >= rows) return;

    // this lane's query row
    const int row = row0 + wave * 32 + n;
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
    const int wrow0 = row0 + wave * 32;
    const bool wave_rows = wrow0 < rows;
    const int wpos0 = wrow0 / p.pack + len.shift;
    const int wpos1 = (min(wrow0 + 31, rows - 1)) / p.pack + len.shift;
    const int bpos0 = row0 / p.pack + len.shift;
    const int bpos1 = (min(row0 + kSeqTileRows, rows) - 1) / p.pack + len.shift;
    const int pos = qi + len.shift;
    const int prefix = p.prefix ? p.prefix[b] : 0;
    const int kend = p.causal ? min(len.k, max(bpos1 + 1, prefix)) : len.k;
    int first = 0, last = (kend + kTileKeys - 1) / kTileKeys;   // tiles
    if (SPLIT) {
        const int each = (last + p.splits - 1) / p.splits;
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
    };

    // ---- which tiles ----
    // The tiles of [first, last) that some row of the block may see, in order.
    // With documents, runs of 64 tiles are looked through at a time: `live` has
    // a bit for each.
    uint64_t live = 0;
    int run = first - 64, next_t = first;
    auto look = [&](int at) __attribute__((always_inline)) {   // all threads: fills docs for tiles at .. at + 63
        const int t = threadIdx.x >> 2, j = (at + t) * kTileKeys + (threadIdx.x & 3) * 16;
        int lo = 0x7fffffff, hi = -1, low = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int k = kdocs[min(j + e, kend - 1)], d = j + e < kend ? k : -1;
            lo = min(lo, d < 0 ? 0x7fffffff : d);
            low = min(low, d);
            hi = max(hi, d);
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
        live = __ballot(at + lane < last && docs.hi[lane] >= bdoc0 && docs.lo[lane] <= bdoc1);
    };
    struct Tile {
        int t, lo, hi, same;
    };
    auto advance = [&]() __attribute__((always_inline)) -> Tile {
        if constexpr (!DOCS) return Tile{next_t++, 0, 0, 1};
        while (live == 0) {
            run += 64;
            if (run >= last) return Tile{last, 0, 0, 0};
            look(run);
        }
        const int i = __builtin_ctzll(live);
        live &= live - 1;
        return Tile{run + i, __builtin_amdgcn_readfirstlane(docs.lo[i]), __builtin_amdgcn_readfirstlane(docs.hi[i]),
                    __builtin_amdgcn_readfirstlane(docs.same[i])};
    };

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
    // bias the score itself is formed).  Off by 9 * 2^-24 cap: enough for weights of
    // 16 bits.  Parts may serve fp32 weights and take the closer form (capped).
    const float f = BIAS || (CAP && SPLIT) ? kLog2e : CAP ? 2.0f * p.cap * kLog2e : p.scale * kLog2e;
    const float capscale = !CAP ? 0.0f : SPLIT ? p.scale / p.cap : 2.0f * kLog2e * p.scale / p.cap;
    const float* bias = BIAS ? p.bias + head * p.bias_h : nullptr;
    const uint32_t kfrag = klds + k_frag_base<D>(lane), vfrag = vlds + v_frag_base<D>(lane);

    Tile cur = advance();
    if (cur.t < last) copy(cur.t, 0);
    for (int stage = 0; cur.t < last; stage ^= 1) {
        const Tile nxt = advance();
        const int j0 = cur.t * kTileKeys, j1 = j0 + kTileKeys - 1;
        // does every row of the block see every key of the tile?
        const bool some = !(j1 < len.k && (!p.causal || j1 <= bpos0 || j1 < prefix) &&
                            (!DOCS || (cur.same && cur.lo == bdoc)) && (!(SPLIT && p.tree) || j1 < len.old));
        if (some && threadIdx.x < 2) bad_keys[stage][threadIdx.x] = 0;
        copies_wait<0>();
        __syncthreads();     // this tile is in LDS, the other stage free
        if (nxt.t < last) copy(nxt.t, stage ^ 1);
        if (some) {
#pragma unroll
            for (int i = 0; i < TILE / 8 / 256; ++i) {
                const int piece = i * 256 + threadIdx.x, key = piece / (D / 8);
                if (clear_piece<BF>(vlds + stage * (TILE * 2) + piece * 16))
                    atomicOr(&bad_keys[stage][key >> 5], 1u << (key & 31));
            }
            if (DOCS && threadIdx.x < kTileKeys) {
                const int j = j0 + threadIdx.x;
                tile_docs[threadIdx.x] = j < len.k ? kdocs[j] : -1;
            }
            __syncthreads();
        }
        const bool sees = wave_rows && (!p.causal || j0 <= wpos1 || j0 < prefix) &&
                          (!DOCS || (cur.hi >= wdoc0 && cur.lo <= wdoc1));
        if (sees) {
            const bool all = j1 < len.k && (!p.causal || j1 <= wpos0 || j1 < prefix) &&
                             (!DOCS || (cur.same && cur.lo == wdoc)) && (!(SPLIT && p.tree) || j1 < len.old);
            uint32_t ka[QT], va[DB];   // lane addresses of the tile's fragments
#pragma unroll
            for (int t = 0; t < QT; ++t) ka[t] = opaque((kfrag ^ (t << 5)) + stage * (TILE * 2));
#pragma unroll
            for (int db = 0; db < DB; ++db) va[db] = opaque((vfrag ^ (db << 6)) + stage * (TILE * 2));
            f32x16 s[2];
            u32x4 pf[2][2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                s[kb] = f32x16{};
#pragma unroll
                for (int t = 0; t < QT; ++t) s[kb] = mfma32<BF>(lds_16(ka[t] + kb * (64 * D)), qf[t], s[kb]);
            }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                if constexpr (CAP || BIAS) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float x = s[kb][i];
                        if constexpr (CAP && SPLIT) x = capped(x * capscale, p.cap);
                        else if constexpr (CAP) x = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(x * capscale));
                        if constexpr (BIAS) {
                            const int j = j0 + kb * 32 + 8 * (i / 4) + 4 * h + i % 4;
                            x = (CAP ? p.cap + 2.0f * p.cap * x : x * p.scale) +
                                bias[min(max(j - pos + p.bias_zero, 0), p.bias_n - 1)];
                        }
                        s[kb][i] = x;
                    }
                }
                if (!all) {
                    const int d = lim - j0 - 4 * h;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[kb][i] = kb * 32 + 8 * (i / 4) + i % 4 < d ? s[kb][i] : -kInf;
                    if constexpr (DOCS) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int4 e = *reinterpret_cast<const int4*>(&tile_docs[kb * 32 + 8 * i + 4 * h]);
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
                            s[kb][i] = in_tree(j0 + kb * 32 + 8 * (i / 4) + 4 * h + i % 4) ? s[kb][i] : -kInf;
                    }
                }
                st.template take<BIAS, SPLIT, DB>(s[kb], f, pf[kb], o);
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const uint32_t a = va[db] + (kb * 2 + ks) * (32 * D);
                        const u32x2 x = lds_tr8(a), y = lds_tr8(a + 16 * D);
                        o[db] = mfma32<BF>(u32x4{x[0], x[1], y[0], y[1]}, pf[kb][ks], o[db]);
                    }
            }
            if (some) {   // keys with infinities or NaN in their V rows
                uint64_t bad = (uint64_t)bad_keys[stage][1] << 32 | bad_keys[stage][0];
                while (bad) {
                    const int j = j0 + __builtin_ctzll(bad);
                    bad &= bad - 1;
                    const bool mine = has_row && j < lim && (!DOCS || (qdoc >= 0 && tile_docs[j - j0] == qdoc)) &&
                                      (!(SPLIT && p.tree) || in_tree(j));
                    add_values<D, BF>(o, vbase + j * p.vs.r, p.D, h, mine);
                }
            }
        }
        cur = nxt;
    }

    // ---- output ----
    const float l = half_sum(st.l);
    if (!has_row) return;
    if constexpr (SPLIT) {
        const int64_t at = ((int64_t)(b * p.heads + hb) * p.splits + split) * ((int64_t)p.Sq * p.pack) + row;
        float* po = p.part_o + at * D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4*>(po + 32 * db + 8 * i + 4 * h) =
                    f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
        if (h == 0) *reinterpret_cast<f32x2*>(p.part_ml + at * 2) = f32x2{st.mf, l};
    } else {
        // a row that sees nothing is 0
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* out = p.out + b * p.os.b + (int64_t)qi * p.os.r + (int64_t)head * p.os.h;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 32 * db + 8 * i + 4 * h;
                if (c < p.D)
                    *reinterpret_cast<u32x2*>(out + c) = u32x2{pack2<BF>(o[db][4 * i] * inv, o[db][4 * i + 1] * inv),
                                                              pack2<BF>(o[db][4 * i + 2] * inv, o[db][4 * i + 3] * inv)};
            }
    }
}

template <int D, bool BF, int MODE>
static hipError_t launch_one(const AttnParams& p, dim3 g, hipStream_t st) {
    hipLaunchKernelGGL((attn_seq_kernel<D, BF, MODE>), g, dim3(256), 0, st, p);
    return hipGetLastError();
}
template <int D, bool BF>
static hipError_t launch_mode(const AttnParams& p, dim3 g, hipStream_t st) {
    const int mode = (p.cap > 0.0f ? kCap : 0) | (p.bias ? kBias : 0) | (p.part_o ? kSplit : 0) | (p.q_docs ? kDocs : 0);
    switch (mode) {
        case 0: return launch_one<D, BF, 0>(p, g, st);
        case kCap: return launch_one<D, BF, kCap>(p, g, st);
        case kBias: return launch_one<D, BF, kBias>(p, g, st);
        case kCap | kBias: return launch_one<D, BF, kCap | kBias>(p, g, st);
        case kDocs: return launch_one<D, BF, kDocs>(p, g, st);
        case kDocs | kCap: return launch_one<D, BF, kDocs | kCap>(p, g, st);
        case kDocs | kBias: return launch_one<D, BF, kDocs | kBias>(p, g, st);
        case kDocs | kCap | kBias: return launch_one<D, BF, kDocs | kCap | kBias>(p, g, st);
        case kSplit: return launch_one<D, BF, kSplit>(p, g, st);
        case kSplit | kCap: return launch_one<D, BF, kSplit | kCap>(p, g, st);
        default: return hipErrorInvalidValue;   // parts have neither documents nor a bias
    }
}

hipError_t launch_attn_seq(AttnParams p, hipStream_t st) {
    p.tiles = (int)(((int64_t)p.Sq * p.pack + kSeqTileRows - 1) / kSeqTileRows);
    const int64_t total = (int64_t)p.B * p.heads * p.tiles * p.splits;
    if (total == 0) return hipSuccess;
    if (total > 0x7fffff00 / 256) return hipErrorInvalidValue;
    const dim3 g((unsigned)((total + 7) / 8 * 8));
    if (p.D > 64) return p.bf16 ? launch_mode<128, true>(p, g, st) : launch_mode<128, false>(p, g, st);
    return p.bf16 ? launch_mode<64, true>(p, g, st) : launch_mode<64, false>(p, g, st);
}

}  // namespace sltx
