// attn_tile.hpp -- the pieces that the attention kernels share (attn_seq_kernel.hpp,
// attn_few.hip): tiles of keys and values in LDS, their MFMA fragments, and the
// softmax's running maximum.
//
// Orientation.  Both products are formed transposed, S^T = K Q^T and
// O^T = V^T P^T, on 32x32x16 MFMAs.  In their result layout lane l holds
// column l & 31 (one query row) and the matrix rows 8*(i/4) + 4*(l/32) + i%4,
// i = 0..15 (16 of 32 keys, or of 32 output columns): a row's maximum and sum
// are taken within a lane and with lane l ^ 32, and the statistics are one
// register each.  The registers that hold P^T after S^T's MFMAs are the second
// product's B fragments as they stand: a contraction may run over its keys in
// any order that both operands share, and V^T is read from LDS in the order
// that P^T has (v_frag).
#pragma once

#include <type_traits>

#include "attn_launch.hpp"
#include "q4_common.hpp"

namespace sltx {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) char* lds_char_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

// ---- tiles in LDS ----
// A tile is ROWS rows of D values of 16 bits (D = 64 or 128; a head dim below
// is padded with zeros).  The 16-byte pieces of a row are permuted by the row,
// against bank conflicts in both ways of reading: K rows are read as pieces by 16
// consecutive rows at a time, V rows as 4 rows x 16 columns.  Some are left:
// counters have 33% of the LDS's active cycles as conflicts at head_dim 64 (6144
// rows), 31% at 128 (750 rows); waits for LDS are 3% of the waves' cycles at most.
template <int D>
__device__ __forceinline__ int k_swizzle(int row) {
    return D == 128 ? row & 15 : (row >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
    return D == 128 ? (row & 7) << 1 : ((row >> 1) & 3) << 1;
}

// The copies of one wave into a tile of which it fills INSTR pieces of 1 KB:
// byte offsets of each lane's piece from the tile's first row in memory.
// Pieces past the head dim get an offset that the buffer's bounds check turns
// into zeros, as it does for the rows past the end (tile_rsrc).
constexpr int kOutside = 0x7fffff00;
template <int D, bool V, int INSTR>
struct TileCopy {
    int off[INSTR];
    __device__ __forceinline__ void init(int first, int lane, int stride, int head_bytes) {
        constexpr int P = D / 8;   // pieces of a row
#pragma unroll
        for (int i = 0; i < INSTR; ++i) {
            const int row = (first + i) * (64 / P) + lane / P, p = lane % P;
            const int c = p ^ (V ? v_swizzle<D>(row) : k_swizzle<D>(row));
            off[i] = c * 16 < head_bytes ? row * stride + c * 16 : kOutside;
        }
    }
};

// The buffer that holds `rows` rows (at least 1) from `base` on.
__device__ __forceinline__ u32x4 tile_rsrc(const uint16_t* base, int rows, int stride, int head_bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    u32x4 r = {(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, (uint32_t)((rows - 1) * stride + head_bytes),
               0x00020000u};
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_readfirstlane(r[i]);
    return r;
}

// One copy of 1 KB, lane l's 16 bytes to lds + 16 l.  Written as asm so that
// the compiler's wait counts do not know of it: it cannot tell a copy into one
// stage from a read of another, and would drain every copy before each read.
// The kernels wait themselves (copies_wait) before the barrier or the read
// that hands a stage over.  The instruction has no register output; m0 is a
// reserved register that nothing else in these kernels uses.
__device__ __forceinline__ void copy_1k(u32x4 rsrc, int off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :: "v"(off), "s"(rsrc), "s"(lds) : "memory");
}
// The same of 4 bytes a lane.
__device__ __forceinline__ void copy_256(u32x4 rsrc, int off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
                 :: "v"(off), "s"(rsrc), "s"(lds) : "memory");
}
// Waits for all but the N copies issued last.
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_char_t)(p));
}

// A value that the compiler does not take apart again.
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
    asm("" : "+v"(x));
    return x;
}
// A kernel's parameters, loaded where they are used: parameters that only the end
// or a rare path needs would otherwise be held in scalar registers throughout.
typedef __attribute__((address_space(4))) const AttnParams* late_params_t;
__device__ __forceinline__ late_params_t late_params() {
    auto k = (late_params_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(k));
    return k;
}
// A pointer that is the same in every lane, held in scalar registers.
__device__ __forceinline__ const uint16_t* uniform(const uint16_t* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
    return reinterpret_cast<const uint16_t*>((uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ u32x4 lds_16(uint32_t a) {
    return *(__attribute__((address_space(3))) const u32x4*)(uintptr_t)(a);
}
__device__ __forceinline__ u32x2 lds_tr8(uint32_t a) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) s16x4*)(uintptr_t)(a)));
}

// Lane addresses of the fragments within a tile at LDS offset 0 (or at a multiple
// of 256 added to the base), and the fragments themselves `tile` bytes further on.
// K as A operand: lane l holds key l & 31, columns 16 t + 8 (l >> 5) .. + 7.
template <int D>
__device__ __forceinline__ uint32_t k_frag_base(int lane) {
    const int row = lane & 31;
    return row * (2 * D) + (((lane >> 5) ^ k_swizzle<D>(row)) << 4);
}
template <int D>
__device__ __forceinline__ u32x4 k_frag(uint32_t tile, uint32_t base, int block, int t) {
    return lds_16((base ^ (t << 5)) + tile + block * (64 * D));
}
// V^T as A operand of 16 keys: lane l holds column 32 db + (l & 31) and, in the
// order of P^T's registers, keys 8 (j / 4) + 4 (l >> 5) + j % 4, j = 0..7, of 16:
// two transposing reads of 4 keys each.
template <int D>
__device__ __forceinline__ uint32_t v_frag_base(int lane) {
    const int row = 4 * (lane >> 5) + ((lane >> 2) & 3);
    return row * (2 * D) + ((((lane >> 4) & 1) << 5) ^ (v_swizzle<D>(row) << 4)) + (lane & 3) * 8;
}
template <int D>
__device__ __forceinline__ u32x4 v_frag(uint32_t tile, uint32_t base, int ks, int db) {
    const uint32_t a = (base ^ (db << 6)) + tile + ks * (32 * D);
    const u32x2 x = lds_tr8(a), y = lds_tr8(a + 16 * D);
    return u32x4{x[0], x[1], y[0], y[1]};
}

// ---- arithmetic ----
template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two values rounded to nearest even.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// acc + both of two packed values
template <bool BF>
__device__ __forceinline__ float add2(uint32_t v, float acc) {
    if constexpr (BF)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, v), bf16x2{(__bf16)1.0f, (__bf16)1.0f}, acc, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, v), f16x2{(f16)1.0f, (f16)1.0f}, acc, false);
}

// max / sum with the other half of the wave (lane l ^ 32)
__device__ __forceinline__ float half_max(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// The score scale * s capped: cap tanh(y), y = yscale * s, yscale = scale / cap.  tanh as
// (1 - e) / (1 + e) with e = exp(-2 |y|); below |y| = 0.25, where 1 - e would cancel,
// x = scale * s times its series in y^2 (next term under 1e-8): within 16 * 2^-24 of the
// value whatever the cap is, up to those of which y and cap are at the ends of fp32.
__device__ __forceinline__ float capped(float s, float yscale, float scale, float cap) {
    const float y = s * yscale, x = s * scale, a = fabsf(y), y2 = y * y;
    const float e = __builtin_amdgcn_exp2f(-2.0f * kLog2e * a);
    const float big = cap * (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
    const float small = x + x * y2 * (-1.0f / 3 + y2 * (2.0f / 15 + y2 * (-17.0f / 315 + y2 * (62.0f / 2835))));
    return a < 0.25f ? small : copysignf(big, x);
}

// ---- non-finite values in masked places ----
// A masked key has weight 0, but 0 times an infinity or NaN in its V row would
// still put NaN into rows that do not see it.  In tiles where some row may not
// see some key, such values are cleared in LDS before the product (clear_piece)
// and added afterwards to the rows that see their key (add_values): they are
// what such a row's sum comes to.
template <bool BF>
__device__ __forceinline__ bool nonfinite(uint32_t x) {   // of the low 16 bits
    constexpr uint32_t e = BF ? 0x7f80u : 0x7c00u;
    return (x & e) == e;
}
// Clears the non-finite values of a tile's piece (16 bytes at LDS address a);
// whether there were any.
template <bool BF>
__device__ __forceinline__ bool clear_piece(uint32_t a) {
    u32x4 v = lds_16(a);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool lo = nonfinite<BF>(v[i]), hi = nonfinite<BF>(v[i] >> 16);
        v[i] = (lo ? 0 : v[i] & 0xffffu) | (hi ? 0 : v[i] & 0xffff0000u);
        bad |= lo | hi;
    }
    if (bad) *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(a) = v;
    return bad;
}
// Adds the non-finite values of V row `v` to the lane's sums (for lanes whose
// row sees it).
template <int D, bool BF>
__device__ __forceinline__ void add_values(f32x16 (&o)[D / 32], const uint16_t* v, int head_dim, int h, bool sees) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 32 * db + 8 * i + 4 * h;
            const u32x2 x = *reinterpret_cast<const u32x2*>(v + min(c, head_dim - 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t y = x[e / 2] >> (e % 2 * 16) & 0xffffu;
                const float z = BF ? bf2f((uint16_t)y) : h2f((uint16_t)y);
                o[db][4 * i + e] += (sees && nonfinite<BF>(y) && c < head_dim) ? z : 0.0f;
            }
            __builtin_amdgcn_sched_barrier(0);   // rare: few registers, not speed
        }
}

// o += V^T P^T over the KS * 16 keys of the tile at `tile`.
template <int D, bool BF, int KS>
__device__ __forceinline__ void weigh_values(f32x16 (&o)[D / 32], const u32x4 (&pf)[KS], uint32_t tile,
                                             uint32_t base) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int db = 0; db < D / 32; ++db) o[db] = mfma32<BF>(v_frag<D>(tile, base, ks, db), pf[ks], o[db]);
        __builtin_amdgcn_sched_barrier(0);   // few fragments at a time
    }
}

// ---- running softmax of one lane's column ----
// Weights are exp2(f x - mf), with x the (capped, biased) score.  mf is f times
// the largest score at some time past, plus kSpare: the row's largest weight
// then is 2^-kSpare, and as long as the 16 weights of a lane sum to less than kMost,
// nothing has to be rescaled.  So the weights are formed without a look at the maximum,
// and their sum tells afterwards whether one may have left that range (or is an
// infinity or NaN).  Only then is the maximum taken, and the step done again (grow).
// bf16 has fp32's range: any scale serves.  fp16 does not: its largest weight
// is 2^8 or more, 2^15 less at most, so that it keeps 11 binary digits of weights down to
// 2^-22 of the largest, and loses those below 2^-33 of it, more than 2^22 of which it
// would take to add up to the output's last digit.  After grow 16 weights sum to 2^-3
// (bf16) or 2^12 (fp16) at most: no row grows twice for one maximum.
template <bool BF>
struct RowState {
    static constexpr float kSpare = BF ? 7.0f : -8.0f, kMost = BF ? 2.0f : 32768.0f;
    // Nothing seen so far: finite, so that masked scores (-inf) get the weight 0
    // and any other an infinite one.
    static constexpr float kNone = -3.4028235e38f;
    float m = kNone, mf = kNone, l = 0.0f;

    // p = weights of 32 keys as P^T fragments, rounded to nearest; sum = their sum
    // as rounded, so that the output is a mean of values, or unrounded where it
    // will divide fp32 weights (EXACT).  Returns whether the lane's weights have left
    // their range.  BIASED: a bias may be as low as the type goes, where f x overflows,
    // so the difference is taken first.
    template <bool BIASED, bool EXACT>
    __device__ __forceinline__ bool weigh(const f32x16& x, float f, u32x4 (&p)[2], float& sum) const {
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            // fused by name: the two copies of this (take, grow) have to agree to the bit
            const float w0 = __builtin_amdgcn_exp2f(BIASED ? fmaf(x[i] - m, f, -kSpare) : fmaf(x[i], f, -mf));
            const float w1 = __builtin_amdgcn_exp2f(BIASED ? fmaf(x[i + 1] - m, f, -kSpare) : fmaf(x[i + 1], f, -mf));
            const uint32_t w = pack2<BF>(w0, w1);
            p[i / 8][i % 8 / 2] = w;
            if constexpr (EXACT) i % 4 ? b += w0 + w1 : a += w0 + w1;
            else i % 4 ? b = add2<BF>(w, b) : a = add2<BF>(w, a);
        }
        sum = a + b;
        return !(sum < kMost);
    }

    // Keys of a block of 32: their weights, with grow where a lane needs it.
    template <bool BIASED, bool EXACT, int DB>
    __device__ __forceinline__ void take(const f32x16& x, float f, u32x4 (&p)[2], f32x16 (&o)[DB]) {
        float sum;
        const bool mine = weigh<BIASED, EXACT>(x, f, p, sum);
        if (__any(mine)) grow<BIASED, EXACT, DB>(mine, x, f, p, sum, o);
        l += sum;
    }

    // The same with the maximum taken first, and what was summed so far rescaled,
    // in the lanes of such rows: no row's result depends on others.
    template <bool BIASED, bool EXACT, int DB>
    __device__ __forceinline__ void grow(bool mine, const f32x16& x, float f, u32x4 (&p)[2], float& sum,
                                         f32x16 (&o)[DB]) {
        const auto both = __builtin_amdgcn_permlane32_swap((uint32_t)mine, (uint32_t)mine, false, false);
        mine = (both[0] | both[1]) != 0;
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
        const float old = m;
        top = half_max(top);
        m = mine ? fmaxf(m, top) : m;
        float a = __builtin_amdgcn_exp2f((old - m) * f);
        if constexpr (!BIASED) {   // exactly what the exponents change by
            const float mf1 = mine ? m * f + kSpare : mf;
            a = __builtin_amdgcn_exp2f(mf - mf1);
            mf = mf1;
        }
        asm volatile("" : "+v"(a));   // keeps the products below behind the branch
        l *= a;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] *= a;
        weigh<BIASED, EXACT>(x, f, p, sum);
    }
};

// Whether new token t sees key j of its sequence.
__device__ __forceinline__ bool cached_sees(const AttnParams& p, const SeqLens& len, int b, int t, int j) {
    if (j < len.old) return true;
    const int u = j - len.old;
    return p.tree ? (p.tree[b * (int64_t)p.Sq + t] >> (u & 63) & 1) != 0 : u <= t;
}

// How the B * splits parts of a head are shared out: every part takes `each` units of
// one sequence's keys, so that long sequences have more of them and none is waited
// for.  `each` is as small as the parts allow: with ceil(all / parts) one sequence
// or another may need a part more than there is, with ceil(all / (parts - B)) none
// does.  A lane holds the parts of `per` sequences (one, up to 64 sequences).
// Measured against as many parts for each (24 heads of 128): one sequence of 16000 and
// seven of 1000 tokens 27.7 us instead of 33.0 for a token each, 31.1 instead of 67.1
// for 16; eight of 3000 the same.
struct Shares {
    int each, per;
    int before, mine;   // parts of the sequences before the lane's, and of its own

    __device__ __forceinline__ static int units(const AttnParams& p, int b) {
        return (seq_lens(p, b).k + (1 << p.unit_bits) - 1) >> p.unit_bits;
    }
    __device__ __forceinline__ int parts(const AttnParams& p, int b) const { return (units(p, b) + each - 1) / each; }

    __device__ __forceinline__ Shares(const AttnParams& p, int lane) {
        const int all = p.B * p.splits;
        if (p.B == 1) {
            each = max(1, (units(p, 0) + all - 1) / all);
            per = before = mine = 0;   // not used
            return;
        }
        per = (p.B + 63) / 64;
        int sum = 0, most = 0;
        for (int b = lane * per; b < min(p.B, lane * per + per); ++b) {
            const int u = units(p, b);
            sum += u;
            most = max(most, u);
        }
        sum = __builtin_amdgcn_readlane(wave_scan(sum), 63);
        each = max(1, (sum + all - 1) / all);
        if (p.splits == 1 || all > kMostSplits) {   // no sequence has more than kMostSplits
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o, 64));
            most = __builtin_amdgcn_readfirstlane(most);
            each = max(each, p.splits == 1 ? most : (most + kMostSplits - 1) / kMostSplits);
        }
        for (;;) {
            mine = 0;
            for (int b = lane * per; b < min(p.B, lane * per + per); ++b) mine += parts(p, b);
            before = wave_scan(mine);
            const bool fits = __builtin_amdgcn_readlane(before, 63) <= all;
            before -= mine;
            if (fits) break;   // the second time at the latest
            each = max(each + 1, (sum + all - p.B - 1) / (all - p.B));
        }
    }
    // The sequence of a part, and which of its parts it is; false: the part has no
    // keys.  Of a single sequence every part is written, with keys or without.
    __device__ __forceinline__ bool find(const AttnParams& p, int part, int& b, int& split) const {
        b = 0, split = part;
        if (p.B == 1) return true;
        const uint64_t owner = __ballot(part >= before && part < before + mine);
        if (owner == 0) return false;
        const int l = __builtin_ctzll(owner);
        split = part - __builtin_amdgcn_readlane(before, l);
        for (b = l * per;; ++b) {
            const int n = parts(p, b);
            if (split < n) return true;
            split -= n;
        }
    }
    // One wave of the launch leaves every sequence's first part and their number for
    // the launch that joins them.
    __device__ __forceinline__ void leave(const AttnParams& p, int lane) const {
        int part = before;
        for (int b = lane * per; b < min(p.B, lane * per + per); ++b) {
            const int n = parts(p, b);
            p.shares[2 * b] = part, p.shares[2 * b + 1] = n;
            part += n;
        }
    }
};

// Keeps the scores of 32 keys from j on (those of a lane at 8 (i / 4) + 4 h).
__device__ __forceinline__ void keep_scores(float* row, int j, int h, float f, const f32x16& x) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(row + j + 8 * i + 4 * h) =
            f32x4{x[4 * i] * f, x[4 * i + 1] * f, x[4 * i + 2] * f, x[4 * i + 3] * f};
}

}  // namespace sltx
