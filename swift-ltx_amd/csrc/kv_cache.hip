// kv_cache.hip -- what keeps a key/value cache: appending rotated keys and
// values, accepting drafted tokens, evicting by accumulated attention weight.
// All of them move bytes: nothing here does arithmetic that counts.
#include "attn_launch.hpp"
#include "q4_common.hpp"

namespace sltx {

// ---- append ----
// A block takes one token: its angles once (in 64 bits: position times
// frequency loses whole turns in 32 at far positions), then all its heads' q, k
// and v, 8 values a thread.  Rotated pairs are (i, i + pairs), or (2i, 2i + 1)
// interleaved; values past 2 pairs pass through.
template <bool BF>
__device__ __forceinline__ float widen(uint32_t x) {
    return BF ? bf2f((uint16_t)x) : h2f((uint16_t)x);
}
template <bool BF>
__device__ __forceinline__ uint32_t narrow(float x) {
    return BF ? f2bf(x) : f2h(x);
}

constexpr int kMaxPairs = 64;

template <bool BF>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendParams p) {
    __shared__ float cs[kMaxPairs], sn[kMaxPairs];
    const int t = blockIdx.x % p.T, b = blockIdx.x / p.T;
    const CacheParams& c = p.c;
    const int64_t at = (int64_t)c.next[b] + (p.depth ? p.depth[(int64_t)b * p.T + t] : t);
    const int64_t slot = (int64_t)c.length[b] + t;
    if (threadIdx.x < p.pairs) {
        const double turns = (double)at * (double)p.inv_freq[threadIdx.x] * 0.15915494309189535;
        const float r = (float)(turns - rint(turns));   // of a turn, -0.5 to 0.5
        sincospif(2.0f * r, &sn[threadIdx.x], &cs[threadIdx.x]);
    }
    __syncthreads();
    const bool fits = slot >= 0 && slot < c.capacity;   // tokens past the capacity are dropped
    const int chunks = c.D / 8, qn = p.Hq * chunks, kn = c.heads * chunks;
    const int64_t lb = (int64_t)p.layer * c.B + b;
    for (int e = threadIdx.x; e < qn + 2 * kn; e += 256) {
        const uint16_t* src;
        uint16_t* dst;
        int col;
        bool turn = true;
        if (e < qn) {
            const int head = e / chunks;
            col = e % chunks * 8;
            src = p.q + b * p.qs.b + t * p.qs.r + head * p.qs.h;
            dst = p.q_out + (((int64_t)b * p.T + t) * p.Hq + head) * c.D;
        } else {
            if (!fits) break;
            const int i = e - qn, v = i >= kn, head = (v ? i - kn : i) / chunks;
            col = (v ? i - kn : i) % chunks * 8;
            src = v ? p.v + b * p.vs.b + t * p.vs.r + head * p.vs.h : p.k + b * p.ks.b + t * p.ks.r + head * p.ks.h;
            dst = (v ? c.v : c.k) + ((lb * c.heads + head) * c.capacity + slot) * c.D;
            turn = !v;
        }
        u32x4 x = *reinterpret_cast<const u32x4*>(src + col);
        if (turn && col < 2 * p.pairs) {
            float y[8], z[8];   // the values and their pairs' others
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = widen<BF>(x[i / 2] >> (i % 2 * 16) & 0xffffu);
            if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = y[i ^ 1];
            } else if (p.pairs % 8 == 0) {
                const u32x4 o = *reinterpret_cast<const u32x4*>(src + (col < p.pairs ? col + p.pairs : col - p.pairs));
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = widen<BF>(o[i / 2] >> (i % 2 * 16) & 0xffffu);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int a = col + i;
                    z[i] = a < 2 * p.pairs ? widen<BF>(src[a < p.pairs ? a + p.pairs : a - p.pairs]) : 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int a = col + i;
                if (a < 2 * p.pairs) {
                    const int pair = p.interleaved ? a / 2 : a < p.pairs ? a : a - p.pairs;
                    const bool first = p.interleaved ? a % 2 == 0 : a < p.pairs;
                    y[i] = y[i] * cs[pair] + (first ? -z[i] : z[i]) * sn[pair];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = narrow<BF>(y[2 * i]) | narrow<BF>(y[2 * i + 1]) << 16;
        }
        *reinterpret_cast<u32x4*>(dst + col) = x;
    }
    if (c.weight && fits && threadIdx.x < 64)
        for (int head = threadIdx.x; head < c.heads; head += 64) {
            const int64_t i = (lb * c.heads + head) * c.capacity + slot;
            c.weight[i] = 0.0f;
            c.position[i] = (int32_t)at;
        }
}

// The same where all of head_dim is rotated in pairs (i, i + D / 2), the usual
// case: a thread takes the 8 pairs of two pieces, so that each piece is read
// once, and its loads (two items' at a time) are under way before the angles are
// there.  750 tokens of 32 + 8 + 8 heads of 128: 5.4 us, 3.4 TB/s (9.2 us in the kernel
// above); 8 tokens of 24 + 8 + 8 heads 3.4 us, a launch and two trips to memory.
template <bool BF>
__global__ __launch_bounds__(256) void kv_append_paired_kernel(AppendParams p) {
    __shared__ __attribute__((aligned(16))) float cs[kMaxPairs], sn[kMaxPairs];
    constexpr int AHEAD = 2;
    const int t = blockIdx.x % p.T, b = blockIdx.x / p.T;
    const CacheParams& c = p.c;
    const int half = c.D / 16, qn = p.Hq * half, kn = c.heads * half, items = qn + 2 * kn;
    const int64_t lb = (int64_t)p.layer * c.B + b;
    u32x4 lo[AHEAD], hi[AHEAD];
    auto source = [&](int e) -> const uint16_t* {
        if (e < qn) return p.q + b * p.qs.b + t * p.qs.r + (e / half) * p.qs.h + e % half * 8;
        const int i = e - qn;
        if (i < kn) return p.k + b * p.ks.b + t * p.ks.r + (i / half) * p.ks.h + i % half * 8;
        return p.v + b * p.vs.b + t * p.vs.r + ((i - kn) / half) * p.vs.h + (i - kn) % half * 8;
    };
    auto load = [&](int e0) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int e = e0 + u * 256;
            if (e < items) {
                const uint16_t* s = source(e);
                lo[u] = *reinterpret_cast<const u32x4*>(s);
                hi[u] = *reinterpret_cast<const u32x4*>(s + c.D / 2);
            }
        }
    };
    load(threadIdx.x);
    const int64_t at = (int64_t)c.next[b] + (p.depth ? p.depth[(int64_t)b * p.T + t] : t);
    const int64_t slot = (int64_t)c.length[b] + t;
    const bool fits = slot >= 0 && slot < c.capacity;   // tokens past the capacity are dropped
    if (threadIdx.x < p.pairs) {
        const double turns = (double)at * (double)p.inv_freq[threadIdx.x] * 0.15915494309189535;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn[threadIdx.x], &cs[threadIdx.x]);
    }
    __syncthreads();
    for (int e0 = threadIdx.x; e0 < items; e0 += AHEAD * 256) {
        if (e0 != (int)threadIdx.x) load(e0);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int e = e0 + u * 256;
            if (e >= items) break;
            const int i = e < qn ? e : e - qn < kn ? e - qn : e - qn - kn, head = i / half, col = i % half * 8;
            uint16_t* dst = e < qn ? p.q_out + (((int64_t)b * p.T + t) * p.Hq + head) * c.D
                                   : (e - qn < kn ? c.k : c.v) + ((lb * c.heads + head) * c.capacity + slot) * c.D;
            u32x4 x = lo[u], y = hi[u];
            if (e < qn + kn) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t rx = 0, ry = 0;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const float f = widen<BF>(x[w] >> (16 * s) & 0xffffu), g = widen<BF>(y[w] >> (16 * s) & 0xffffu);
                        const float co = cs[col + 2 * w + s], si = sn[col + 2 * w + s];
                        rx |= narrow<BF>(f * co - g * si) << (16 * s);
                        ry |= narrow<BF>(g * co + f * si) << (16 * s);
                    }
                    x[w] = rx;
                    y[w] = ry;
                }
            }
            if (e < qn || fits) {
                *reinterpret_cast<u32x4*>(dst + col) = x;
                *reinterpret_cast<u32x4*>(dst + col + c.D / 2) = y;
            }
        }
    }
    if (c.weight && fits)
        for (int head = threadIdx.x; head < c.heads; head += 256) {
            const int64_t i = (lb * c.heads + head) * c.capacity + slot;
            c.weight[i] = 0.0f;
            c.position[i] = (int32_t)at;
        }
}

hipError_t launch_kv_append(const AppendParams& p, hipStream_t st) {
    const int64_t blocks = (int64_t)p.c.B * p.T;
    if (blocks == 0) return hipSuccess;
    if (blocks > 0x7fffff00 / 256) return hipErrorInvalidValue;
    const dim3 g((unsigned)blocks), t(256);
    if (2 * p.pairs == p.c.D && p.pairs % 8 == 0 && !p.interleaved) {
        if (p.bf16) hipLaunchKernelGGL(kv_append_paired_kernel<true>, g, t, 0, st, p);
        else hipLaunchKernelGGL(kv_append_paired_kernel<false>, g, t, 0, st, p);
    } else if (p.bf16) hipLaunchKernelGGL(kv_append_kernel<true>, g, t, 0, st, p);
    else hipLaunchKernelGGL(kv_append_kernel<false>, g, t, 0, st, p);
    return hipGetLastError();
}

// ---- accept ----
constexpr int kMaxPath = 64;

// The tokens of sequence b's path that are accepted: its first count[b], as far
// as they name drafted tokens that are in the cache, and have a slot themselves (a path
// that names a token twice may be longer than the room is).  One wave; all lanes.
__device__ __forceinline__ int accepted(const CacheParams& c, int b, int drafted, const int32_t* path,
                                        int path_len, const int32_t* count, int* node) {
    const int lane = threadIdx.x & 63;
    const int most = count ? min(max(count[b], 0), path_len) : path_len;
    const int length = c.length[b];
    *node = lane < path_len ? path ? path[(int64_t)b * path_len + lane] : lane : -1;
    const bool good = lane < most && *node >= 0 && *node < drafted && length >= 0 &&
                      (int64_t)length + max(*node, lane) < c.capacity;
    const uint64_t bad = ~__ballot(good);
    return bad ? __builtin_ctzll(bad) : 64;
}

// One block for each layer, sequence and head: the accepted rows are all read
// before the first is written, so any order of the path is safe.  5 rows of K and V in
// 28 layers and 8 heads of 128: 3.5 us, a launch and three trips to memory; up to 9
// rows in 16 layers, 16 sequences and 8 heads of 64 (9 MB read and written) 6.8 us.
__global__ __launch_bounds__(256) void kv_accept_kernel(CacheParams c, int drafted, const int32_t* path,
                                                        int path_len, const int32_t* count) {
    __shared__ int nodes[kMaxPath];
    const int lbh = blockIdx.x, b = lbh / c.heads % c.B;
    int node;
    const int n = accepted(c, b, drafted, path, path_len, count, &node);
    if (threadIdx.x < 64) nodes[threadIdx.x] = node;
    __syncthreads();
    const int chunks = c.D / 8;
    const int64_t row0 = (int64_t)lbh * c.capacity + c.length[b];
    constexpr int MOST = kMaxPath * 16 / 256;   // 16-byte pieces of a thread, head_dim 128
    u32x4 kr[MOST], vr[MOST];
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        const int e = i * 256 + threadIdx.x, r = e / chunks;
        if (r < n && nodes[r] != r) {
            const int64_t s = (row0 + nodes[r]) * c.D + e % chunks * 8;
            kr[i] = *reinterpret_cast<const u32x4*>(c.k + s);
            vr[i] = *reinterpret_cast<const u32x4*>(c.v + s);
        }
    }
    float w = 0.0f;
    int32_t at = 0;
    const int r1 = threadIdx.x;
    if (c.weight && r1 < n) w = c.weight[row0 + nodes[r1]], at = c.position[row0 + nodes[r1]];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        const int e = i * 256 + threadIdx.x, r = e / chunks;
        if (r < n && nodes[r] != r) {
            const int64_t d = (row0 + r) * c.D + e % chunks * 8;
            *reinterpret_cast<u32x4*>(c.k + d) = kr[i];
            *reinterpret_cast<u32x4*>(c.v + d) = vr[i];
        }
    }
    if (c.weight && r1 < n) c.weight[row0 + r1] = w, c.position[row0 + r1] = at;
}

// Lengthens the sequences; a launch of its own, after every block has read the
// old lengths: 1.5 to 2.3 us.
__global__ __launch_bounds__(64) void kv_advance_kernel(CacheParams c, int drafted, const int32_t* path,
                                                        int path_len, const int32_t* count) {
    const int b = blockIdx.x;
    int node;
    const int n = accepted(c, b, drafted, path, path_len, count, &node);
    if (threadIdx.x == 0) {
        c.length[b] += n;
        c.next[b] += n;
    }
}
__global__ __launch_bounds__(256) void kv_advance_chain_kernel(CacheParams c, int drafted, const int32_t* count) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= c.B) return;
    const int length = c.length[b];
    int n = count ? min(max(count[b], 0), drafted) : drafted;
    n = max(0, min(n, c.capacity - length));
    c.length[b] = length + n;
    c.next[b] += n;
}

hipError_t launch_kv_accept(const CacheParams& c, int drafted, const int32_t* path, int path_len,
                            const int32_t* count, hipStream_t st) {
    if (c.B == 0) return hipSuccess;
    if (!path) {
        hipLaunchKernelGGL(kv_advance_chain_kernel, dim3((c.B + 255) / 256), dim3(256), 0, st, c, drafted, count);
        return hipGetLastError();
    }
    const int64_t blocks = (int64_t)c.layers * c.B * c.heads;
    if (blocks > 0x7fffff00 / 256) return hipErrorInvalidValue;
    hipLaunchKernelGGL(kv_accept_kernel, dim3((unsigned)blocks), dim3(256), 0, st, c, drafted, path, path_len, count);
    hipLaunchKernelGGL(kv_advance_kernel, dim3(c.B), dim3(64), 0, st, c, drafted, path, path_len, count);
    return hipGetLastError();
}

// ---- evict ----
// Which entries stay is a selection of the `budget` largest keys: the weight as
// an unsigned number of the same order (NaN lowest, -0 as 0), the largest of all
// for protected positions; of equal keys the lowest slots.  A radix select over
// four digits of 8 bits, then one pass in slot order for the holes (slots below
// the budget whose entry goes) and the comers (entries from slots above it that
// stay), which a second launch moves into them.  A chain of short steps: 1792 times
// 1025 entries 10.0 us, 128 times 6001 9.4; to start the digits at the first bit in
// which the keys differ (fewer of them, fewer equal ones) gave nothing.
struct EvictParams {
    CacheParams c;
    int budget, sinks, recent;
    int32_t *moves, *holes, *comers;   // [layers * B * heads], [...][most] twice
    int most;
};

__device__ __forceinline__ uint32_t evict_key(const EvictParams& p, int32_t at, float w, int64_t after) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    const uint32_t k = w != w ? 0 : u >> 31 ? ~u : u | 0x80000000u;
    return at < p.sinks || (int64_t)at >= after - p.recent ? 0xffffffffu : k;
}

// A block for each layer, sequence and head.  Wave w takes the slots from w * 64 R
// on, R at a time in each lane; their keys are read once and kept in registers
// where R covers them (up to 16384 entries: R = 16 with 16 waves), else (R = 0)
// read again in each of the seven passes.  Measured, the whole call with steps of a
// digit 0.2 us longer than now: 128 times 6001 entries 29.2 us with R = 8, 33.9 with
// R = 0; 1792 times 1025 entries 22.1 with 4 waves and R = 8, 44.2 with 16 waves, 33.9
// with those and R = 0.
template <int WAVES, int R>
__global__ __launch_bounds__(WAVES * 64) void kv_evict_select_kernel(EvictParams p) {
    __shared__ int hist[2][256];   // one is cleared while the other is filled
    __shared__ int sums[WAVES][2];
    __shared__ int found[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lbh = blockIdx.x, b = lbh / p.c.heads % p.c.B;
    const int n = min(p.c.length[b], p.c.capacity);
    if (n <= p.budget) {
        if (tid == 0) p.moves[lbh] = 0;
        return;
    }
    const int64_t after = p.c.next[b], base = (int64_t)lbh * p.c.capacity;
    const int run = (n + WAVES * 64 - 1) / (WAVES * 64);   // 64 slots each
    const int s0 = wave * run * 64 + lane;                 // this lane's are s0 + 64 i
    const int mine = min(run, max(0, (n - s0 + 63) / 64));
    uint32_t held[R > 0 ? R : 1];
    if constexpr (R > 0) {   // all loads on their way before the first key
        int32_t at[R];
        float w[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t e = base + min(s0 + i * 64, n - 1);
            at[i] = p.c.position[e];
            w[i] = p.c.weight[e];
        }
#pragma unroll
        for (int i = 0; i < R; ++i) held[i] = i < mine ? evict_key(p, at[i], w[i], after) : 0;
    }
    // f(slot, key, whether it is one of this lane's), by every lane as often
    auto each = [&](auto&& f) {
        if constexpr (R > 0) {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i < run) f(s0 + i * 64, held[i], i < mine);
        } else {
            for (int i = 0; i < run; ++i) {
                const int64_t e = base + min(s0 + i * 64, n - 1);
                f(s0 + i * 64, i < mine ? evict_key(p, p.c.position[e], p.c.weight[e], after) : 0, i < mine);
            }
        }
    };
    uint32_t prefix = 0;
    int want = p.budget;   // of the keys that start with the prefix
    bool exact = false;    // every key that starts with the prefix stays
    if (tid < 256) hist[24 >> 3 & 1][tid] = 0;
    __syncthreads();
    for (int shift = 24; shift >= 0 && !exact; shift -= 8) {
        int *h = hist[shift >> 3 & 1], *other = hist[~shift >> 3 & 1];
        each([&](int, uint32_t k, bool in) {
            if (in && (shift == 24 || k >> (shift + 8) == prefix >> (shift + 8))) atomicAdd(&h[k >> shift & 255], 1);
        });
        if (tid < 256) other[tid] = 0;
        __syncthreads();
        if (wave == 0) {   // the digit in which the count from the top reaches `want`
            int c[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += c[i] = h[255 - (lane * 4 + i)];
            int before = wave_scan(sum) - sum;
            if (before < want && before + sum >= want) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (before < want && before + c[i] >= want) {
                        found[0] = 255 - (lane * 4 + i);
                        found[1] = want - before;
                        found[2] = before + c[i] == want;
                        break;
                    }
                    before += c[i];
                }
            }
        }
        __syncthreads();
        prefix |= (uint32_t)found[0] << shift;
        want = found[1];
        exact = found[2] != 0;
    }
    // `prefix` is the smallest key that may stay; `want` of the entries with just
    // it do, the lowest slots, or (exact) every entry from it on.
    const uint64_t below = (1ull << lane) - 1;
    int tie0 = 0;
    if (!exact) {
        int ties = 0;
        each([&](int, uint32_t k, bool in) { ties += __popcll(__ballot(in && k == prefix)); });
        if (lane == 0) sums[wave][0] = ties;
        __syncthreads();
        for (int w = 0; w < wave; ++w) tie0 += sums[w][0];
        __syncthreads();
    }
    for (int pass = 0; pass < 2; ++pass) {   // count, then write
        int tie = tie0, hole = 0, comer = 0;
        if (pass == 1)
            for (int w = 0; w < wave; ++w) hole += sums[w][0], comer += sums[w][1];
        each([&](int slot, uint32_t k, bool in) {
            bool keep = in && k >= prefix;
            if (!exact) {
                const uint64_t t = __ballot(in && k == prefix);
                keep = keep && (k > prefix || tie + __popcll(t & below) < want);
                tie += __popcll(t);
            }
            const bool is_hole = in && slot < p.budget && !keep, is_comer = keep && slot >= p.budget;
            const uint64_t hm = __ballot(is_hole), cm = __ballot(is_comer);
            if (pass == 1) {
                if (is_hole) p.holes[(int64_t)lbh * p.most + hole + __popcll(hm & below)] = slot;
                if (is_comer) p.comers[(int64_t)lbh * p.most + comer + __popcll(cm & below)] = slot;
            }
            hole += __popcll(hm);
            comer += __popcll(cm);
        });
        if (pass == 0) {
            if (lane == 0) sums[wave][0] = hole, sums[wave][1] = comer;
            __syncthreads();
        } else if (wave == WAVES - 1 && lane == 0) {
            p.moves[lbh] = hole;
        }
    }
}

// Moves the comers into the holes: disjoint slots, in any order.  A row's pieces
// go to neighbouring lanes.  1024 entries of 128 heads of 64, 85% of them from above
// the budget: 13.9 us for 57 MB read and written, 4.1 TB/s; one entry of 1792: 4.4 us.
__global__ __launch_bounds__(256) void kv_evict_move_kernel(EvictParams p) {
    const int lbh = blockIdx.y, b = lbh / p.c.heads % p.c.B;
    const uint32_t chunks = p.c.D / 8;
    const int moves = p.moves[lbh];
    const int32_t *holes = p.holes + (int64_t)lbh * p.most, *comers = p.comers + (int64_t)lbh * p.most;
    const int64_t base = (int64_t)lbh * p.c.capacity;
    for (uint32_t e = blockIdx.x * 256 + threadIdx.x; e < (uint32_t)moves * chunks; e += gridDim.x * 256) {
        const uint32_t m = e / chunks, piece = e % chunks;   // up to 2^27 * 16 pieces
        const int64_t d = base + holes[m], s = base + comers[m];
        const u32x4 k = *reinterpret_cast<const u32x4*>(p.c.k + s * p.c.D + piece * 8);
        const u32x4 v = *reinterpret_cast<const u32x4*>(p.c.v + s * p.c.D + piece * 8);
        *reinterpret_cast<u32x4*>(p.c.k + d * p.c.D + piece * 8) = k;
        *reinterpret_cast<u32x4*>(p.c.v + d * p.c.D + piece * 8) = v;
        if (piece == 0) {
            p.c.weight[d] = p.c.weight[s];
            p.c.position[d] = p.c.position[s];
        }
    }
    // no block of this launch reads the lengths
    if (blockIdx.x == 0 && threadIdx.x == 0 && lbh / p.c.heads / p.c.B == 0 && lbh % p.c.heads == 0)
        p.c.length[b] = min(p.c.length[b], p.budget);
}

size_t kv_evict_workspace_bytes(const CacheParams& c, int budget) {
    const size_t lbh = (size_t)c.layers * c.B * c.heads;
    return lbh * (1 + 2 * (size_t)std::min(budget, c.capacity - budget)) * sizeof(int32_t);
}

hipError_t launch_kv_evict(const CacheParams& c, int budget, int sinks, int recent, void* ws, hipStream_t st) {
    const int64_t lbh = (int64_t)c.layers * c.B * c.heads;
    if (lbh == 0 || budget == c.capacity) return hipSuccess;
    if (lbh > 65535) return hipErrorInvalidValue;
    EvictParams p = {c, budget, sinks, recent, nullptr, nullptr, nullptr, std::min(budget, c.capacity - budget)};
    p.moves = static_cast<int32_t*>(ws);
    p.holes = p.moves + lbh;
    p.comers = p.holes + lbh * p.most;
    // By the capacity: the lengths are on the device.
    const dim3 g((unsigned)lbh);
    if (c.capacity <= 256 * 8) hipLaunchKernelGGL((kv_evict_select_kernel<4, 8>), g, dim3(256), 0, st, p);
    else if (c.capacity <= 1024 * 8) hipLaunchKernelGGL((kv_evict_select_kernel<16, 8>), g, dim3(1024), 0, st, p);
    else if (c.capacity <= 1024 * 16) hipLaunchKernelGGL((kv_evict_select_kernel<16, 16>), g, dim3(1024), 0, st, p);
    else hipLaunchKernelGGL((kv_evict_select_kernel<16, 0>), g, dim3(1024), 0, st, p);
    const int64_t pieces = (int64_t)p.most * (c.D / 8);
    const unsigned x = (unsigned)std::max<int64_t>(1, std::min<int64_t>((pieces + 255) / 256, (2048 + lbh - 1) / lbh));
    hipLaunchKernelGGL(kv_evict_move_kernel, dim3(x, (unsigned)lbh), dim3(256), 0, st, p);
    return hipGetLastError();
}

}  // namespace sltx
