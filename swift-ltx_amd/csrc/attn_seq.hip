// attn_seq.hip -- launches attention of many query rows (attn_seq_kernel.hpp), and
// its kernels for head dims up to 64.
#include "attn_seq_kernel.hpp"

namespace sltx {

// Blocks of 64 rows where blocks of 128 would leave CUs without one; under a causal
// mask or documents, whose blocks differ in length, up to three for each CU.
// Measured (us, blocks of 64 / of 128 rows): 64 heads of 128 rows 5.7 / 6.3; causal,
// 24 heads of 128 columns: 750 rows 19.2 / 23.7, 1500 rows (288 blocks) 32.7 / 41.6;
// causal, 32 heads of 64: 2048 rows (512 blocks) 32.6 / 38.4; but 4096 rows of 32
// heads of 128 (1024 blocks) 188 / 152, and not causal, 2048 rows of 24 heads (384
// blocks) 84 / 71.  A cache's parts, whose ranges of keys fill the GPU, where half
// of a block of 128 rows would have none.
bool attn_seq_halves(const AttnParams& p) {
    const int64_t heads = (int64_t)p.B * p.heads, rows = (int64_t)p.Sq * p.pack;
    if (p.part_o) return rows <= kSeqTileRows / 2;
    return heads * ((rows + kSeqTileRows - 1) / kSeqTileRows) < (p.causal || p.q_docs ? 3 : 1) * kCUs;
}

hipError_t launch_attn_seq(AttnParams p, hipStream_t st) {
    p.halves = attn_seq_halves(p);
    const int rows = p.halves ? kSeqTileRows / 2 : kSeqTileRows;
    p.tiles = (int)(((int64_t)p.Sq * p.pack + rows - 1) / rows);
    const int64_t all = (int64_t)p.B * p.heads * p.splits, total = all * p.tiles;
    if (total == 0) return hipSuccess;
    if (total > 0x7fffff00 / 256) return hipErrorInvalidValue;
    p.by_xcd = all % 8 == 0;
    p.long_first = p.causal || p.q_docs;
    const dim3 g((unsigned)total);
    return p.D > 64 ? launch_attn_seq_d128(p, g, st) : launch_dim<64>(p, g, st);
}

}  // namespace sltx
