// attn_seq_d128.hip -- the kernels of attn_seq_kernel.hpp for head dims of 65 to 128.
#include "attn_seq_kernel.hpp"

namespace sltx {

hipError_t launch_attn_seq_d128(const AttnParams& p, dim3 g, hipStream_t st) { return launch_dim<128>(p, g, st); }

}  // namespace sltx
