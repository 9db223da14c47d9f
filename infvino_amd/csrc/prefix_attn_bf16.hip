// The bf16 kernels of attention with shared first tokens.
#include "prefix_attn.hpp"

namespace ivh {

void launch_prefix_bf16(const PrefixParams & p, hipStream_t s) { launch_prefix_type<kSeqBF16>(p, s); }

}  // namespace ivh
