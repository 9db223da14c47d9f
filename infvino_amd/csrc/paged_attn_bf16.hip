// The paged attention's bf16 kernels.
#include "paged_attn.hpp"

namespace ivh {

void launch_paged_bf16(const PagedParams & p, hipStream_t s) { launch_paged_type<kSeqBF16>(p, s); }

}  // namespace ivh
