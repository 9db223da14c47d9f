// The split of attention with shared first tokens, and its fp16 kernels (prefix_attn.hpp; the bf16 ones are
// built beside them).
#include "prefix_attn.hpp"

namespace ivh {

size_t prefix_split(PrefixParams & p, int max_new, int max_len, int max_shared)
{
  const CacheParams & c = p.own.c;
  p.first = p.own;
  p.own.lead = 0;
  if (p.own.groups > 0) {
    p.first.c.batch = p.own.groups;
    paged_split(p.first, (c.tokens + p.own.groups - 1) / p.own.groups, max_shared);
    p.own.lead = p.first.parts;
    p.first.c.batch = c.batch;
  }
  paged_split(p.own, max_new, std::max(1, max_len - (p.own.groups > 0 ? max_shared : 0)));
  p.own.all_parts = p.first.all_parts = p.own.lead + p.own.parts;
  return (size_t)p.own.all_parts * c.tokens * p.own.heads * (c.dim + 2) * sizeof(float);
}

void launch_prefix_attention(const PrefixParams & p, hipStream_t s)
{
  if (p.own.c.type == kSeqF16) launch_prefix_type<kSeqF16>(p, s);
  else launch_prefix_bf16(p, s);
}

}  // namespace ivh
