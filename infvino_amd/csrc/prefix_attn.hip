// The split of attention with shared first tokens, and its fp16 kernels (prefix_attn.hpp; the bf16 ones are
// built beside them).
#include "prefix_attn.hpp"

namespace ivh {

namespace {
// Work-groups over shared keys: of 128 rows three a CU (256 of them in all: 376 us, 512: 218, 768: 194, 48 x 4 drafted tokens
// behind 32000); of 32 rows at least one a CU, beside those of own keys (256 to 320: 45 to 47 us, 512: 52, 128: 83, 64 sequences behind 8192)
constexpr long kSharedWgs = 768, kWideWgs = 256;
}  // namespace

size_t prefix_split(PrefixParams & p, int max_new, int max_len, int max_shared)
{
  const CacheParams & c = p.own.c;
  p.first = p.own;
  p.own.lead = 0;
  if (p.own.groups > 0) {
    p.first.c.batch = p.own.groups;
    const long tokens = (c.tokens + p.own.groups - 1) / p.own.groups, rows = tokens * p.own.group;
    // both sides of each bound are in prefix_attn.hpp
    p.many = c.dim <= 64 && rows >= 512 && max_shared >= 16384;
    p.wide = !p.many && (c.dim <= 64 ? rows > 16 : c.dim <= 128 && rows >= 96);
    if (p.many || p.wide) {
      PagedParams & f = p.first;
      const long wgs0 = (long)p.own.groups * c.heads, steps = std::max(1, max_shared / 64), tile = p.many ? 128 : 32;
      f.row_slots = (int)std::min<long>({(rows + tile - 1) / tile, 1024, std::max<long>(1, (1L << 21) / wgs0)});
      const long wgs = wgs0 * f.row_slots, want = p.many ? std::max<long>(1, kSharedWgs / wgs) : (kWideWgs + wgs - 1) / wgs;
      f.parts = (int)std::min<long>({want, steps, 256, std::max<long>(1, (1L << 22) / wgs)});
      f.part_steps = (int)((steps + f.parts - 1) / f.parts);
      f.parts = (int)((steps + f.part_steps - 1) / f.part_steps);
    } else {
      paged_split(p.first, (int)tokens, max_shared);
    }
    p.own.lead = p.first.parts;
    p.first.c.batch = c.batch;
  }
  paged_split(p.own, max_new, std::max(1, max_len - (p.own.groups > 0 ? max_shared : 0)));
  p.both = p.own.lead > 0 && !p.many && (p.wide || (p.first.row_tiles == p.own.row_tiles && p.first.row_waves == p.own.row_waves));
  if (p.both) {
    const long units = (long)p.own.groups * c.heads * p.first.parts;
    p.both = units * p.first.row_slots <= 1L << 22;  // of the 2^24 work-groups that a launch holds; wide ones are
    p.own.shared_wgs = (int)((units + kXcds - 1) / kXcds * kXcds * p.first.row_slots);
    p.own.shared_slots = p.first.row_slots;
    p.own.shared_steps = p.first.part_steps;
  }
  p.own.all_parts = p.first.all_parts = p.own.lead + p.own.parts;
  return (size_t)p.own.all_parts * c.tokens * p.own.heads * (c.dim + 2) * sizeof(float);
}

void launch_prefix_attention(const PrefixParams & p, hipStream_t s)
{
  if (p.own.c.type == kSeqF16) launch_prefix_type<kSeqF16>(p, s);
  else launch_prefix_bf16(p, s);
}

}  // namespace ivh
