// The paged attention's split and its fp16 kernels (paged_attn.hpp; the bf16 ones are built beside
// them).
#include "paged_attn.hpp"

namespace ivh {

size_t paged_split(PagedParams & p, int max_new, int max_len)
{
  const CacheParams & c = p.c;
  const long rows = (long)std::max(1, std::min(max_new, c.tokens)) * p.group;
  // Two row tiles a wave share its key and value fragments where registers allow it.  With more rows
  // waves take rows instead of keys, but not where work-groups of a row tile each fill two rounds of the
  // chip at most: there the keys are short of hands, and the second reader of a key finds it in L2 (24
  // sequences, 5 new tokens of 8 heads a key head, window 1024: 17.6 us, 20.8 with waves over rows; one sequence,
  // 32 new tokens, 5000 keys 17.6 and 21.1; 16 new tokens, 4096 keys, 64 channels 19.0 and 18.4).
  const int most = c.dim <= 64 ? 2 : 1;
  p.row_tiles = rows <= 16 ? 1 : most;
  const int per_wave = 16 * p.row_tiles;
  const bool few = (long)c.batch * c.heads * ((rows + per_wave - 1) / per_wave) <= 512;
  p.row_waves = rows <= per_wave || few ? 1 : rows <= 2 * per_wave ? 2 : 4;
  const int per_wg = per_wave * p.row_waves;
  p.row_slots = (int)std::min<long>({(rows + per_wg - 1) / per_wg, 1024, (1L << 23) / ((long)c.batch * c.heads)});
  // Keys: a work-group for each CU where there are keys enough (more parts cost more in joining
  // than they bring: 32 rows over 60000 keys 28 us with 256 work-groups, 36 with 1024).  With few rows none is
  // longer than 24 steps a wave, so that a ragged batch's long sequences do not outlast the others (64 of
  // 900 to 16001 keys 209 us, 218 unsplit; 64 of 8192 each pay for it, 191 us, 182 unsplit); with many the partial sums would
  // be too large for that.
  long len = std::min<long>(max_len, (long)c.width * c.page);
  if (p.window) len = std::min<long>(len, (long)p.window + p.sinks + max_new + 128);
  const long steps = (len + 63) / 64, waves = 4 / p.row_waves;
  const long wgs = (long)c.batch * c.heads * p.row_slots;
  const long balance = p.row_waves < 4 ? (steps + 24 * waves - 1) / (24 * waves) : 1;
  long want = std::max<long>((256 + wgs - 1) / wgs, balance);
  // Between one round of the chip and two, one if its waves have few steps, else two (12 sequences of 3000 keys
  // 21 us in one round, 25 in 1.1; 16 new tokens over 60000 keys 42 in two, 47 in one, 54 in 1.3).
  if (wgs * want > 256 && wgs * want < 512) {
    const long one = std::max<long>(1, 256 / wgs);
    want = steps <= 24 * waves * one ? one : (512 + wgs - 1) / wgs;
  }
  const long top = std::max<long>(1, (steps + waves - 1) / waves);
  // a launch holds fewer than 2^24 work-groups of 256 lanes
  p.parts = (int)std::min<long>({std::max<long>(want, 1), top, 256, std::max<long>(1, (1L << 23) / wgs)});
  // the join has up to a work-group for each row, of which a launch holds as many: more rows fill the chip
  if ((long)c.tokens * p.heads >= 1L << 24) p.parts = 1;
  p.part_steps = (int)((((steps + p.parts - 1) / p.parts) + waves - 1) / waves * waves);
  p.parts = (int)std::max<long>(1, (steps + p.part_steps - 1) / p.part_steps);
  if (p.parts == 1) return 0;
  return (size_t)p.parts * c.tokens * p.heads * (c.dim + 2) * sizeof(float);
}

long paged_wgs(const PagedParams & p, long seqs)
{
  return (seqs * p.c.heads * p.parts + kXcds - 1) / kXcds * kXcds * p.row_slots;
}

JoinSplit join_split(const PagedParams & p)
{
  // a lot for every two parts where lanes allow it, and where rows alone do not fill the chip many times over
  const long rows = (long)p.c.tokens * p.heads;
  const int lanes = p.c.dim / 4, lots = rows < 1L << 23 ? std::max(1, std::min(p.parts / 2, 256 / lanes)) : 1, per = 256 / (lanes * lots);
  return JoinSplit{lots, per, (rows + per - 1) / per};
}

void launch_paged_attention(const PagedParams & p, hipStream_t s)
{
  if (p.c.type == kSeqF16) launch_paged_type<kSeqF16>(p, s);
  else launch_paged_bf16(p, s);
}

}  // namespace ivh
