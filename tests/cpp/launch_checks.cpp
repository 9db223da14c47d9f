// Host-side check of how the sequence operators' calls are split, at the largest calls that the entry points accept and at
// random ones below: every launch has at least one and fewer than 2^24 work-groups of 256 lanes, joins cover every row, and
// workspaces are those of the parts.  No device is needed: a split is arithmetic.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <random>

#include "seq_ops.hpp"

static int fails = 0;
#define EXPECT(c)                                                                \
  do {                                                                           \
    if (!(c)) {                                                                  \
      std::fprintf(stderr, "line %d: %s (%s)\n", __LINE__, #c, what);            \
      ++fails;                                                                   \
    }                                                                            \
  } while (0)

static constexpr long kLaunch = 1L << 24;

static void join(const ivh::PagedParams & p, const char * what)
{
  const ivh::JoinSplit j = ivh::join_split(p);
  const long rows = (long)p.c.tokens * p.heads;
  EXPECT(j.lots >= 1 && j.per >= 1 && j.lots * j.per * (p.c.dim / 4) <= 256);
  EXPECT(j.wgs * j.per >= rows && (j.wgs - 1) * j.per < rows);
  EXPECT(ivh::kJoinWgs < kLaunch);
}

static void prefix(int batch, int groups, int tokens, int heads, int kv, int dim, int width, int max_new, int max_len, int max_shared)
{
  char what[200];
  std::snprintf(what, sizeof what, "prefix: batch %d groups %d tokens %d heads %d / %d dim %d width %d hints %d %d %d", batch, groups, tokens, heads, kv, dim,
                width, max_new, max_len, max_shared);
  ivh::PrefixParams p;
  ivh::CacheParams & c = p.own.c;
  c.heads = kv, c.dim = dim, c.page = 16, c.width = width, c.batch = batch, c.tokens = tokens;
  p.own.heads = heads, p.own.group = heads / kv, p.own.groups = groups;
  const size_t bytes = ivh::prefix_split(p, max_new, max_len, max_shared);
  EXPECT(bytes == (size_t)p.own.all_parts * tokens * heads * (dim + 2) * 4);
  const long own = ivh::paged_wgs(p.own, batch), shared = p.own.lead > 0 ? ivh::paged_wgs(p.first, groups) : 0;
  EXPECT(own >= 1 && own + (p.both ? p.own.shared_wgs : 0) < kLaunch);
  EXPECT(p.both ? p.own.shared_wgs >= 1 : shared < kLaunch);
  EXPECT((p.own.lead > 0) == (groups > 0));
  p.own.parts = p.own.all_parts;
  join(p.own, what);
}

static void paged(int batch, int tokens, int heads, int kv, int dim, int width, int max_new, int max_len)
{
  char what[200];
  std::snprintf(what, sizeof what, "paged: batch %d tokens %d heads %d / %d dim %d width %d hints %d %d", batch, tokens, heads, kv, dim, width, max_new, max_len);
  ivh::PagedParams p;
  ivh::CacheParams & c = p.c;
  c.heads = kv, c.dim = dim, c.page = 16, c.width = width, c.batch = batch, c.tokens = tokens;
  p.heads = heads, p.group = heads / kv;
  const size_t bytes = ivh::paged_split(p, max_new, max_len);
  EXPECT(bytes == (p.parts > 1 ? (size_t)p.parts * tokens * heads * (dim + 2) * 4 : 0));
  const long wgs = ivh::paged_wgs(p, batch);
  EXPECT(wgs >= 1 && wgs < kLaunch);
  if (p.parts > 1) join(p, what);
}

static void linear(int batch, int tokens, int heads, int key_heads, int key_dim, int dim, int max_new)
{
  char what[200];
  std::snprintf(what, sizeof what, "linear: batch %d tokens %d heads %d / %d dims %d %d max_new %d", batch, tokens, heads, key_heads, key_dim, dim, max_new);
  ivh::LinearParams p;
  p.heads = heads, p.group = heads / key_heads, p.key_dim = key_dim, p.dim = dim, p.batch = batch, p.tokens = tokens;
  const size_t bytes = ivh::linear_split(p, std::min(max_new ? max_new : tokens, tokens));
  const long wgs = ivh::linear_wgs(p);
  EXPECT(wgs >= 1 && wgs < kLaunch);
  EXPECT(bytes == 0 || (p.seg >= 64 && bytes == ((size_t)tokens / p.seg + batch) * heads * ((size_t)key_dim * dim + 2) * 4));
}

int main()
{
  const int most = 1 << 26;
  for (int dim = 16; dim <= 256; dim += 16)
    for (int width : {1, 8, 1 << 20, 1 << 26})
      for (int shared : {1, 100, 20000, 1 << 30})
        for (int heads : {1, 64, 4096}) {
          const int rows = most / heads, keys = width > (1 << 30) / 16 ? 1 << 30 : width * 16;
          for (int tokens : {1, 5, rows - 1, rows})
            for (int batch : {1, std::min(tokens, 1 << 20)})
              for (int kv : {1, heads}) {
                if ((int64_t)batch * kv > 1 << 22) continue;
                for (int groups : {0, 1, batch}) prefix(batch, groups, tokens, heads, kv, dim, width, 1, std::min(keys, 1 << 30), std::min(shared, keys));
                paged(batch, tokens, heads, kv, dim, width, 1, keys);
              }
        }
  for (int batch : {1, 1 << 10, 1 << 20})
    for (int heads : {1, 64, 4096})
      for (int tokens : {0, 1, 17, 1 << 20, most})
        for (int dim = 16; dim <= 256; dim += 48) {
          if ((int64_t)batch * heads > 1 << 20) continue;
          for (int key_heads : {1, heads})
            for (int max_new : {0, 1, 300, tokens}) linear(batch, tokens, heads, key_heads, dim, 272 - dim, max_new);
        }
  std::mt19937_64 rng(5);
  auto upto = [&](double hi) { return (int)std::exp(std::uniform_real_distribution<double>(0.0, std::log(hi + 0.99))(rng)); };
  for (int i = 0; i < 200000; ++i) {
    const int kv = upto(4096), group = upto(64), heads = kv * group, tokens = upto(std::max(1, most / heads)), dim = 16 * upto(16), width = upto(1 << 26);
    const int batch = upto(std::min(1 << 20, (1 << 22) / kv)), groups = i % 5 ? upto(std::min(1 << 20, (1 << 22) / kv)) : 0;
    if ((int64_t)tokens * heads > most) continue;
    prefix(batch, groups, tokens, heads, kv, dim, width, upto(tokens), upto(1 << 30), std::min<int64_t>(upto(1 << 30), (int64_t)width * 16));
    paged(batch, tokens, heads, kv, dim, width, upto(tokens), upto(1 << 30));
    const int lh = upto(4096);
    linear(upto(std::max(1, (1 << 20) / lh)), upto(most), lh, 1, 16 * upto(16), 16 * upto(16), upto(most));
  }
  std::printf("launch_checks: %d failures\n", fails);
  return fails != 0;
}
