// Attention of a sequence's newest tokens over its paged key/value cache, on gfx950 MFMA.
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j],  j <= i, and with a window i - j < window or
//   j < sinks
//
// One pass over the keys with a running maximum and sum (in fp32).  The cache is read once, so
// HBM bounds the call while the rows (new tokens x query heads of a key head) are few: no LDS
// stands between the cache and the matrix cores.  The stored layouts put 16 bytes that one lane
// of a fragment wants side by side, and a wave's 64 lanes in runs of 256 bytes:
//   * a wave takes 64 keys a step as four granules of 16.  S^T = K Q^T on 16x16x32 MFMA: tile t
//     (0..3) has granule g's tokens 4t..4t+3 in its rows 4g..4g+3, so the lanes of group g (lane / 16)
//     end up with all 16 scores of granule g of their query (lane % 16).
//   * O^T = V^T P^T wants of group g the values and probabilities of 8 tokens of one granule: the
//     probabilities are in place, with no lane exchange, and 16 bytes of the stored values are
//     16 (8-bit) or 8 tokens of one channel.
// e4m3 codes become f16 or bf16 exactly; the key scale multiplies the scores, one factor a lane.
// The value scale goes into the exponent: with w = exp2(t + log2 vs - M), M the running maximum of
// t + log2 vs, the output is sum w V / sum (w / vs), so no product of a code and its scale can leave
// the 16-bit range.  Weights are rounded to 16 bits for the second product.  A page's keys count in the
// sum however small its values are (zeros have the scale 2^-32): the sum is of the weights before
// their rounding where fp16 would lose them, else of the rounded ones.
//
// Few rows: a work-group's four waves take every fourth step, and further work-groups further keys;
// the partial sums are joined through LDS and by a second kernel.  Many rows: each wave takes rows
// of its own.
//
// Measured, 32 query heads on 8 key heads of 128 channels, 8-bit pages: 64 sequences of 8192 tokens
// 191 us, 5.6 TB/s of cache (16-bit pages 361, 5.9); 64 of 900 to 16001 208 us, 5.3 TB/s: HBM.  One of 5000
// 12 us, of which the join is 4: the chain offsets, table, keys, values and a second launch.  5 new
// tokens of 24 sequences in a window of 1024 16.4 to 16.7 us: the same chain and 5 steps a wave.  512 new tokens
// of one over 8192 keys 147 us, 0.45 PFLOP/s: a wave reads every key for its own 16 rows, from L2.
#pragma once

#include <algorithm>
#include <stdexcept>

#include "conv_common.hpp"
#include "seq_common.hpp"

namespace ivh {

namespace {

// the steps of 64 keys that rows at places imin..imax need: `first` of them over the first
// tokens, the others from step `from` on
struct Steps {
  int total, first, from;
};
__device__ __forceinline__ Steps key_steps(int full, int imin, int imax, int window, int sinks, int skip)
{
  const int end = imax >= full ? full : imax + 1;
  const int lo = window ? (int)min(max((long)imin - window + 1, 0L), (long)max(end, 0)) : min(skip, max(end, 0));
  Steps s;
  s.from = lo / 64;
  s.first = min((min(sinks, lo) + 63) / 64, s.from);
  s.total = end > 0 ? s.first + (end + 63) / 64 - s.from : 0;
  return s;
}
__device__ __forceinline__ int step_key(const Steps & s, int n) { return 64 * (n < s.first ? n : s.from + n - s.first); }

// Which keys a build takes: all of a sequence; those behind what its group shares; a group's shared ones,
// for the rows of all its sequences; or the last two side by side, `shared_wgs` work-groups for the latter, in
// tiles of 16 rows or by shared_rows.
enum KeysOf : int { kAllKeys, kOwnKeys, kSharedKeys, kBothKeys, kBothWide };

// A group's first sequence and rows, and the leading keys that are taken once for all of them: whole
// pages and steps, of which the first new row of every sequence sees each, so that nothing is masked.
struct SharedPart {
  int first, c0, c1, keys;
};
__device__ __forceinline__ int whole_keys(const CacheParams & c, int keys)
{
#pragma unroll
  for (int i = 32; i >= 1; i /= 2) keys = min(keys, __shfl_xor(keys, i));
  const int unit = max(c.page, 64);
  return __builtin_amdgcn_readfirstlane(keys / unit * unit);
}
// of group g, or where that is -1 of sequence b's group (no keys if it has none)
__device__ __forceinline__ SharedPart shared_part(const PagedParams & p, int g, int b)
{
  const CacheParams & c = p.c;
  const int lane = threadIdx.x & 63;
  auto seq = [&](int i) { return min(max(i, 0), c.batch); };
  auto row = [&](int i) { return min(max(i, 0), c.tokens); };
  if (p.groups < 64 && c.batch <= 128) {
    // what is read does not wait for one another: a trip to memory instead of four
    const int m = p.member[min(lane, p.groups)], s = p.shared[min(lane, p.groups - 1)];
    int r0[2], r1[2], len[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = min(lane + 64 * i, c.batch - 1);
      r0[i] = c.cu[at];
      r1[i] = c.cu[at + 1];
      len[i] = c.lens[at];
    }
    if (g < 0) {
      const unsigned long long below = __ballot(lane < p.groups && m <= b);
      if (below == 0) return SharedPart{0, 0, 0, 0};
      g = 63 - __clzll(below);
      if (b >= __builtin_amdgcn_readlane(m, g + 1)) return SharedPart{0, 0, 0, 0};
    }
    const int b0 = seq(__builtin_amdgcn_readlane(m, g)), b1 = max(seq(__builtin_amdgcn_readlane(m, g + 1)), b0);
    if (b1 == b0) return SharedPart{0, 0, 0, 0};
    int keys = min(max(__builtin_amdgcn_readlane(s, g), 0), c.width * c.page);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = lane + 64 * i, c0 = row(r0[i]), n = max(row(r1[i]), c0) - c0;
      if (at >= b0 && at < b1 && n > 0) keys = min(keys, max(max(len[i], 0) - n + 1, 0));
    }
    const int c0 = row(b0 < 64 ? __builtin_amdgcn_readlane(r0[0], b0) : __builtin_amdgcn_readlane(r0[1], b0 - 64));
    const int c1 = row(b1 <= 64 ? __builtin_amdgcn_readlane(r1[0], b1 - 1) : __builtin_amdgcn_readlane(r1[1], b1 - 65));
    return SharedPart{b0, c0, max(c1, c0), whole_keys(c, keys)};
  }
  if (g < 0) {
    g = find_seq(p.groups, b, [&](int i) { return (long)p.member[i]; });
    if (p.member[g] > b || b >= p.member[g + 1]) return SharedPart{0, 0, 0, 0};
  }
  const int b0 = seq(p.member[g]), b1 = max(seq(p.member[g + 1]), b0);
  int keys = min(max(p.shared[g], 0), c.width * c.page);
  for (int i = b0 + lane; i < b1; i += 64) {
    const int c0 = row(c.cu[i]), n = max(row(c.cu[i + 1]), c0) - c0;
    if (n > 0) keys = min(keys, max(max(c.lens[i], 0) - n + 1, 0));
  }
  const int c0 = row(c.cu[b0]);
  return SharedPart{b0, c0, max(row(c.cu[b1]), c0), whole_keys(c, keys)};
}

}  // namespace

// A group's shared keys for 32 rows (prefix_attn.hpp).
template <int TYPE, int BITS, int DP, bool FULL> __device__ __forceinline__ void shared_rows(const PagedParams & p, int block, float * lds);

// QT: 16-row tiles of a wave; WK: waves that share rows and split the keys, 4 / WK row ranges.
// DP: head size rounded up to 64, 128 or 256; FULL: it is that size.
template <int TYPE, int BITS, int DP, bool FULL, int QT, int WK, int KEYS>
__global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) paged_attn_kernel(const PagedParams p, int units)
{
  extern __shared__ __attribute__((aligned(16))) float lds[];
  constexpr bool BOTH = KEYS == kBothKeys || KEYS == kBothWide;
  const bool shared = KEYS == kSharedKeys || (BOTH && (int)blockIdx.x < p.shared_wgs);
  const int block = blockIdx.x - (BOTH && !shared ? p.shared_wgs : 0);
  if constexpr (KEYS == kBothWide) {
    if (shared) {
      shared_rows<TYPE, BITS, DP, FULL>(p, block, lds);
      return;
    }
  }
  const int row_slots = KEYS == kBothKeys && shared ? p.shared_slots : p.row_slots;
  const int parts = KEYS == kBothKeys && shared ? p.lead : p.parts, part_steps = KEYS == kBothKeys && shared ? p.shared_steps : p.part_steps;
  using T = St<TYPE>;
  typedef typename T::e E;
  constexpr int EK = BITS == 8 ? 16 : 8;        // channels of a 16-byte key piece
  constexpr int KL = DP / (4 * EK);             // key pieces of a lane and tile
  constexpr int VL = BITS == 8 ? 1 : 2;         // value pieces of a lane and channel block
  constexpr int NB = DP / 16;                   // channel blocks
  constexpr int NS = DP / 32;                   // 32-channel slices
  constexpr int ROWS = 16 * QT * (4 / WK);      // rows of a work-group
  // weights and the sums of values hold a power of two more: in fp16 those of 2^-21 of the largest are normal
  // numbers then and the largest is below 2^15; in bf16 small ones stay above fp32's lowest exponent
  // where pages' scales are 2^120 for the type's largest values and 2^-32 for zeros
  constexpr int UP = TYPE == kSeqF16 ? 7 : BITS == 8 ? 64 : 0;

  const CacheParams & c = p.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int wk = wave % WK, wr = wave / WK;
  // A unit (part of the keys, sequence, key head) has row_slots work-groups, on one XCD; units go
  // round the XCDs, so that each gets its share of long and short sequences, and of their last parts,
  // which only long ones have and which come last.
  int w = block / kXcds;
  const int slot = w % row_slots;
  w = w / row_slots * kXcds + block % kXcds;
  const int seqs = (KEYS != kAllKeys && shared ? p.groups : c.batch) * c.heads;
  if (w >= (BOTH ? seqs * parts : units)) return;
  const int part = w / seqs;
  w -= part * seqs;
  const int h = w % c.heads, b = w / c.heads;

  int c0, c1, full, place0, skip = 0;  // place0: of the first new token
  const int32_t * table = c.table;
  if (KEYS != kAllKeys && shared) {
    const SharedPart part_of = shared_part(p, b, 0);
    if (part_of.keys == 0) return;
    c0 = part_of.c0;
    c1 = part_of.c1;
    full = place0 = part_of.keys;  // every row sees all of them
    table += (long)part_of.first * c.width;
  } else {
    c0 = min(max(c.cu[b], 0), c.tokens);
    c1 = min(max(c.cu[b + 1], c0), c.tokens);
    const long len = c.lens[b];
    full = (int)min(max(len, 0L), (long)c.width * c.page);
    place0 = (int)max(len, 0L) - (c1 - c0);
    table += (long)b * c.width;
    if (KEYS != kAllKeys && p.groups > 0) skip = shared_part(p, -1, b).keys;
  }
  const int nnew = c1 - c0, rows = nnew * p.group;
  const int lp = 31 - __clz(c.page);  // page is a power of two
  const long page_bytes = (long)c.page * c.dim * (BITS / 8);
  const int nblk = c.dim / 16;
  // a negative scale turns the queries' signs, so that the largest score has the largest exponent
  const float scale = fmaxf(fabsf(p.scale_log2), 1.2e-38f);  // not 0: masked scores stay -inf
  const unsigned flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;

  for (int tile = slot; tile * ROWS < rows; tile += row_slots) {
    const int row0 = tile * ROWS + wr * 16 * QT, rend = min(rows, row0 + 16 * QT);  // this wave's rows
    const int wg_last = min(rows, tile * ROWS + ROWS) - 1;
    // the steps are the work-group's, the masks this wave's (which may have no rows)
    const Steps steps = key_steps(full, place0 + tile * ROWS / p.group, place0 + wg_last / p.group, p.window, p.sinks, skip);
    const int imin = place0 + row0 / p.group, imax = place0 + (max(rend, row0 + 1) - 1) / p.group;
    const int per = max(part_steps, (steps.total + parts - 1) / parts);
    const int n0 = part * per, n1 = rend > row0 ? min(steps.total, n0 + per) : 0;

    // what this lane's query of each row tile sees: keys lo .. lo + n and the first `first`
    int seen_lo[QT], seen_n[QT], seen_first[QT];
    // Q^T fragments in the order of the key pieces: 8-bit pieces hold 16 channels, two slices
    u4v qf[QT][NS];
    auto query_ch = [&](int s) { return BITS == 8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g; };
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int row = row0 + 16 * t + r, tok = row / p.group;
      const bool live = row < rows;
      const int place = place0 + tok, hi = live ? min(place, full - 1) : -1;
      seen_lo[t] = p.window ? (int)max((long)place - p.window + 1, 0L) : skip;
      seen_n[t] = hi - seen_lo[t];
      seen_first[t] = p.window ? min(p.sinks, hi + 1) : 0;
      // rows and channels that are not there read some that are: a branch would make each load wait
      // for the one before
      const int there = live ? row : 0, from = there / p.group;
      const E * q = static_cast<const E *>(p.q) + (long)(c0 + from) * p.q_token + (long)(h * p.group + there - from * p.group) * p.q_head;
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[t][s] = *reinterpret_cast<const u4v *>(q + (FULL || query_ch(s) < c.dim ? query_ch(s) : 0));
    }
    auto settle_queries = [&]() __attribute__((always_inline)) {  // when they are there
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int s = 0; s < NS; ++s)
          qf[t][s] = row0 + 16 * t + r < rows && (FULL || query_ch(s) < c.dim) ? qf[t][s] ^ flip : u4v{0, 0, 0, 0};
    };

    f4v o[QT][NB];
    float M[QT], L[QT];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        M[t] = kLowest;
        L[t] = 0.0f;
#pragma unroll
        for (int j = 0; j < NB; ++j) o[t][j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
      }
    };

    // page of the granule that this lane reads keys from (r / 4), and of its own group's
    auto page_of = [&](int n, int gran) { return table[min((step_key(steps, n) + 16 * gran) >> lp, c.width - 1)]; };
    u4v kf[4][KL], vf[NB][VL];
    float ksc = 1.0f, vsc = 1.0f;
    bool vok = true;
    auto load_k = [&](int n, int id) __attribute__((always_inline)) {
      const bool ok = (unsigned)id < (unsigned)c.pages;
      const uint8_t * base = static_cast<const uint8_t *>(c.kc) + ((long)(ok ? id : 0) * c.heads + h) * page_bytes;
      const int quad = ((step_key(steps, n) + 16 * (r >> 2)) & (c.page - 1)) / 4;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const int ch = FULL ? 4 * i + g : min(4 * i + g, c.dim / EK - 1);
          kf[t][i] = *reinterpret_cast<const u4v *>(base + ((unsigned)((quad + t) * (c.dim / EK) + ch) * 64u + (unsigned)(r & 3) * 16u));
        }
    };
    auto load_v = [&](int n, int id) __attribute__((always_inline)) {
      vok = (unsigned)id < (unsigned)c.pages;
      const long page = (long)(vok ? id : 0) * c.heads + h;
      if (BITS == 8) {
        ksc = c.ks[page];
        vsc = c.vs[page];
      }
      const uint8_t * base = static_cast<const uint8_t *>(c.vc) + page * page_bytes;
      const int gran = ((step_key(steps, n) + 16 * g) & (c.page - 1)) / 16;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < VL; ++i)
          vf[j][i] = *reinterpret_cast<const u4v *>(base + ((unsigned)((gran * VL + i) * c.dim) + 16u * (FULL ? j : min(j, nblk - 1)) + r) * 16u);
    };
    // S^T of the step whose keys are in kf
    auto scores = [&](f4v (&s)[QT][4]) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          u4v x = kf[t][i];
          if (!FULL && (4 * i + g) * EK >= c.dim) x = u4v{0, 0, 0, 0};
          if constexpr (BITS == 8) {
            const u4v lo = {T::fp8_lo(x[0]), T::fp8_hi(x[0]), T::fp8_lo(x[1]), T::fp8_hi(x[1])};
            const u4v hi = {T::fp8_lo(x[2]), T::fp8_hi(x[2]), T::fp8_lo(x[3]), T::fp8_hi(x[3])};
#pragma unroll
            for (int u = 0; u < QT; ++u) {
              s[u][t] = T::mma16(lo, qf[u][2 * i], i ? s[u][t] : f4v{0.0f, 0.0f, 0.0f, 0.0f});
              s[u][t] = T::mma16(hi, qf[u][2 * i + 1], s[u][t]);
            }
          } else {
#pragma unroll
            for (int u = 0; u < QT; ++u) s[u][t] = T::mma16(x, qf[u][i], i ? s[u][t] : f4v{0.0f, 0.0f, 0.0f, 0.0f});
          }
        }
    };
    // whether every row of the wave sees all keys of step n
    auto inner_of = [&](int n, bool ok) {
      const int key = step_key(steps, n);
      return key + 63 <= imin && key + 63 < full && (p.window == 0 || imax - key < p.window || key + 63 < p.sinks) && __all(ok);
    };
    // masks, running maximum, weights in 16 bits
    auto weights = [&](int key0, bool inner, bool ok, float ks, float vs, f4v (&s)[QT][4], u4v (&pf)[QT][2]) __attribute__((always_inline)) {
      if (!inner && !(ok && key0 + 16 * g < full)) ks = vs = 1.0f;  // a granule without tokens: its scales may be anything
      // a product of small scales is not 0 either
      const float mul = BITS == 8 ? fmaxf(scale * ks, 1.2e-38f) : scale, ev = BITS == 8 ? __builtin_amdgcn_logf(vs) : 0.0f;
      // 2^-UP / vs, whose exponent may not fit
      const float unv = __builtin_amdgcn_rcpf(__builtin_amdgcn_frexp_mantf(vs));
      const int unv_exp = -UP - __builtin_amdgcn_frexp_expf(vs);
      float top[QT];
      bool grow = false;
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        if (!inner) {
          const int base = key0 + 16 * g;
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int j = base + x;
            const bool see = ok && ((seen_n[u] >= 0 && (unsigned)j - (unsigned)seen_lo[u] <= (unsigned)seen_n[u]) || j < seen_first[u]);
            s[u][x / 4][x % 4] = see ? s[u][x / 4][x % 4] : -__builtin_inff();
          }
        }
        float a = s[u][0][0], d = s[u][0][1];
#pragma unroll
        for (int x = 2; x < 16; x += 4) {
          a = top_of(a, s[u][x / 4][x % 4], s[u][x / 4][x % 4 + 1]);
          if (x + 2 < 16) d = top_of(d, s[u][(x + 2) / 4][(x + 2) % 4], s[u][(x + 2) / 4][(x + 2) % 4 + 1]);
        }
        // the page's scales are the lane group's: they enter before the groups are compared
        top[u] = across16(across32(fmaf(top_of(a, d, d), mul, ev), MaxOp()), MaxOp());
        grow = grow || top[u] > M[u] + 8.0f;
      }
      // the reference exponent follows the maximum only when that is 2^8 above it: weights that are
      // larger by that lose nothing in either 16-bit type
      if (__any(grow)) {
#pragma unroll
        for (int u = 0; u < QT; ++u) {
          const float m = fmaxf(M[u], top[u]), a = __builtin_amdgcn_exp2f(M[u] - m);
          M[u] = m;
          L[u] *= a;
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) o[u][j][v] *= a;
        }
      }
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        const float shift = ev + UP - M[u];
        float sum = 0.0f, sum2 = 0.0f;
#pragma unroll
        for (int x = 0; x < 16; x += 2) {
          const f4v & y = s[u][x / 4];
          const float e0 = __builtin_amdgcn_exp2f(fmaf(y[x % 4], mul, shift)), e1 = __builtin_amdgcn_exp2f(fmaf(y[x % 4 + 1], mul, shift));
          const unsigned e = pack2<TYPE>(e0, e1);
          pf[u][x / 8][x % 8 / 2] = e;
          if (TYPE == kSeqF16 && BITS == 8) {  // rounded to fp16, those of a page of small values are gone
            sum += e0;
            sum2 += e1;
          } else {
            sum = T::add2(e, sum);
          }
        }
        if (TYPE == kSeqF16 && BITS == 8) sum += sum2;
        if (BITS == 8) L[u] += __builtin_ldexpf(sum * unv, unv_exp);
        else L[u] = fmaf(sum, __builtin_ldexpf(1.0f, -UP), L[u]);
      }
    };
    // values that no row sees (behind the last key, outside every window, in no page) may be
    // anything: zeros in their place
    auto keep = [&](int key0, bool ok) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < VL; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          constexpr int PER = BITS == 8 ? 4 : 2;
          unsigned m = 0;
#pragma unroll
          for (int t = 0; t < PER; ++t) {
            const int j = key0 + 16 * g + (BITS == 8 ? 4 * q + t : 8 * i + 2 * q + t);
            const bool any = ok && j < full && j <= imax && (p.window == 0 || imin - j < p.window || j < p.sinks);
            m |= any ? (BITS == 8 ? 0xffu << (8 * t) : 0xffffu << (16 * t)) : 0u;
          }
#pragma unroll
          for (int j = 0; j < NB; ++j) vf[j][i][q] &= m;
        }
    };
    // O^T += V^T P^T
    auto values = [&](const u4v (&pf)[QT][2]) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        u4v v0, v1;
        if constexpr (BITS == 8) {
          const u4v x = vf[j][0];
          v0 = u4v{T::fp8_lo(x[0]), T::fp8_hi(x[0]), T::fp8_lo(x[1]), T::fp8_hi(x[1])};
          v1 = u4v{T::fp8_lo(x[2]), T::fp8_hi(x[2]), T::fp8_lo(x[3]), T::fp8_hi(x[3])};
        } else {
          v0 = vf[j][0];
          v1 = vf[j][VL - 1];
        }
#pragma unroll
        for (int u = 0; u < QT; ++u) {
          o[u][j] = T::mma16(v0, pf[u][0], o[u][j]);
          o[u][j] = T::mma16(v1, pf[u][1], o[u][j]);
        }
      }
    };
    // Step n, whose keys and values are on their way; the next step's are asked for as soon as the
    // registers are free (id: its pages), which keeps 8 to 16 KB of a wave in flight.
    auto step = [&](int n, auto more, int idk, int idv) __attribute__((always_inline)) {
      f4v s[QT][4];
      u4v pf[QT][2];
      scores(s);
      const bool ok = vok;
      const float ks = ksc, vs = BITS == 8 ? fmaxf(vsc, 1e-30f) : 1.0f;
      if (more) load_k(n + WK, idk);
      const bool inner = inner_of(n, ok);
      weights(step_key(steps, n), inner, ok, ks, vs, s, pf);
      if (!inner) keep(step_key(steps, n), ok);
      values(pf);
      if (more) load_v(n + WK, idv);
    };
    constexpr std::integral_constant<bool, true> more{};
    constexpr std::integral_constant<bool, false> last{};

    clear();
    int n = n0 + wk;
    if (n < n1) {
      // page numbers of two steps before the first step's data, in the order of the loop: the
      // compiler's counted waits then hold for the first pass through it as well
      const int firstk = page_of(n, r >> 2), firstv = page_of(n, g);
      int idk = page_of(min(n + WK, n1 - 1), r >> 2), idv = page_of(min(n + WK, n1 - 1), g);
      __builtin_amdgcn_sched_barrier(0);
      load_k(n, firstk);
      load_v(n, firstv);
      settle_queries();
      for (; n + WK < n1; n += WK) {
        const int nk = idk, nv = idv;  // pages two steps ahead
        idk = page_of(min(n + 2 * WK, n1 - 1), r >> 2);
        idv = page_of(min(n + 2 * WK, n1 - 1), g);
        step(n, more, nk, nv);
      }
      step(n, last, 0, 0);
    }
    // With several tokens among the rows an infinity or NaN among the values reaches rows that do
    // not see it, as 0 x inf, and stays in their sums.  If a result is not finite the wave's steps are
    // taken again with such values left out of the product and added to the rows that do see them.
    if (imax > imin) {
      bool odd = false;
#pragma unroll
      for (int u = 0; u < QT; ++u)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) odd = odd || !(fabsf(o[u][j][v]) < __builtin_inff());
      if (__any(odd)) {
        clear();
        for (n = n0 + wk; n < n1; n += WK) {
          const int key0 = step_key(steps, n);
          f4v s[QT][4];
          u4v pf[QT][2];
          load_k(n, page_of(n, r >> 2));
          load_v(n, page_of(n, g));
          scores(s);
          const float vs = BITS == 8 ? fmaxf(vsc, 1e-30f) : 1.0f;
          weights(key0, false, vok, ksc, vs, s, pf);
          keep(key0, vok);
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int i = 0; i < VL; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const unsigned x = vf[j][i][q];
                // top bits of the elements to drop, spread over them
                const unsigned d = BITS == 8 ? (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) : T::odd_bits(x);
                vf[j][i][q] = x & ~(BITS == 8 ? (d >> 7) * 0xffu : (d >> 15) * 0xffffu);
              }
          values(pf);
          for (int key = key0; key < min(key0 + 64, full); ++key) {
            const int id = table[key >> lp], in = key & (c.page - 1);
            if ((unsigned)id >= (unsigned)c.pages) continue;
            const uint8_t * base = static_cast<const uint8_t *>(c.vc) + ((long)id * c.heads + h) * page_bytes;
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                const int ch = (FULL ? 16 * j : 16 * min(j, nblk - 1)) + 4 * g + v;
                float x;
                if (BITS == 8) x = __builtin_amdgcn_cvt_f32_fp8((int)base[((in / 16) * c.dim + ch) * 16 + in % 16], 0);
                else x = (float)reinterpret_cast<const E *>(base)[((in / 8) * c.dim + ch) * 8 + in % 8];
                if (fabsf(x) < __builtin_inff()) continue;
#pragma unroll
                for (int u = 0; u < QT; ++u)
                  if ((seen_n[u] >= 0 && (unsigned)key - (unsigned)seen_lo[u] <= (unsigned)seen_n[u]) || key < seen_first[u]) o[u][j][v] += x;
              }
          }
        }
      }
    }

    // ---- join: the sums of a query's four lane groups, then the waves that share its keys
#pragma unroll
    for (int u = 0; u < QT; ++u) L[u] = across16(across32(L[u], SumOp()), SumOp());
    constexpr int PITCH = DP + 4;  // floats of a row in LDS: 16-byte pieces of 16 rows in distinct banks
    float * oml = lds + (WK / 2) * (4 / WK) * 16 * QT * PITCH;
#pragma unroll
    for (int half = WK / 2; half >= 1; half /= 2) {  // upper half of the waves into LDS, lower half adds
      float * mine = lds + ((wk % half) + wr * half) * 16 * QT * PITCH;
      float * ml = oml + ((wk % half) + wr * half) * 16 * QT * 2;
      __syncthreads();
      if (wk >= half && wk < 2 * half) {
#pragma unroll
        for (int u = 0; u < QT; ++u) {
#pragma unroll
          for (int j = 0; j < NB; ++j) *reinterpret_cast<f4v *>(mine + (16 * u + r) * PITCH + 16 * j + 4 * g) = o[u][j];
          if (g == 0) *reinterpret_cast<f2v *>(ml + 2 * (16 * u + r)) = f2v{M[u], L[u]};
        }
      }
      __syncthreads();
      if (wk < half) {
#pragma unroll
        for (int u = 0; u < QT; ++u) {
          const f2v t = *reinterpret_cast<const f2v *>(ml + 2 * (16 * u + r));
          const float m = fmaxf(M[u], t[0]), a = __builtin_amdgcn_exp2f(M[u] - m), e = __builtin_amdgcn_exp2f(t[0] - m);
          M[u] = m;
          L[u] = L[u] * a + t[1] * e;
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            const f4v x = *reinterpret_cast<const f4v *>(mine + (16 * u + r) * PITCH + 16 * j + 4 * g);
#pragma unroll
            for (int v = 0; v < 4; ++v) o[u][j][v] = o[u][j][v] * a + x[v] * e;
          }
        }
      }
    }
    if (wk == 0) {
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        const int at_row = row0 + 16 * u + r, tok = at_row / p.group, head = h * p.group + at_row - tok * p.group;
        if (at_row >= rows) continue;
        if (UP)
#pragma unroll
          for (int j = 0; j < NB; ++j) o[u][j] *= __builtin_ldexpf(1.0f, -UP);
        const long row = (long)(c0 + tok) * p.heads + head;
        if (KEYS == kAllKeys && p.parts == 1) {
          const float inv = L[u] != 0.0f ? 1.0f / L[u] : 0.0f;  // a row that saw nothing is zero (NaN stays)
          E * out = static_cast<E *>(p.o) + (long)(c0 + tok) * p.o_token + (long)head * p.o_head;
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            if (!FULL && j >= nblk) continue;
            const u2v y = {pack2<TYPE>(o[u][j][0] * inv, o[u][j][1] * inv), pack2<TYPE>(o[u][j][2] * inv, o[u][j][3] * inv)};
            *reinterpret_cast<u2v *>(out + 16 * j + 4 * g) = y;
          }
        } else {
          const long total = (long)c.tokens * p.heads, at = (long)(part + (KEYS != kAllKeys && !shared ? p.lead : 0)) * total + row;
          const long all = KEYS == kAllKeys ? p.parts : p.all_parts;
          if (n0 < n1) {
            float * out = p.ws + at * c.dim;
#pragma unroll
            for (int j = 0; j < NB; ++j)
              if (FULL || j < nblk) *reinterpret_cast<f4v *>(out + 16 * j + 4 * g) = o[u][j];
          }
          f2v * ml = reinterpret_cast<f2v *>(p.ws + all * total * c.dim);
          if (g == 0) ml[at] = f2v{M[u], L[u]};
          // a sequence that shares nothing leaves the parts of groups empty
          if (KEYS != kAllKeys && !shared && skip == 0 && part == 0 && g == 0)
            for (int i = 0; i < p.lead; ++i) ml[i * total + row] = f2v{kLowest, 0.0f};
        }
      }
    }
  }
}

// Joins the parts of a row.  dim / 4 lanes have 4 channels each of every lots-th part, with a running
// maximum; the lots of a row meet in LDS.  A part that had no keys for the row left a sum of zero, and its
// values are not read.  first: the launch's first row.
template <int TYPE>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedParams p, int lots, long first)
{
  typedef typename St<TYPE>::e E;
  __shared__ __attribute__((aligned(16))) float sum[256 * 4];
  __shared__ float top[256], den[256];
  const CacheParams & c = p.c;
  const int lanes = c.dim / 4, tid = threadIdx.x, at = tid / lanes, ch = 4 * (tid - at * lanes);
  const int per = 256 / (lanes * lots), lot = at / per, sub = at - lot * per;  // rows of a work-group
  const long n = (long)c.tokens * p.heads, row = first + (long)blockIdx.x * per + sub;
  const int token = (int)(row / p.heads), head = (int)(row - (long)token * p.heads);
  // rows of no sequence stay as they are
  const bool on = lot < lots && row < n && token >= c.cu[0] && token < c.cu[c.batch];
  const f2v * ml = reinterpret_cast<const f2v *>(p.ws + (long)p.parts * n * c.dim);
  float M = kLowest, L = 0.0f;
  f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (on) {
#pragma unroll 4
    for (int i = lot; i < p.parts; i += lots) {
      const long x = (long)i * n + row;
      const f2v t = ml[x];
      if (t[1] == 0.0f) continue;
      const f4v v = *reinterpret_cast<const f4v *>(p.ws + x * c.dim + ch);
      const float m = fmaxf(M, t[0]), a = __builtin_amdgcn_exp2f(M - m), e = __builtin_amdgcn_exp2f(t[0] - m);
      M = m;
      L = L * a + t[1] * e;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = o[k] * a + v[k] * e;
    }
  }
  if (lots > 1) {
    *reinterpret_cast<f4v *>(sum + 4 * tid) = o;
    top[tid] = M;
    den[tid] = L;
    __syncthreads();
    if (!on || lot) return;
    for (int i = 1; i < lots; ++i) {
      const int other = tid + i * per * lanes;
      const f4v v = *reinterpret_cast<const f4v *>(sum + 4 * other);
      const float m = fmaxf(M, top[other]), a = __builtin_amdgcn_exp2f(M - m), e = __builtin_amdgcn_exp2f(top[other] - m);
      M = m;
      L = L * a + den[other] * e;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = o[k] * a + v[k] * e;
    }
  } else if (!on) {
    return;
  }
  const float inv = L != 0.0f ? 1.0f / L : 0.0f;
  const u2v y = {pack2<TYPE>(o[0] * inv, o[1] * inv), pack2<TYPE>(o[2] * inv, o[3] * inv)};
  *reinterpret_cast<u2v *>(static_cast<E *>(p.o) + (long)token * p.o_token + (long)head * p.o_head + ch) = y;
}

namespace {

template <int TYPE, int BITS, int DP, bool FULL, int QT, int WK, int KEYS> void launch_paged(const PagedParams & p, hipStream_t s)
{
  auto kern = paged_attn_kernel<TYPE, BITS, DP, FULL, QT, WK, KEYS>;
  const size_t own = (size_t)(WK / 2) * (4 / WK) * 16 * QT * (DP + 4 + 2) * sizeof(float), wide = (size_t)2 * 32 * (DP + 4 + 2) * sizeof(float);
  const size_t lds = KEYS == kBothWide ? std::max(own, wide) : own;
  const long seqs = KEYS == kSharedKeys ? p.groups : p.c.batch;
  const dim3 grid((unsigned)(paged_wgs(p, seqs) + (KEYS == kBothKeys || KEYS == kBothWide ? p.shared_wgs : 0))), blk(256);
  hipLaunchKernelGGL(kern, grid, blk, lds, s, p, (int)(seqs * p.c.heads * p.parts));
}

template <int TYPE, int BITS, int DP, bool FULL, int KEYS> void launch_paged_rows(const PagedParams & p, hipStream_t s)
{
  constexpr int MOST = DP <= 64 ? 2 : 1;
  if (p.row_waves == 1) {
    if (p.row_tiles == 1) launch_paged<TYPE, BITS, DP, FULL, 1, 4, KEYS>(p, s);
    else launch_paged<TYPE, BITS, DP, FULL, MOST, 4, KEYS>(p, s);
  } else if (p.row_waves == 2) {
    launch_paged<TYPE, BITS, DP, FULL, MOST, 2, KEYS>(p, s);
  } else {
    launch_paged<TYPE, BITS, DP, FULL, MOST, 1, KEYS>(p, s);
  }
}

template <int TYPE, int BITS, int KEYS = kAllKeys> void launch_paged_dim(const PagedParams & p, hipStream_t s)
{
  if (p.c.dim == 64) launch_paged_rows<TYPE, BITS, 64, true, KEYS>(p, s);
  else if (p.c.dim < 64) launch_paged_rows<TYPE, BITS, 64, false, KEYS>(p, s);
  else if (p.c.dim == 128) launch_paged_rows<TYPE, BITS, 128, true, KEYS>(p, s);
  else if (p.c.dim < 128) launch_paged_rows<TYPE, BITS, 128, false, KEYS>(p, s);
  else if constexpr (KEYS == kBothWide) throw std::logic_error("head size");
  else if (p.c.dim == 256) launch_paged_rows<TYPE, BITS, 256, true, KEYS>(p, s);
  else launch_paged_rows<TYPE, BITS, 256, false, KEYS>(p, s);
}

template <int TYPE> void launch_paged_join(const PagedParams & p, hipStream_t s)
{
  const JoinSplit j = join_split(p);
  for (long first = 0; first < j.wgs; first += kJoinWgs)
    hipLaunchKernelGGL((paged_join_kernel<TYPE>), dim3((unsigned)std::min(j.wgs - first, kJoinWgs)), dim3(256), 0, s, p, j.lots, first * j.per);
}

template <int TYPE> void launch_paged_type(const PagedParams & p, hipStream_t s)
{
  if (p.c.bits == 8) launch_paged_dim<TYPE, 8>(p, s);
  else launch_paged_dim<TYPE, 16>(p, s);
  if (p.parts > 1) launch_paged_join<TYPE>(p, s);
}

}  // namespace

}  // namespace ivh
