// Attention over a paged cache whose first pages the sequences of a group share, on gfx950 MFMA.
//
//   o[i] = (e^(m1 - m) o1 + e^(m2 - m) o2) / (e^(m1 - m) l1 + e^(m2 - m) l2),  m = max(m1, m2)
//
// with (m1, l1, o1) the maximum, sum and weighted values over the group's shared keys and (m2, l2, o2) those over
// the sequence's own: the shared keys are read once for the rows of all sequences, which are contiguous.
// All parts are joined by a kernel behind them.  Own keys take the paged attention's kernel; shared ones
//   * for up to 16 rows of a group (95 with heads of more than 64 channels), and where heads have more than 128, that
//     kernel as well, in work-groups of the same launch where the tiles agree.  With few rows the keys' latency counts.  8 key
//     heads, 8 bits, so and by 32 rows a wave: 128 channels behind 8192 tokens 48 rows 16.0 and 17.1 us, 96 19.8 and 20.1, 128 22.2 and
//     21.4 (behind 1024 15.3 and 17.5, 16.0 and 17.1 with 96 and 128 rows); 64 channels behind 1024 16 rows 13.4 and 13.4, 24 19.5 and 13.3;
//   * by 32 rows (shared_rows), in the same launch: each key that L2 gives has twice the rows of that kernel's tiles.
//     64 sequences of 4 rows a key head behind 8192 tokens, own keys of 20 to 1501, 8 bits: 52 -> 44 us, the kernel 38 to 39,
//     of which the keys' 94 MB are 18 at a copy's rate; 5 groups of 112 rows behind 700 to 6007 tokens in 16 bits 53 -> 37 us;
//     24 rows of 64 channels behind 1024 tokens 18 -> 13 us;
//   * with many rows of up to 64 channels behind a long prefix the keys' conversion and L2 bound that: a work-group has 128
//     rows, a wave 32 of them, and walks 64 keys a step (shared_attn_kernel).  The steps' keys and values stand in LDS in two
//     stages, in 16 bits, each 1024 bytes a fragment of 32 x 32 x 16 MFMA in the order of its lanes: they are read without a
//     bank conflict, and 8-bit codes are widened once for the four waves.  1536 rows a key head behind 32000 tokens: 180 us,
//     0.56 PFLOP/s; behind 16384 120 us in all, 127 by shared_rows, behind 8192 81 and 73.  Where the sides meet, 8 key heads, so and by
//     shared_rows, 8 and 16 bits: behind 16384 512 rows 56 and 55, 63 and 69 us, 384 rows 49 and 47, 53 and 53, 1024 88 and 98, 95 and 126;
//     behind 8192 512 rows 44 and 33, 49 and 40, 1024 61 and 54, 67 and 68; behind 32768 256 rows 52 and 55, 58 and 69.  With 128 channels
//     the accumulators leave two waves a SIMD and the barriers cost more than the copies save: 768 rows behind 32768 tokens 234
//     us, 191 by shared_rows.
// Both:
//   * S^T = K Q^T with keys in rows in an order of which a lane holds, of a 32-key part, the 16 keys of one granule
//     (8-bit pages) or two runs of 8 (16-bit): they are operands of O^T = V^T P^T as they are;
//   * weights, running maxima and scales as in paged_attn.hpp: weights are rounded to 16 bits for the second product, half a step each
//     and independently (outputs are 5 to 20 % further from 64 bits than with fp32 weights), since an operand of the matrix cores has
//     no more, and the sum is that of the rounded ones; nothing is masked but pages that hold nothing.
#pragma once

#include "paged_attn.hpp"

namespace ivh {

namespace {

typedef __attribute__((address_space(3))) void prefix_lds;

// 64 x 16 bytes straight into LDS (16-bit pages): lane i's from its address, to `to` + 16 i.  In assembler, so that copies stay in
// flight over barriers; shared_wait before the barrier that publishes them.
__device__ __forceinline__ void shared_copy(const uint8_t * at, void * to)
{
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(at), "s"(__builtin_amdgcn_readfirstlane((unsigned)(unsigned long)(prefix_lds *)to))
               : "memory", "m0");
#endif
}
__device__ __forceinline__ void shared_wait()
{
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(vm_wait(0));
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#endif
}

constexpr int kSharedRows = 128;

}  // namespace

// DP: head size rounded up to 64; FULL: it is that size.
template <int TYPE, int BITS, int DP, bool FULL>
__global__ void __launch_bounds__(256, 2) shared_attn_kernel(const PagedParams p, int units)
{
  using T = St<TYPE>;
  typedef typename T::e E;
  constexpr int EK = BITS == 8 ? 16 : 8;             // channels of a 16-byte key piece
  constexpr int KF = DP / (2 * EK);                  // key fragments of 32 keys
  constexpr int VS = BITS == 8 ? 1 : 2;              // value fragments of 32 keys and 32 channels
  constexpr int NB = DP / 32, NS = DP / 16;          // channel blocks of the second, slices of the first product
  constexpr int WIDE = BITS == 8 ? 2 : 1;            // fragments in LDS of one in memory
  constexpr int FRAGS = 2 * (NS + 2 * NB);           // in LDS, of a step: keys, then values
  constexpr int OWN_K = KF / 2, OWN_V = VS * NB / 2; // fragments in memory that a wave brings
  constexpr int UP = TYPE == kSeqF16 ? 7 : BITS == 8 ? 64 : 0;  // weights hold a power of two more, as in paged_attn.hpp
  __shared__ __attribute__((aligned(16))) unsigned char stage[2][FRAGS * 1024];

  const CacheParams & c = p.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  // as the paged attention: the row slots of a unit (part of the keys, group, key head) on one XCD
  int w = blockIdx.x / kXcds;
  const int slot = w % p.row_slots;
  w = w / p.row_slots * kXcds + blockIdx.x % kXcds;
  if (w >= units) return;
  const int seqs = p.groups * c.heads, part = w / seqs;
  w -= part * seqs;
  const int h = w % c.heads;
  const SharedPart own = shared_part(p, w / c.heads, 0);
  if (own.keys == 0) return;
  const int c0 = own.c0, rows = (own.c1 - c0) * p.group;
  const int32_t * table = c.table + (long)own.first * c.width;
  const int lp = 31 - __clz(c.page), last = (own.keys >> lp) - 1;
  const long page_bytes = (long)c.page * c.dim * (BITS / 8);
  const int total = own.keys / 64, per = max(p.part_steps, (total + p.parts - 1) / p.parts);
  const int n0 = part * per, n1 = min(total, n0 + per);
  // a negative scale turns the queries' signs, so that the largest score has the largest exponent
  const float scale = fmaxf(fabsf(p.scale_log2), 1.2e-38f);
  const unsigned flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;

  // what this lane copies of a fragment: granule and piece of its key row, channel of its value row
  const int mi = col >> 3, mh = col >> 2 & 1, mj = col & 3;
  const int key_gran = BITS == 8 ? mh : mi >> 1, key_quad = BITS == 8 ? mi : 2 * mh + (mi & 1);
  auto page_at = [&](int n, int gran) { return table[min((64 * n + 16 * gran) >> lp, last)]; };
  struct Ids {
    int id[4];
  };
  auto ask_ids = [&](int n) {
    Ids x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.id[i] = page_at(n, i);
    return x;
  };
  auto settle_ids = [&](const Ids & ids) {  // the same in every lane
    Ids x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.id[i] = __builtin_amdgcn_readfirstlane(ids.id[i]);
    return x;
  };
  auto valid = [&](int id) { return (unsigned)id < (unsigned)c.pages; };
  auto page_of = [&](int id) { return ((long)(valid(id) ? id : 0) * c.heads + h); };
  // A wave brings every fourth fragment, 32 keys at a time: 8-bit ones through registers, where they are widened
  const unsigned key_lane = (unsigned)(key_quad * (c.dim / EK) * 64 + mj * 16);
  u4v raw[BITS == 8 ? OWN_K + OWN_V : 1];
  auto bring = [&](int n, const Ids & ids, unsigned char * to) __attribute__((always_inline)) {
    auto granule = [&](const void * pages, int kt, int gran, unsigned piece) {  // where one begins, and its page
      const int in = ((64 * n + 16 * (2 * kt + gran)) & (c.page - 1)) / 16;
      return static_cast<const uint8_t *>(pages) + page_of(kt ? gran ? ids.id[3] : ids.id[2] : gran ? ids.id[1] : ids.id[0]) * page_bytes + in * piece;
    };
    const unsigned gran_bytes = 16u * c.dim * (BITS / 8);
#pragma unroll
    for (int x = 0; x < OWN_K; ++x) {
      const int f = 4 * x + wave, kt = f / KF, piece = 2 * (f % KF) + half;
      const uint8_t * a = granule(c.kc, kt, 0, gran_bytes), * b = granule(c.kc, kt, 1, gran_bytes);
      const uint8_t * k = (key_gran ? b : a) + key_lane + (unsigned)(FULL ? piece : min(piece, c.dim / EK - 1)) * 64u;
      if constexpr (BITS == 8) raw[x] = *reinterpret_cast<const u4v *>(k);
      else shared_copy(k, to + 1024 * f);
    }
#pragma unroll
    for (int x = 0; x < OWN_V; ++x) {
      const int f = 4 * x + wave, kt = f / (VS * NB), s = f / NB % VS, j = f % NB, ch = 32 * j + col;
      const uint8_t * a = granule(c.vc, kt, BITS == 8 ? 0 : s, gran_bytes), * b = BITS == 8 ? granule(c.vc, kt, 1, gran_bytes) : a + 16 * c.dim;
      const uint8_t * v = (half ? b : a) + (unsigned)(FULL ? ch : min(ch, c.dim - 1)) * 16u;
      if constexpr (BITS == 8) raw[OWN_K + x] = *reinterpret_cast<const u4v *>(v);
      else shared_copy(v, to + 1024 * (2 * NS + (kt * NB + j) * 2 + s));
    }
  };
  auto widen = [&](unsigned char * to) __attribute__((always_inline)) {
    if constexpr (BITS == 8) {
#pragma unroll
      for (int x = 0; x < OWN_K + OWN_V; ++x) {
        const int f = x < OWN_K ? 4 * x + wave : KF * 2 + 4 * (x - OWN_K) + wave;
        unsigned char * at = to + 2048 * f + 16 * lane;
        const u4v y = raw[x];
        *reinterpret_cast<u4v *>(at) = u4v{T::fp8_lo(y[0]), T::fp8_hi(y[0]), T::fp8_lo(y[1]), T::fp8_hi(y[1])};
        *reinterpret_cast<u4v *>(at + 1024) = u4v{T::fp8_lo(y[2]), T::fp8_hi(y[2]), T::fp8_lo(y[3]), T::fp8_hi(y[3])};
      }
    }
  };
  struct Scales {
    float k[2], v[2];  // of this lane's granule of each 32 keys
    bool ok[2];        // whether pages hold something: 8 bits this lane's granule; 16 bits both
    bool ok2[2];
  };
  auto ask_scales = [&](const Ids & ids) __attribute__((always_inline)) {
    Scales x;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int id = half ? ids.id[2 * kt + 1] : ids.id[2 * kt];
      x.k[kt] = x.v[kt] = 1.0f;
      if (BITS == 8) {
        x.k[kt] = c.ks[page_of(id)];
        x.v[kt] = c.vs[page_of(id)];
      }
      x.ok[kt] = valid(BITS == 8 ? id : ids.id[2 * kt]);
      x.ok2[kt] = valid(BITS == 8 ? id : ids.id[2 * kt + 1]);
    }
    return x;
  };

  for (int tile = slot; tile * kSharedRows < rows; tile += p.row_slots) {
    const int row0 = tile * kSharedRows + 32 * wave, row = row0 + col;
    const bool on = row0 < rows;
    u4v qf[NS];
    {
      const int there = min(row, rows - 1), tok = there / p.group;
      const E * q = static_cast<const E *>(p.q) + (long)(c0 + tok) * p.q_token + (long)(h * p.group + there - tok * p.group) * p.q_head;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int ch = BITS == 8 ? 16 * (2 * (i / 2) + half) + 8 * (i % 2) : 16 * i + 8 * half;
        const u4v x = *reinterpret_cast<const u4v *>(q + (FULL || ch < c.dim ? ch : 0));
        qf[i] = FULL || ch < c.dim ? x ^ flip : u4v{0, 0, 0, 0};
      }
    }
    f16v o[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) o[j] = f16v{};
    float M = kLowest, L = 0.0f;

    auto step = [&](const unsigned char * from, const Scales & sc) __attribute__((always_inline)) {
      // both halves of the keys side by side: their products, and their weights, do not wait for one another
      const unsigned char * at = from + 16 * lane;
      f16v s[2] = {};
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          u4v x = *reinterpret_cast<const u4v *>(at + (kt * NS + i) * 1024);
          if (!FULL && (2 * (i / WIDE) + half) * EK >= c.dim) x = u4v{0, 0, 0, 0};
          s[kt] = T::mma32(x, qf[i], s[kt]);
        }
      const bool whole = __all(sc.ok[0] && sc.ok2[0] && sc.ok[1] && sc.ok2[1]);
      float mul[2], ev[2], vs[2], top = kLowest;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        float ks = sc.k[kt];
        vs[kt] = BITS == 8 ? fmaxf(sc.v[kt], 1e-30f) : 1.0f;
        if (!whole) {
          if (!sc.ok[kt]) ks = vs[kt] = 1.0f;
#pragma unroll
          for (int v = 0; v < 16; ++v) s[kt][v] = (v < 8 ? sc.ok[kt] : sc.ok2[kt]) ? s[kt][v] : -__builtin_inff();
        }
        mul[kt] = BITS == 8 ? fmaxf(scale * ks, 1.2e-38f) : scale;
        ev[kt] = BITS == 8 ? __builtin_amdgcn_logf(vs[kt]) : 0.0f;
        float a = s[kt][0], d = s[kt][1];
#pragma unroll
        for (int v = 2; v < 16; v += 4) {
          a = top_of(a, s[kt][v], s[kt][v + 1]);
          if (v + 2 < 16) d = top_of(d, s[kt][v + 2], s[kt][v + 3]);
        }
        top = __builtin_elementwise_maximum(top, fmaf(top_of(a, d, d), mul[kt], ev[kt]));
      }
      top = across32(top, MaxOp());
      if (__any(top > M + 8.0f)) {
        const float m = fmaxf(M, top), e = __builtin_amdgcn_exp2f(M - m);
        M = m;
        L *= e;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[j][v] *= e;
      }
      u4v pf[2][2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const float shift = ev[kt] + UP - M;
        float sum = 0.0f, sum2 = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
          const float e0 = __builtin_amdgcn_exp2f(fmaf(s[kt][v], mul[kt], shift)), e1 = __builtin_amdgcn_exp2f(fmaf(s[kt][v + 1], mul[kt], shift));
          const unsigned e = pack2<TYPE>(e0, e1);
          pf[kt][v / 8][v % 8 / 2] = e;
          if (TYPE == kSeqF16 && BITS == 8) {
            sum += e0;
            sum2 += e1;
          } else {
            sum = T::add2(e, sum);
          }
        }
        if (BITS == 8)
          L += __builtin_ldexpf((sum + sum2) * __builtin_amdgcn_rcpf(__builtin_amdgcn_frexp_mantf(vs[kt])), -UP - __builtin_amdgcn_frexp_expf(vs[kt]));
        else L = fmaf(sum, __builtin_ldexpf(1.0f, -UP), L);
      }
      at += 2 * NS * 1024;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            u4v x = *reinterpret_cast<const u4v *>(at + ((kt * NB + j) * 2 + g) * 1024);
            if (!whole && !(g ? sc.ok2[kt] : sc.ok[kt])) x = u4v{0, 0, 0, 0};  // values of a page that holds nothing may be anything
            o[j] = T::mma32(x, pf[kt][g], o[j]);
          }
    };

    if (n0 < n1) {
      Ids ids = settle_ids(ask_ids(n0)), ahead = ask_ids(min(n0 + 1, n1 - 1));
      bring(n0, ids, stage[n0 & 1]);
      Scales next = ask_scales(ids);
      widen(stage[n0 & 1]);
      shared_wait();
      for (int n = n0; n < n1; ++n) {
        const Scales now = next;
        const bool more = n + 1 < n1;
        if (more) {
          ids = settle_ids(ahead);
          bring(n + 1, ids, stage[(n + 1) & 1]);
          next = ask_scales(ids);
          ahead = ask_ids(min(n + 2, n1 - 1));
        }
        if (on) step(stage[n & 1], now);
        if (more) widen(stage[(n + 1) & 1]);
        shared_wait();
      }
    }
    L = across32(L, SumOp());
    if (on && row < rows) {
      const int tok = row / p.group, head = h * p.group + row - tok * p.group;
      const long all = (long)c.tokens * p.heads, at = (long)part * all + (long)(c0 + tok) * p.heads + head;
      if (n0 < n1) {
        float * out = p.ws + at * c.dim;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int ch = 32 * j + 8 * i + 4 * half;
            f4v y = {o[j][4 * i], o[j][4 * i + 1], o[j][4 * i + 2], o[j][4 * i + 3]};
            if (UP) y *= __builtin_ldexpf(1.0f, -UP);
            if (FULL || ch < c.dim) *reinterpret_cast<f4v *>(out + ch) = y;
          }
      }
      if (half == 0) reinterpret_cast<f2v *>(p.ws + p.all_parts * all * c.dim)[at] = f2v{M, L};
    }
  }
}

// 32 rows of a key head, the four waves taking every fourth 32 keys: fragments straight from the cache into registers, in
// the order of shared_attn_kernel's; what the waves have is joined through LDS.  A tile of 16 rows, as the paged attention
// has it, reads the shared keys from L2 twice as often, which bounds it (64 sequences of 4 rows a key head behind 8192
// tokens: 0.27 GB, 11 TB/s).
template <int TYPE, int BITS, int DP, bool FULL> __device__ __forceinline__ void shared_rows(const PagedParams & p, int block, float * lds)
{
  using T = St<TYPE>;
  typedef typename T::e E;
  constexpr int EK = BITS == 8 ? 16 : 8;
  constexpr int KF = DP / (2 * EK), VS = BITS == 8 ? 1 : 2, NB = DP / 32, NS = DP / 16;
  constexpr int UP = TYPE == kSeqF16 ? 7 : BITS == 8 ? 64 : 0;
  const CacheParams & c = p.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  int w = block / kXcds;
  const int slot = w % p.shared_slots;
  w = w / p.shared_slots * kXcds + block % kXcds;
  const int seqs = p.groups * c.heads, part = w / seqs;
  if (part >= p.lead) return;
  w -= part * seqs;
  const int h = w % c.heads;
  const SharedPart own = shared_part(p, w / c.heads, 0);
  if (own.keys == 0) return;
  const int c0 = own.c0, rows = (own.c1 - c0) * p.group;
  const int32_t * table = c.table + (long)own.first * c.width;
  const int lp = 31 - __clz(c.page), last = (own.keys >> lp) - 1;
  const long page_bytes = (long)c.page * c.dim * (BITS / 8);
  const int total = own.keys / 64, per = max(p.shared_steps, (total + p.lead - 1) / p.lead);
  const int t0 = 2 * min(total, part * per), t1 = 2 * min(total, part * per + per);  // 32 keys each
  const float scale = fmaxf(fabsf(p.scale_log2), 1.2e-38f);
  const unsigned flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
  const int mi = col >> 3, mh = col >> 2 & 1, mj = col & 3;
  const int key_gran = BITS == 8 ? mh : mi >> 1, key_quad = BITS == 8 ? mi : 2 * mh + (mi & 1);
  const unsigned key_lane = (unsigned)(key_quad * (c.dim / EK) * 64 + mj * 16), gran_bytes = 16u * c.dim * (BITS / 8);

  auto page_at = [&](int t, int gran) { return table[min((32 * t + 16 * gran) >> lp, last)]; };
  auto valid = [&](int id) { return (unsigned)id < (unsigned)c.pages; };
  auto granule = [&](int id, int t, int gran) {  // its first byte among the keys, or values, of all pages
    return ((long)(valid(id) ? id : 0) * c.heads + h) * page_bytes + ((32 * t + 16 * gran) & (c.page - 1)) / 16 * gran_bytes;
  };

  for (int tile = slot; tile * 32 < rows; tile += p.shared_slots) {
    const int row = tile * 32 + col;
    u4v qf[NS];
    {
      const int there = min(row, rows - 1), tok = there / p.group;
      const E * q = static_cast<const E *>(p.q) + (long)(c0 + tok) * p.q_token + (long)(h * p.group + there - tok * p.group) * p.q_head;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int ch = BITS == 8 ? 16 * (2 * (i / 2) + half) + 8 * (i % 2) : 16 * i + 8 * half;
        qf[i] = *reinterpret_cast<const u4v *>(q + (FULL || ch < c.dim ? ch : 0));
      }
    }
    f16v o[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) o[j] = f16v{};
    float M = kLowest, L = 0.0f;
    u4v kf[KF], vf[VS * NB];
    auto load_k = [&](int t, int id0, int id1) __attribute__((always_inline)) {
      const uint8_t * k = static_cast<const uint8_t *>(c.kc) + granule(key_gran ? id1 : id0, t, key_gran) + key_lane;
#pragma unroll
      for (int i = 0; i < KF; ++i) kf[i] = *reinterpret_cast<const u4v *>(k + (unsigned)(FULL ? 2 * i + half : min(2 * i + half, c.dim / EK - 1)) * 64u);
    };
    float ks = 1.0f, vs = 1.0f;
    auto load_v = [&](int t, int id0, int id1) __attribute__((always_inline)) {
      if constexpr (BITS == 8) {
        const int id = half ? id1 : id0;
        const long page = (long)(valid(id) ? id : 0) * c.heads + h;
        ks = c.ks[page];
        vs = c.vs[page];
        const uint8_t * v = static_cast<const uint8_t *>(c.vc) + granule(id, t, half);
#pragma unroll
        for (int j = 0; j < NB; ++j) vf[j] = *reinterpret_cast<const u4v *>(v + (unsigned)(FULL ? 32 * j + col : min(32 * j + col, c.dim - 1)) * 16u);
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint8_t * v = static_cast<const uint8_t *>(c.vc) + granule(s ? id1 : id0, t, s) + half * c.dim * 16;
#pragma unroll
          for (int j = 0; j < NB; ++j) vf[s * NB + j] = *reinterpret_cast<const u4v *>(v + (unsigned)(FULL ? 32 * j + col : min(32 * j + col, c.dim - 1)) * 16u);
        }
      }
    };
    int id0 = 0, id1 = 0, next0 = 0, next1 = 0;
    int t = t0 + wave;
    if (t < t1) {
      id0 = page_at(t, 0);
      id1 = page_at(t, 1);
      const int ahead = min(t + 4, t1 - 1);
      next0 = page_at(ahead, 0);
      next1 = page_at(ahead, 1);
      load_k(t, id0, id1);
      load_v(t, id0, id1);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int ch = BITS == 8 ? 16 * (2 * (i / 2) + half) + 8 * (i % 2) : 16 * i + 8 * half;
        qf[i] = FULL || ch < c.dim ? qf[i] ^ flip : u4v{0, 0, 0, 0};
      }
    }
    for (; t < t1; t += 4) {
      const bool more = t + 4 < t1;
      f16v s;
#pragma unroll
      for (int i = 0; i < KF; ++i) {
        u4v x = kf[i];
        if (!FULL && (2 * i + half) * EK >= c.dim) x = u4v{0, 0, 0, 0};
        if constexpr (BITS == 8) {
          s = T::mma32(u4v{T::fp8_lo(x[0]), T::fp8_hi(x[0]), T::fp8_lo(x[1]), T::fp8_hi(x[1])}, qf[2 * i], i ? s : f16v{});
          s = T::mma32(u4v{T::fp8_lo(x[2]), T::fp8_hi(x[2]), T::fp8_lo(x[3]), T::fp8_hi(x[3])}, qf[2 * i + 1], s);
        } else {
          s = T::mma32(x, qf[i], i ? s : f16v{});
        }
      }
      const bool ok0 = valid(id0), ok1 = valid(id1), whole = ok0 && ok1;
      float k1 = ks, v1 = BITS == 8 ? fmaxf(vs, 1e-30f) : 1.0f;
      const int after = min(t + 8, t1 - 1);
      if (more) {
        load_k(t + 4, next0, next1);
        id0 = next0;
        id1 = next1;
        next0 = page_at(after, 0);
        next1 = page_at(after, 1);
      }
      if (!whole) {
        if (BITS == 8 && !(half ? ok1 : ok0)) k1 = v1 = 1.0f;
#pragma unroll
        for (int v = 0; v < 16; ++v) s[v] = (BITS == 8 ? (half ? ok1 : ok0) : v < 8 ? ok0 : ok1) ? s[v] : -__builtin_inff();
      }
      const float mul = BITS == 8 ? fmaxf(scale * k1, 1.2e-38f) : scale, ev = BITS == 8 ? __builtin_amdgcn_logf(v1) : 0.0f;
      float a = s[0], d = s[1];
#pragma unroll
      for (int v = 2; v < 16; v += 4) {
        a = top_of(a, s[v], s[v + 1]);
        if (v + 2 < 16) d = top_of(d, s[v + 2], s[v + 3]);
      }
      const float top = across32(fmaf(top_of(a, d, d), mul, ev), MaxOp());
      if (__any(top > M + 8.0f)) {
        const float m = fmaxf(M, top), e = __builtin_amdgcn_exp2f(M - m);
        M = m;
        L *= e;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[j][v] *= e;
      }
      const float shift = ev + UP - M;
      u4v pf[2];
      float sum = 0.0f, sum2 = 0.0f;
#pragma unroll
      for (int v = 0; v < 16; v += 2) {
        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[v], mul, shift)), e1 = __builtin_amdgcn_exp2f(fmaf(s[v + 1], mul, shift));
        const unsigned e = pack2<TYPE>(e0, e1);
        pf[v / 8][v % 8 / 2] = e;
        if (TYPE == kSeqF16 && BITS == 8) {
          sum += e0;
          sum2 += e1;
        } else {
          sum = T::add2(e, sum);
        }
      }
      if (BITS == 8)
        L += __builtin_ldexpf((sum + sum2) * __builtin_amdgcn_rcpf(__builtin_amdgcn_frexp_mantf(v1)), -UP - __builtin_amdgcn_frexp_expf(v1));
      else L = fmaf(sum, __builtin_ldexpf(1.0f, -UP), L);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        u4v x0, x1;
        if constexpr (BITS == 8) {
          u4v x = vf[j];
          if (!whole && !(half ? ok1 : ok0)) x = u4v{0, 0, 0, 0};  // values of a page that holds nothing may be anything
          x0 = u4v{T::fp8_lo(x[0]), T::fp8_hi(x[0]), T::fp8_lo(x[1]), T::fp8_hi(x[1])};
          x1 = u4v{T::fp8_lo(x[2]), T::fp8_hi(x[2]), T::fp8_lo(x[3]), T::fp8_hi(x[3])};
        } else {
          x0 = ok0 ? vf[j] : u4v{0, 0, 0, 0};
          x1 = ok1 ? vf[NB + j] : u4v{0, 0, 0, 0};
        }
        o[j] = T::mma32(x0, pf[0], o[j]);
        o[j] = T::mma32(x1, pf[1], o[j]);
      }
      if (more) load_v(t + 4, id0, id1);
    }
    L = across32(L, SumOp());

    // ---- the waves' sums are joined as in paged_attn.hpp
    constexpr int PITCH = DP + 4;
    f2v * ml = reinterpret_cast<f2v *>(lds + 2 * 32 * PITCH);
#pragma unroll
    for (int hw = 2; hw >= 1; hw /= 2) {
      float * mine = lds + (wave % hw) * 32 * PITCH + col * PITCH + 4 * half;
      __syncthreads();
      if (wave >= hw && wave < 2 * hw) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f4v y = {o[j][4 * i], o[j][4 * i + 1], o[j][4 * i + 2], o[j][4 * i + 3]};
            *reinterpret_cast<f4v *>(mine + 32 * j + 8 * i) = y;
          }
        if (half == 0) ml[(wave % hw) * 32 + col] = f2v{M, L};
      }
      __syncthreads();
      if (wave < hw) {
        const f2v y = ml[wave * 32 + col];
        const float m = fmaxf(M, y[0]), a = __builtin_amdgcn_exp2f(M - m), e = __builtin_amdgcn_exp2f(y[0] - m);
        M = m;
        L = L * a + y[1] * e;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f4v x = *reinterpret_cast<const f4v *>(mine + 32 * j + 8 * i);
#pragma unroll
            for (int v = 0; v < 4; ++v) o[j][4 * i + v] = o[j][4 * i + v] * a + x[v] * e;
          }
      }
    }
    if (wave == 0 && row < rows) {
      const int tok = row / p.group, head = h * p.group + row - tok * p.group;
      const long all = (long)c.tokens * p.heads, at = (long)part * all + (long)(c0 + tok) * p.heads + head;
      if (t0 < t1) {
        float * out = p.ws + at * c.dim;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int ch = 32 * j + 8 * i + 4 * half;
            f4v y = {o[j][4 * i], o[j][4 * i + 1], o[j][4 * i + 2], o[j][4 * i + 3]};
            if (UP) y *= __builtin_ldexpf(1.0f, -UP);
            if (FULL || ch < c.dim) *reinterpret_cast<f4v *>(out + ch) = y;
          }
      }
      if (half == 0) reinterpret_cast<f2v *>(p.ws + p.all_parts * all * c.dim)[at] = f2v{M, L};
    }
    __syncthreads();  // LDS is read before the next tile's waves write it
  }
}

namespace {

template <int TYPE, int BITS, int DP, bool FULL> void launch_shared(const PagedParams & p, hipStream_t s)
{
  const dim3 grid((unsigned)paged_wgs(p, p.groups));
  hipLaunchKernelGGL((shared_attn_kernel<TYPE, BITS, DP, FULL>), grid, dim3(256), 0, s, p, p.groups * p.c.heads * p.parts);
}

template <int TYPE, int BITS> void launch_shared_dim(const PagedParams & p, hipStream_t s)
{
  if (p.c.dim == 64) launch_shared<TYPE, BITS, 64, true>(p, s);
  else launch_shared<TYPE, BITS, 64, false>(p, s);
}

template <int TYPE, int BITS> void launch_prefix_keys(const PrefixParams & p, hipStream_t s)
{
  if (p.both) {
    if (p.wide) launch_paged_dim<TYPE, BITS, kBothWide>(p.own, s);
    else launch_paged_dim<TYPE, BITS, kBothKeys>(p.own, s);
    return;
  }
  if (p.own.lead > 0) {
    if (p.many) launch_shared_dim<TYPE, BITS>(p.first, s);
    else launch_paged_dim<TYPE, BITS, kSharedKeys>(p.first, s);
  }
  launch_paged_dim<TYPE, BITS, kOwnKeys>(p.own, s);
}

template <int TYPE> void launch_prefix_type(const PrefixParams & p, hipStream_t s)
{
  if (p.own.c.bits == 8) launch_prefix_keys<TYPE, 8>(p, s);
  else launch_prefix_keys<TYPE, 16>(p, s);
  PagedParams join = p.own;
  join.parts = p.own.all_parts;
  launch_paged_join<TYPE>(join, s);
}

}  // namespace

}  // namespace ivh
