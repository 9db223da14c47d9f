// Attention over a paged cache whose first pages the sequences of a group share, on gfx950 MFMA.
//
//   o[i] = (e^(m1 - m) o1 + e^(m2 - m) o2) / (e^(m1 - m) l1 + e^(m2 - m) l2),  m = max(m1, m2)
//
// with (m1, l1, o1) the maximum, sum and weighted values over the group's shared keys and (m2, l2, o2) those over
// the sequence's own: the shared keys are read once for the rows of all sequences, which are contiguous.
// Shared keys, own keys, and the join of all parts.  Own keys, and shared ones with few rows, take
// the paged attention's kernel; with many rows the matrix cores bound the shared keys:
//   * a work-group has 128 rows of a key head, a wave 32 of them, and walks 64 keys a step.  The steps' keys and values
//     stand in LDS in two stages, in 16 bits, each 1024 bytes a fragment of 32 x 32 x 16 MFMA in the order of its lanes: they are
//     read without a bank conflict, and 8-bit codes are widened once for the four waves;
//   * S^T = K Q^T with keys in rows in an order of which a lane holds, of a 32-key part, the 16 keys of one granule
//     (8-bit pages) or two runs of 8 (16-bit): they are operands of O^T = V^T P^T as they are;
//   * weights, running maxima and scales as in paged_attn.hpp; nothing is masked but pages that hold nothing.
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

// DP: head size rounded up to 64, 128 or 256; FULL: it is that size.
template <int TYPE, int BITS, int DP, bool FULL>
__global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) shared_attn_kernel(const PagedParams p, int units)
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
  const SharedPart own = shared_part(p, w / c.heads);
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

namespace {

template <int TYPE, int BITS, int DP, bool FULL> void launch_shared(const PagedParams & p, hipStream_t s)
{
  const long units = (long)p.groups * p.c.heads * p.parts;
  const dim3 grid((unsigned)((units + kXcds - 1) / kXcds * kXcds * p.row_slots));
  hipLaunchKernelGGL((shared_attn_kernel<TYPE, BITS, DP, FULL>), grid, dim3(256), 0, s, p, (int)units);
}

template <int TYPE, int BITS> void launch_shared_dim(const PagedParams & p, hipStream_t s)
{
  if (p.c.dim == 64) launch_shared<TYPE, BITS, 64, true>(p, s);
  else if (p.c.dim < 64) launch_shared<TYPE, BITS, 64, false>(p, s);
  else if (p.c.dim == 128) launch_shared<TYPE, BITS, 128, true>(p, s);
  else if (p.c.dim < 128) launch_shared<TYPE, BITS, 128, false>(p, s);
  else if (p.c.dim == 256) launch_shared<TYPE, BITS, 256, true>(p, s);
  else launch_shared<TYPE, BITS, 256, false>(p, s);
}

template <int TYPE, int BITS> void launch_prefix_keys(const PrefixParams & p, hipStream_t s)
{
  if (p.both) {
    launch_paged_dim<TYPE, BITS, kBothKeys>(p.own, s);
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
