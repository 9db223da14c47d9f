// Rotary positions with several axes, and the append of rotated keys and of values to a paged
// cache, on gfx950.
//
// Rotation: a head's frequency f turns the pair (a, b) of its channels (f, f + rot / 2) or
// (2f, 2f + 1) by the angle t = pos[axis(f)][token] * freq[f]:
//   a' = a cos t - b sin t,   b' = b cos t + a sin t
// in fp32, rounded once.  Both kernels move every channel once and do three multiply-adds on it,
// so the memory bounds them; the angles (a 64-bit product and a sine each) are the one thing that
// can cost more and are shared by a token's heads.
#include <algorithm>
#include <stdexcept>

#include "conv_common.hpp"
#include "seq_common.hpp"

namespace ivh {

namespace {

template <int N> struct Pack;  // N 16-bit values
template <> struct Pack<4> { typedef u2v t; };
template <> struct Pack<8> { typedef u4v t; };

struct RopeGeo {
  int hg;         // head groups: a thread takes heads g, g + hg, ..
  int pieces;     // 2 VEC-channel pieces of a head
  int rotating;   // of those, the ones that turn; the others are copied
  FastDiv dv_pieces, dv_hg;
  unsigned total; // tokens x hg x pieces
  int copy;       // the others have to be copied (not in place)
};

}  // namespace

// A thread owns 2 VEC channels (16 or 32 bytes) of a token in every hg-th head: it forms their
// VEC angles once and walks the heads; neighbouring threads hold neighbouring pieces, so each step of the walk reads
// and writes whole lines.
template <int TYPE, int VEC, bool ADJ>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p, const RopeGeo g)
{
  typedef typename St<TYPE>::e E;
  typedef typename Pack<VEC>::t V;
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= g.total) return;
  const unsigned row = fastdiv(idx, g.dv_pieces), piece = idx - row * g.pieces;
  const unsigned token = fastdiv(row, g.dv_hg), grp = row - token * g.hg;
  const bool turn = (int)piece < g.rotating;
  if (!turn && !g.copy) return;
  int lo, hi;  // the piece's two runs of VEC channels
  if (!turn) {
    lo = p.r.rot + 2 * VEC * (piece - g.rotating);
    hi = lo + VEC;
  } else if (ADJ) {
    lo = 2 * VEC * piece;
    hi = lo + VEC;
  } else {
    lo = VEC * piece;
    hi = p.r.half + lo;
  }
  float c[VEC], s[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    c[i] = 1.0f;
    s[i] = 0.0f;
  }
  if (turn) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int f = VEC * piece + i;
      const f2v cs = rot_cossin(p.r.pos[rot_axis(p.r, f) * p.r.pos_axis + token], p.r.freq[f]);
      c[i] = cs[0];
      s[i] = cs[1];
    }
  }
  const E * x = static_cast<const E *>(p.x) + (long)token * p.x_token;
  E * y = static_cast<E *>(p.y) + (long)token * p.y_token;
#pragma unroll 4
  for (int h = grp; h < p.heads; h += g.hg) {
    V a = *reinterpret_cast<const V *>(x + (long)h * p.x_head + lo);
    V b = *reinterpret_cast<const V *>(x + (long)h * p.x_head + hi);
    if (turn) {
      if (ADJ) {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const f2v u = unpack2<TYPE>(a[i]), w = unpack2<TYPE>(b[i]);
          const int j = i + VEC / 2;
          a[i] = pack2<TYPE>(u[0] * c[i] - u[1] * s[i], u[1] * c[i] + u[0] * s[i]);
          b[i] = pack2<TYPE>(w[0] * c[j] - w[1] * s[j], w[1] * c[j] + w[0] * s[j]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const f2v u = unpack2<TYPE>(a[i]), w = unpack2<TYPE>(b[i]);
          const int j = 2 * i;
          a[i] = pack2<TYPE>(u[0] * c[j] - w[0] * s[j], u[1] * c[j + 1] - w[1] * s[j + 1]);
          b[i] = pack2<TYPE>(w[0] * c[j] + u[0] * s[j], w[1] * c[j + 1] + u[1] * s[j + 1]);
        }
      }
    }
    *reinterpret_cast<V *>(y + (long)h * p.y_head + lo) = a;
    *reinterpret_cast<V *>(y + (long)h * p.y_head + hi) = b;
  }
}

namespace {

bool aligned(const void * ptr, long a, long b, int elems)
{
  return reinterpret_cast<uintptr_t>(ptr) % (2 * elems) == 0 && a % elems == 0 && b % elems == 0;
}

template <int TYPE, int VEC> void launch_rope_vec(const RopeParams & p, hipStream_t s)
{
  const bool same = p.x == p.y && p.x_token == p.y_token && p.x_head == p.y_head;
  RopeGeo g;
  g.pieces = p.dim / (2 * VEC);
  g.rotating = p.r.rot / (2 * VEC);
  g.copy = !same;
  // one head a thread until the chip is full (256 CUs x 2048 lanes), then up to 8 that share the angles
  const long lanes = p.tokens * g.pieces * p.heads;
  g.hg = lanes <= (1L << 20) ? p.heads : (p.heads + 7) / 8;
  g.dv_pieces = fastdiv_make(g.pieces);
  g.dv_hg = fastdiv_make(g.hg);
  // slices of tokens, so that a launch's lanes stay below 2^31
  const long per = std::max<long>(1, (1L << 30) / ((long)g.pieces * g.hg));
  for (long t0 = 0; t0 < p.tokens; t0 += per) {
    RopeParams q = p;
    q.tokens = std::min(per, p.tokens - t0);
    q.x = static_cast<const uint16_t *>(p.x) + t0 * p.x_token;
    q.y = static_cast<uint16_t *>(p.y) + t0 * p.y_token;
    if (q.r.pos) q.r.pos += t0;
    g.total = (unsigned)(q.tokens * g.hg * g.pieces);
    const dim3 grid((g.total + 255) / 256), blk(256);
    if (p.r.adjacent) hipLaunchKernelGGL((rope_kernel<TYPE, VEC, true>), grid, blk, 0, s, q, g);
    else hipLaunchKernelGGL((rope_kernel<TYPE, VEC, false>), grid, blk, 0, s, q, g);
  }
}

}  // namespace

void launch_rope(const RopeParams & p, hipStream_t s)
{
  // 16-byte runs where the halves, the copied rest and the rows allow them, else 8-byte ones
  const bool wide = p.r.rot % 16 == 0 && p.dim % 16 == 0 && aligned(p.x, p.x_token, p.x_head, 8) &&
                    aligned(p.y, p.y_token, p.y_head, 8);
  if (p.type == kSeqF16) wide ? launch_rope_vec<kSeqF16, 8>(p, s) : launch_rope_vec<kSeqF16, 4>(p, s);
  else wide ? launch_rope_vec<kSeqBF16, 8>(p, s) : launch_rope_vec<kSeqBF16, 4>(p, s);
}

// ---------------------------------------------------------------- append to a paged cache
//
// A work-group owns one (sequence, page that gets new tokens, head) and either its keys or its
// values; pages are found on the device from the sequences' lengths.  Sequence b's pages are
// numbered from cu[b] / page + 2 b: n new tokens touch at most n / page + 2 pages, so the ranges
// do not overlap and tokens / page + 2 batch work-groups cover them, without a scan or the host
// knowing the lengths.
//
// 8-bit pages have one scale for a page and head: the smallest power of two s with
// max |x| <= 448 s (448 is e4m3's largest value), at least 2^-32, and no smaller than the scale of
// older tokens in the page.  When that grows, the page's other codes (older tokens' and whatever
// its empty slots hold) are rounded to the new scale; as a power of two it leaves their mantissas alone, so that they only lose
// the bits that fall below e4m3's last place.
// The new values wait in registers for the page's maximum: each input is read once.

namespace {

constexpr float kMaxCode = 448.0f, kLowestScale = 2.3283064365386963e-10f;  // 2^-32

struct PageWork {
  int row0;        // first row of the page's new tokens in k, v
  int lo, hi;      // its slots: new ones are [lo, hi), older ones [0, lo)
  long base;       // page x heads, for pages and scales
};

// Page w of the numbering above; false: none, or a page number outside the cache.
__device__ __forceinline__ bool page_work(const CacheParams & c, int w, PageWork & o)
{
  const int * cu = c.cu;
  const int tokens = c.tokens, page = c.page;
  auto start = [&](int b) { return (long)(min(max(cu[b], 0), tokens) / page) + 2L * b; };
  const int b = __builtin_amdgcn_readfirstlane(find_seq(c.batch, w, start));
  const int c0 = min(max(cu[b], 0), tokens), c1 = min(max(cu[b + 1], c0), tokens);
  const long old = (long)c.lens[b] - (c1 - c0);  // place of the first new token; below 0: not stored
  const long first = (old > 0 ? old : 0) / page;
  const long at = first + (w - start(b));
  if (at < first || at >= c.width) return false;
  const long lo = max(old, at * page), hi = min((long)c.lens[b], (at + 1) * page);
  if (lo >= hi) return false;
  const int id = c.table[(long)b * c.width + at];
  if ((unsigned)id >= (unsigned)c.pages) return false;
  o.row0 = c0 + (int)(lo - old);
  o.lo = (int)(lo - at * page);
  o.hi = (int)(hi - at * page);
  o.base = (long)id * c.heads;
  return true;
}

__device__ __forceinline__ float finite_abs(float x)
{
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.0f;  // infinities and NaN have no part in a scale
}

// the smallest power of two s with amax <= 448 s = 1.75 x 2^8 s, from the bits of amax
__device__ __forceinline__ float page_scale(float amax)
{
  if (amax < kLowestScale) return kLowestScale;
  const unsigned u = __builtin_bit_cast(unsigned, amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
  return fmaxf(__builtin_bit_cast(float, (unsigned)max(e, 1) << 23), kLowestScale);
}

// e4m3 codes of four values of the page's scale: nearest, ties to even; infinities become the
// largest value, NaN stays NaN
__device__ __forceinline__ float clamp_code(float x)
{
  x = x > kMaxCode ? kMaxCode : x;
  return x < -kMaxCode ? -kMaxCode : x;
}
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d)
{
  unsigned r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_code(a), clamp_code(b), 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(clamp_code(c), clamp_code(d), r, true);
}
__device__ __forceinline__ unsigned rescale4(unsigned x, float ratio)
{
  const f2v a = __builtin_amdgcn_cvt_pk_f32_fp8(x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(x, true);
  return codes4(a[0] * ratio, a[1] * ratio, b[0] * ratio, b[1] * ratio);
}

// maximum over the work-group, and the page's new scale
__device__ __forceinline__ float group_scale(float amax, float old, float * red)
{
  for (int m = 1; m < 64; m *= 2) amax = fmaxf(amax, __shfl_xor(amax, m));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  return fmaxf(page_scale(amax), old);
}

}  // namespace

// Keys.  A thread owns a token's 16 bytes of the stored page (EK channels), U of them: the
// channels' partners come from a second read that hits the cache, and a granule's tokens times
// frequencies of cosines and sines from LDS.
template <int TYPE, int BITS, int U>
__device__ __forceinline__ void append_keys(const AppendParams & p, const PageWork & w, int h, float * red, f2v * cs)
{
  typedef typename St<TYPE>::e E;
  constexpr int EK = BITS == 8 ? 16 : 8, Q = EK / 4;
  const CacheParams & c = p.c;
  const RotParams & r = p.r;
  const int tid = threadIdx.x, chunks = c.dim / EK, n = w.hi - w.lo;
  const int rot = r.rot, half = r.half;
  for (int i = tid; i < n * half; i += 256) {
    const int t = i / half, f = i - t * half;
    cs[i] = rot_cossin(r.pos[rot_axis(r, f) * r.pos_axis + w.row0 + t], r.freq[f]);
  }
  __syncthreads();
  const E * src = static_cast<const E *>(p.k) + (long)h * p.k_head;
  uint8_t * dst = static_cast<uint8_t *>(c.kc) + (w.base + h) * ((long)c.page * c.dim * (BITS / 8));
  auto place = [&](int slot, int ch) { return ((slot / 4 * chunks + ch) * 4 + slot % 4) * 16; };
  float v[U][EK];
  float amax = 0.0f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = tid + 256 * u, t = i / chunks, ch = i - t * chunks;
    if (i >= n * chunks) continue;
    const E * row = src + (long)(w.row0 + t) * p.k_token;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int m = ch * EK + 4 * q;  // rot and half are multiples of 4: a run of 4 has one kind
      const u2v own = *reinterpret_cast<const u2v *>(row + m);
      const f2v a = unpack2<TYPE>(own[0]), b = unpack2<TYPE>(own[1]);
      float * o = v[u] + 4 * q;
      if (m >= rot) {
        o[0] = a[0]; o[1] = a[1]; o[2] = b[0]; o[3] = b[1];
      } else if (r.adjacent) {
        const f2v c0 = cs[t * half + m / 2], c1 = cs[t * half + m / 2 + 1];
        o[0] = a[0] * c0[0] - a[1] * c0[1]; o[1] = a[1] * c0[0] + a[0] * c0[1];
        o[2] = b[0] * c1[0] - b[1] * c1[1]; o[3] = b[1] * c1[0] + b[0] * c1[1];
      } else {
        const bool first = m < half;
        const u2v other = *reinterpret_cast<const u2v *>(row + (first ? m + half : m - half));
        const f2v d = unpack2<TYPE>(other[0]), e = unpack2<TYPE>(other[1]);
        const f2v * t4 = cs + t * half + (first ? m : m - half);
        const float g = first ? -1.0f : 1.0f;
        o[0] = a[0] * t4[0][0] + g * (d[0] * t4[0][1]); o[1] = a[1] * t4[1][0] + g * (d[1] * t4[1][1]);
        o[2] = b[0] * t4[2][0] + g * (e[0] * t4[2][1]); o[3] = b[1] * t4[3][0] + g * (e[1] * t4[3][1]);
      }
    }
    if (BITS == 8) {
#pragma unroll
      for (int k = 0; k < EK; ++k) amax = fmaxf(amax, finite_abs(v[u][k]));
    } else {
      const u4v y = {pack2<TYPE>(v[u][0], v[u][1]), pack2<TYPE>(v[u][2], v[u][3]), pack2<TYPE>(v[u][4], v[u][5]),
                     pack2<TYPE>(v[u][6], v[u][7])};
      *reinterpret_cast<u4v *>(dst + place(w.lo + t, ch)) = y;
    }
  }
  if constexpr (BITS == 8) {
    const float before = w.lo ? c.ks[w.base + h] : 0.0f;
    const float s = group_scale(amax, before, red), inv = 1.0f / s;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid + 256 * u, t = i / chunks, ch = i - t * chunks;
      if (i >= n * chunks) continue;
      u4v y;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        y[q] = codes4(v[u][4 * q] * inv, v[u][4 * q + 1] * inv, v[u][4 * q + 2] * inv, v[u][4 * q + 3] * inv);
      *reinterpret_cast<u4v *>(dst + place(w.lo + t, ch)) = y;
    }
    if (w.lo && before != s) {
      const float ratio = before * inv;
      for (int i = tid; i < (c.page - n) * chunks; i += 256) {
        const int t = i / chunks;
        u4v * at = reinterpret_cast<u4v *>(dst + place(t < w.lo ? t : t + n, i - t * chunks));
        u4v y = *at;
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = rescale4(y[q], ratio);
        *at = y;
      }
    }
    if (tid == 0) c.ks[w.base + h] = s;
  }
}

// Values.  A thread owns two channels of EV tokens (a granule), 2 x 16 bytes side by side in the
// stored page, U of them.
template <int TYPE, int BITS, int U>
__device__ __forceinline__ void append_values(const AppendParams & p, const PageWork & w, int h, float * red)
{
  typedef typename St<TYPE>::e E;
  constexpr int EV = BITS == 8 ? 16 : 8;
  const CacheParams & c = p.c;
  const int tid = threadIdx.x, pairs = c.dim / 2;
  const int g0 = w.lo / EV, work = ((w.hi + EV - 1) / EV - g0) * pairs;  // granules with new tokens
  const E * src = static_cast<const E *>(p.v) + (long)h * p.v_head;
  uint8_t * dst = static_cast<uint8_t *>(c.vc) + (w.base + h) * ((long)c.page * c.dim * (BITS / 8));
  unsigned x[U][EV];
  float amax = 0.0f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = tid + 256 * u, g = i / pairs, ch = 2 * (i - g * pairs), slot0 = (g0 + g) * EV;
    if (i >= work) continue;
#pragma unroll
    for (int t = 0; t < EV; ++t) {
      const int slot = slot0 + t;
      const bool fresh = slot >= w.lo && slot < w.hi;
      x[u][t] = fresh ? *reinterpret_cast<const unsigned *>(src + (long)(w.row0 + slot - w.lo) * p.v_token + ch) : 0u;
    }
    if (BITS == 8) {
#pragma unroll
      for (int t = 0; t < EV; ++t) {
        const f2v a = unpack2<TYPE>(x[u][t]);
        amax = fmaxf(amax, fmaxf(finite_abs(a[0]), finite_abs(a[1])));
      }
    } else {
      u4v * at = reinterpret_cast<u4v *>(dst + ((long)(g0 + g) * c.dim + ch) * 16);
      u4v y0, y1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // two tokens of one channel, then of the next
        y0[q] = (x[u][2 * q] & 0xffffu) | (x[u][2 * q + 1] << 16);
        y1[q] = (x[u][2 * q] >> 16) | (x[u][2 * q + 1] & 0xffff0000u);
      }
      if (slot0 < w.lo || slot0 + EV > w.hi) {  // older tokens and slots behind the last one stay
        const u4v z0 = at[0], z1 = at[1];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const unsigned m = (slot0 + 2 * q >= w.lo && slot0 + 2 * q < w.hi ? 0xffffu : 0u) |
                             (slot0 + 2 * q + 1 >= w.lo && slot0 + 2 * q + 1 < w.hi ? 0xffff0000u : 0u);
          y0[q] = (y0[q] & m) | (z0[q] & ~m);
          y1[q] = (y1[q] & m) | (z1[q] & ~m);
        }
      }
      at[0] = y0;
      at[1] = y1;
    }
  }
  if constexpr (BITS == 8) {
    const float before = w.lo ? c.vs[w.base + h] : 0.0f;
    const float s = group_scale(amax, before, red), inv = 1.0f / s;
    const bool grown = w.lo && before != s;
    const float ratio = before * inv;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid + 256 * u, g = i / pairs, ch = 2 * (i - g * pairs), slot0 = (g0 + g) * EV;
      if (i >= work) continue;
      u4v * at = reinterpret_cast<u4v *>(dst + ((long)(g0 + g) * c.dim + ch) * 16);
      u4v y0, y1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f2v a = unpack2<TYPE>(x[u][4 * q]), b = unpack2<TYPE>(x[u][4 * q + 1]);
        const f2v d = unpack2<TYPE>(x[u][4 * q + 2]), e = unpack2<TYPE>(x[u][4 * q + 3]);
        y0[q] = codes4(a[0] * inv, b[0] * inv, d[0] * inv, e[0] * inv);
        y1[q] = codes4(a[1] * inv, b[1] * inv, d[1] * inv, e[1] * inv);
      }
      if (slot0 < w.lo || slot0 + EV > w.hi) {
        const u4v z0 = at[0], z1 = at[1];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          unsigned fresh = 0;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int slot = slot0 + 4 * q + t;
            if (slot >= w.lo && slot < w.hi) fresh |= 0xffu << (8 * t);
          }
          const unsigned o0 = grown ? rescale4(z0[q], ratio) : z0[q], o1 = grown ? rescale4(z1[q], ratio) : z1[q];
          y0[q] = (y0[q] & fresh) | (o0 & ~fresh);
          y1[q] = (y1[q] & fresh) | (o1 & ~fresh);
        }
      }
      at[0] = y0;
      at[1] = y1;
    }
    if (grown) {  // the granules without new tokens
      const int some = (w.hi + EV - 1) / EV - g0;
      for (int i = tid; i < (c.page / EV - some) * c.dim; i += 256) {
        u4v * at = reinterpret_cast<u4v *>(dst + (long)(i < g0 * c.dim ? i : i + some * c.dim) * 16);
        u4v y = *at;
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = rescale4(y[q], ratio);
        *at = y;
      }
    }
    if (tid == 0) c.vs[w.base + h] = s;
  }
}

// UK, UV: 16-byte pieces of keys and 32-byte pieces of values a thread holds of a whole page.
template <int TYPE, int BITS, int UK, int UV>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p)
{
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ float red[4];
  PageWork w;
  if (!page_work(p.c, blockIdx.x, w)) return;
  if (blockIdx.z == 0) append_keys<TYPE, BITS, UK>(p, w, blockIdx.y, red, reinterpret_cast<f2v *>(lds));
  else append_values<TYPE, BITS, UV>(p, w, blockIdx.y, red);
}

namespace {

template <int TYPE, int BITS> void launch_append(const AppendParams & p, hipStream_t s)
{
  const CacheParams & c = p.c;
  const dim3 grid((unsigned)((long)c.tokens / c.page + 2L * c.batch), c.heads, 2), blk(256);
  const size_t lds = (size_t)c.page * p.r.half * sizeof(f2v);
  const int E = BITS == 8 ? 16 : 8;
  const int need = (int)std::max<long>(1, ((long)c.page * c.dim / E + 255) / 256);  // pieces a thread
  auto go = [&](auto kern) {
    if (lds > 65536) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) throw std::runtime_error(std::string("HIP error: ") + hipGetErrorString(e));
    }
    hipLaunchKernelGGL(kern, grid, blk, lds, s, p);
  };
  // a value piece is two channels of a granule: half as many as key pieces
  if (need <= 1) go(kv_append_kernel<TYPE, BITS, 1, 1>);
  else if (need <= 2) go(kv_append_kernel<TYPE, BITS, 2, 1>);
  else if (need <= 4) go(kv_append_kernel<TYPE, BITS, 4, 2>);
  else if (need <= 8) go(kv_append_kernel<TYPE, BITS, 8, 4>);
  else go(kv_append_kernel<TYPE, BITS, 16, 8>);
}

}  // namespace

void launch_kv_append(const AppendParams & p, hipStream_t s)
{
  const bool f16 = p.c.type == kSeqF16;
  if (p.c.bits == 8) f16 ? launch_append<kSeqF16, 8>(p, s) : launch_append<kSeqBF16, 8>(p, s);
  else f16 ? launch_append<kSeqF16, 16>(p, s) : launch_append<kSeqBF16, 16>(p, s);
}

}  // namespace ivh
