// Rotary positions with several axes, and the append of rotated keys and of values to a paged
// cache, on gfx950.
//
// Rotation: a head's frequency f turns the pair (a, b) of its channels (f, f + rot / 2) or
// (2f, 2f + 1) by the angle t = pos[axis(f)][token] * freq[f]:
//   a' = a cos t - b sin t,   b' = b cos t + a sin t
// in fp32, rounded once.  Both kernels move every channel once and do three multiply-adds on it,
// so the memory bounds them; the angles (a two-part product and some 30 operations each) are the one
// thing that can cost more and are shared by a token's heads.
//
// Measured (a 1 GiB copy reaches 5.2 TB/s here): 32768 tokens of 40 heads of 128 channels, bf16,
// three axes: 135 us, 5.0 TB/s.  6400 tokens of 32 heads of 80 channels cut from packed rows 14.9 us,
// 4.4 TB/s.  One token: 4 us, launch and two trips to memory.
//
// The append gives a work-group a page (or the part of it that is new) of a run of heads, keys
// and values apart: a page's scale needs the page's maximum, so the rows wait in registers while it
// is found.  20033 tokens of 8 heads of 128 channels into an 8-bit cache: 37 us, 3.3 TB/s, held by the
// chain of rows, maximum, codes with three work-groups a CU; the same in 16 bits, 7000 tokens of 4 heads
// of 256 channels, 13 us.  A token each of 60 sequences: 5.6 us, the chain of offsets, table, rows.
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
      const f2v cs = rot_cossin(p.r.pos[rot_axis(p.r, f) * p.r.pos_axis + token], p.r.freq[f], rot_turns(p.r.freq[f]));
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
  // a thread's heads share its angles: as many as leave two waves a SIMD, up to 8 (6400 tokens of 32
  // heads of 80 channels: 16 us, with four waves a SIMD 18, with one head a thread 25)
  const long lanes = p.tokens * g.pieces * p.heads;
  const int per_thread = (int)std::min<long>({8, std::max<long>(1, lanes >> 17), p.heads});
  g.hg = (p.heads + per_thread - 1) / per_thread;
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
  auto start = [&](int b, int first) { return (long)(min(max(first, 0), tokens) / page) + 2L * b; };
  int b, c0, c1, len;
  if (c.batch < 64) {  // all sequences at once, a lane each: one trip to memory instead of two
    const int lane = threadIdx.x & 63, x = cu[min(lane, c.batch)], y = c.lens[min(lane, c.batch - 1)];
    const unsigned long long below = __ballot(lane < c.batch && start(lane, x) <= w);
    b = below ? 63 - __clzll(below) : 0;
    c0 = __builtin_amdgcn_readlane(x, b);
    c1 = __builtin_amdgcn_readlane(x, b + 1);
    len = __builtin_amdgcn_readlane(y, b);
  } else {
    b = __builtin_amdgcn_readfirstlane(find_seq(c.batch, w, [&](int i) { return start(i, cu[i]); }));
    c0 = cu[b];
    c1 = cu[b + 1];
    len = c.lens[b];
  }
  c0 = min(max(c0, 0), tokens);
  c1 = min(max(c1, c0), tokens);
  const long old = (long)len - (c1 - c0);  // place of the first new token; below 0: not stored
  const long first = (old > 0 ? old : 0) / page;
  const long at = first + (w - start(b, c0));
  if (at < first || at >= c.width) return false;
  const long lo = max(old, at * page), hi = min((long)len, (at + 1) * page);
  if (lo >= hi) return false;
  const int id = c.table[(long)b * c.width + at];
  if ((unsigned)id >= (unsigned)c.pages) return false;
  o.row0 = c0 + (int)(lo - old);
  o.lo = (int)(lo - at * page);
  o.hi = (int)(hi - at * page);
  o.base = (long)id * c.heads;
  return true;
}

// the smallest power of two s with amax <= 448 s = 1.75 x 2^8 s, from the bits of amax
__device__ __forceinline__ float page_scale(float amax)
{
  if (amax < kLowestScale) return kLowestScale;
  const unsigned u = __builtin_bit_cast(unsigned, amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
  return fmaxf(__builtin_bit_cast(float, (unsigned)max(e, 1) << 23), kLowestScale);
}

// e4m3 codes of four values in units of the page's scale, nearest, ties to even; NaN stays NaN
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d)
{
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}
__device__ __forceinline__ unsigned rescale4(unsigned x, float ratio)
{
  const f2v a = __builtin_amdgcn_cvt_pk_f32_fp8(x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(x, true);
  return codes4(a[0] * ratio, a[1] * ratio, b[0] * ratio, b[1] * ratio);
}

// maximum over the work-group
template <int NT> __device__ __forceinline__ float group_max(float amax, float * red)
{
  for (int m = 1; m < 64; m *= 2) amax = fmaxf(amax, __shfl_xor(amax, m));
  if (NT == 64) return amax;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// The page's new scale; amax: this thread's largest magnitude.  If there is an infinity among the
// work-group's values (all of its threads see that), `finite` gives the thread's largest finite one, and
// saturate is set: infinities are to become the largest code.  A NaN is passed over by the maximum.
template <int NT, class Fn>
__device__ __forceinline__ float group_scale(float amax, float before, float (*red)[4], bool & saturate, Fn && finite)
{
  amax = group_max<NT>(amax, red[0]);
  saturate = !(amax < __builtin_inff());
  if (saturate) amax = group_max<NT>(finite(), red[2]);
  return fmaxf(page_scale(amax), before);
}
__device__ __forceinline__ float finite_abs(float x)
{
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.0f;
}
__device__ __forceinline__ float saturated(float x)
{
  x = x > kMaxCode ? kMaxCode : x;
  return x < -kMaxCode ? -kMaxCode : x;
}

}  // namespace

// Cosines and sines of the page's new tokens in LDS, two planes [token][pitch] of 16-byte runs of 4
// frequencies.  A thread reads Q runs that follow each other, its neighbour the Q after: runs are
// stored with the neighbours' side by side and a pitch of 2 mod 8 runs, so that the lanes that are
// served together lie in distinct banks.
template <int Q> struct AngleTable {
  int lots, pitch;
  static __host__ __device__ int lots_of(int half) { return (half / 4 + Q - 1) / Q; }
  static __host__ __device__ int pitch_of(int half) { return (Q * lots_of(half) + 5) / 8 * 8 + 2; }
  __device__ __forceinline__ AngleTable(int half) : lots(lots_of(half)), pitch(pitch_of(half)) {}
  __device__ __forceinline__ int at(int t, int f) const { return (t * pitch + f / 4 % Q * lots + f / 4 / Q) * 4 + f % 4; }
};

template <int NT, int Q>
__device__ __forceinline__ void page_angles(const RotParams & r, const PageWork & w, float * cos, float * sin)
{
  const AngleTable<Q> table(r.half);
  const int per = NT / r.half, t0 = threadIdx.x / r.half, f = threadIdx.x - t0 * r.half, n = w.hi - w.lo;
  if (t0 >= per) return;
  const float freq = r.freq[f];
  const f2v turns = rot_turns(freq);
  const int32_t * pos = r.pos + rot_axis(r, f) * r.pos_axis + w.row0;
  for (int t = t0; t < n; t += per) {
    const f2v cs = rot_cossin(pos[t], freq, turns);
    cos[table.at(t, f)] = cs[0];
    sin[table.at(t, f)] = cs[1];
  }
}

// Keys of heads [h0, h1).  A thread owns two runs of R channels of a token whose pairs lie within the
// two: channels f.. and rot / 2 + f.., or 2 R in a row (adjacent pairs, and what is not rotated); U such
// units.  The next head's rows are asked for as soon as this one's are turned.
template <int TYPE, int BITS, int NT, int R, int U>
__device__ __forceinline__ void append_keys(const AppendParams & p, const PageWork & w, int h0, int h1, float (*red)[4], float * cos,
                                            float * sin)
{
  typedef typename St<TYPE>::e E;
  constexpr int EK = BITS == 8 ? 16 : 8, Q = R / 4;
  const CacheParams & c = p.c;
  const RotParams & r = p.r;
  const int units = c.dim / (2 * R), chunks = c.dim / EK, n = w.hi - w.lo;
  const int per = NT / units, t0 = threadIdx.x / units, unit = threadIdx.x - t0 * units;  // tokens of a pass; this thread's
  const bool on = t0 < per, turn = unit * 2 * R < r.rot;
  const bool split = turn && !r.adjacent;
  const int lo = split ? unit * R : unit * 2 * R, hi = split ? lo + r.half : lo + R, f0 = unit * R;
  const AngleTable<Q> table(r.half);
  // bytes of channel m of a slot in the stored page
  auto place = [&](int slot, int m) { return ((slot / 4 * chunks + m / EK) * 4 + slot % 4) * 16 + m % EK * (BITS / 8); };
  auto fetch = [&](int h, int t, u2v (&x)[2][Q]) __attribute__((always_inline)) {
    const E * row = static_cast<const E *>(p.k) + (long)h * p.k_head + (long)(w.row0 + t) * p.k_token;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      x[0][q] = *reinterpret_cast<const u2v *>(row + lo + 4 * q);
      x[1][q] = *reinterpret_cast<const u2v *>(row + hi + 4 * q);
    }
  };
  auto turned = [&](int t, const u2v (&x)[2][Q], f4v (&v)[2][Q]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const f2v a = unpack2<TYPE>(x[i][q][0]), b = unpack2<TYPE>(x[i][q][1]);
        v[i][q] = f4v{a[0], a[1], b[0], b[1]};
      }
    if (!turn) return;
    if (r.adjacent) {  // pair j of the 2 R channels: v[j / (R / 2)], elements 2 (j % (R / 2)) and the next
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int at = table.at(t, f0 + 4 * q);
        const f4v c4 = *reinterpret_cast<const f4v *>(cos + at), s4 = *reinterpret_cast<const f4v *>(sin + at);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = 4 * q + k;
          f4v & y = v[j / (2 * Q)][j % (2 * Q) / 2];
          const float a = y[j % 2 * 2], b = y[j % 2 * 2 + 1];
          y[j % 2 * 2] = a * c4[k] - b * s4[k];
          y[j % 2 * 2 + 1] = b * c4[k] + a * s4[k];
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int at = table.at(t, f0 + 4 * q);
        const f4v c4 = *reinterpret_cast<const f4v *>(cos + at), s4 = *reinterpret_cast<const f4v *>(sin + at);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float a = v[0][q][k], b = v[1][q][k];
          v[0][q][k] = a * c4[k] - b * s4[k];
          v[1][q][k] = b * c4[k] + a * s4[k];
        }
      }
    }
  };
  if constexpr (BITS == 16) {
    if (r.half) page_angles<NT, Q>(r, w, cos, sin);
    __syncthreads();
    for (int h = h0; h < h1; ++h) {
      uint8_t * dst = static_cast<uint8_t *>(c.kc) + (w.base + h) * ((long)c.page * c.dim * 2);
#pragma unroll 2
      for (int t = on ? t0 : n; t < n; t += per) {
        u2v x[2][Q];
        f4v v[2][Q];
        fetch(h, t, x);
        turned(t, x, v);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int q = 0; q < Q; q += 2) {
            uint8_t * at = dst + place(w.lo + t, (i ? hi : lo) + 4 * q);
            const u2v y = {pack2<TYPE>(v[i][q][0], v[i][q][1]), pack2<TYPE>(v[i][q][2], v[i][q][3])};
            if constexpr (Q == 1) {
              *reinterpret_cast<u2v *>(at) = y;
            } else {
              const f4v & z = v[i][q + 1];
              *reinterpret_cast<u4v *>(at) = u4v{y[0], y[1], pack2<TYPE>(z[0], z[1]), pack2<TYPE>(z[2], z[3])};
            }
          }
      }
    }
  } else {
    u2v x[U][2][Q];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (on && t0 + per * u < n) fetch(h0, t0 + per * u, x[u]);
    if (r.half) page_angles<NT, Q>(r, w, cos, sin);
    __syncthreads();
    for (int h = h0; h < h1; ++h) {
      uint8_t * dst = static_cast<uint8_t *>(c.kc) + (w.base + h) * ((long)c.page * c.dim);
      const float before = w.lo ? c.ks[w.base + h] : 0.0f;
      f4v v[U][2][Q];
      auto all = [&](auto && fn) __attribute__((always_inline)) {  // fn over the thread's values
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (on && t0 + per * u < n) {
#pragma unroll
            for (int i = 0; i < 2 * Q; ++i)
#pragma unroll
              for (int k = 0; k < 4; ++k) v[u][i / Q][i % Q][k] = fn(v[u][i / Q][i % Q][k]);
          }
      };
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + per * u;
        if (!on || t >= n) continue;
        turned(t, x[u], v[u]);
        if (h + 1 < h1) fetch(h + 1, t, x[u]);
      }
      float amax = 0.0f;
      all([&](float y) {
        amax = fmaxf(amax, fabsf(y));
        return y;
      });
      bool saturate;
      const float s = group_scale<NT>(amax, before, red + (h & 1), saturate, [&]() {
        float m = 0.0f;
        all([&](float y) {
          m = fmaxf(m, finite_abs(y));
          return y;
        });
        return m;
      });
      const float inv = 1.0f / s;
      all([&](float y) { return y * inv; });
      if (saturate) all([&](float y) { return saturated(y); });
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + per * u;
        if (!on || t >= n) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          unsigned y[Q];
#pragma unroll
          for (int q = 0; q < Q; ++q) y[q] = codes4(v[u][i][q][0], v[u][i][q][1], v[u][i][q][2], v[u][i][q][3]);
          uint8_t * at = dst + place(w.lo + t, i ? hi : lo);
          if constexpr (Q == 4) *reinterpret_cast<u4v *>(at) = u4v{y[0], y[1], y[2], y[3]};
          else if constexpr (Q == 2) *reinterpret_cast<u2v *>(at) = u2v{y[0], y[1]};
          else *reinterpret_cast<unsigned *>(at) = y[0];
        }
      }
      if (w.lo && before != s) {
        const float ratio = before * inv;
        for (int i = threadIdx.x; i < (c.page - n) * chunks; i += NT) {
          const int t = i / chunks;
          u4v * at = reinterpret_cast<u4v *>(dst + place(t < w.lo ? t : t + n, (i - t * chunks) * EK));
          u4v y = *at;
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = rescale4(y[q], ratio);
          *at = y;
        }
      }
      if (threadIdx.x == 0) c.ks[w.base + h] = s;
    }
  }
}

// Values of heads [h0, h1).  A thread owns two channels of EV tokens (a granule), 2 x 16 bytes side by
// side in the stored page, U of them.
template <int TYPE, int BITS, int NT, int U>
__device__ __forceinline__ void append_values(const AppendParams & p, const PageWork & w, int h0, int h1, float (*red)[4])
{
  typedef typename St<TYPE>::e E;
  constexpr int EV = BITS == 8 ? 16 : 8;
  const CacheParams & c = p.c;
  const int tid = threadIdx.x, pairs = c.dim / 2;
  const int g0 = w.lo / EV, ng = (w.hi + EV - 1) / EV - g0;  // granules with new tokens
  const int per = NT / pairs, first = tid / pairs, ch = 2 * (tid - first * pairs);  // granules of a pass; this thread's
  const bool on = first < per;
  auto fetch = [&](int h, int slot0, unsigned * x) __attribute__((always_inline)) {
    const E * src = static_cast<const E *>(p.v) + (long)h * p.v_head + ch;
#pragma unroll
    for (int t = 0; t < EV; ++t) {
      const int slot = slot0 + t;
      const bool fresh = slot >= w.lo && slot < w.hi;
      x[t] = fresh ? *reinterpret_cast<const unsigned *>(src + (long)(w.row0 + slot - w.lo) * p.v_token) : 0u;
    }
  };
  if constexpr (BITS == 16) {
    for (int h = h0; h < h1; ++h) {
      uint8_t * dst = static_cast<uint8_t *>(c.vc) + (w.base + h) * ((long)c.page * c.dim * 2);
      for (int g = on ? first : ng; g < ng; g += per) {
        const int slot0 = (g0 + g) * EV;
        unsigned x[EV];
        fetch(h, slot0, x);
        u4v * at = reinterpret_cast<u4v *>(dst + ((long)(g0 + g) * c.dim + ch) * 16);
        u4v y0, y1;
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // two tokens of one channel, then of the next
          y0[q] = (x[2 * q] & 0xffffu) | (x[2 * q + 1] << 16);
          y1[q] = (x[2 * q] >> 16) | (x[2 * q + 1] & 0xffff0000u);
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
  } else {
    unsigned x[U][EV];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (on && first + per * u < ng) fetch(h0, (g0 + first + per * u) * EV, x[u]);
    for (int h = h0; h < h1; ++h) {
      uint8_t * dst = static_cast<uint8_t *>(c.vc) + (w.base + h) * ((long)c.page * c.dim);
      const float before = w.lo ? c.vs[w.base + h] : 0.0f;
      float amax = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!on || first + per * u >= ng) continue;
#pragma unroll
        for (int t = 0; t < EV; ++t) {
          const f2v a = unpack2<TYPE>(x[u][t]);
          amax = fmaxf(fmaxf(amax, fabsf(a[0])), fabsf(a[1]));
        }
      }
      bool saturate;
      const float s = group_scale<NT>(amax, before, red + (h & 1), saturate, [&]() {
        float m = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!on || first + per * u >= ng) continue;
#pragma unroll
          for (int t = 0; t < EV; ++t) {
            const f2v a = unpack2<TYPE>(x[u][t]);
            m = fmaxf(fmaxf(m, finite_abs(a[0])), finite_abs(a[1]));
          }
        }
        return m;
      });
      const float inv = 1.0f / s;
      const bool grown = w.lo && before != s;
      const float ratio = before * inv;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int g = first + per * u, slot0 = (g0 + g) * EV;
        if (!on || g >= ng) continue;
        u4v * at = reinterpret_cast<u4v *>(dst + ((long)(g0 + g) * c.dim + ch) * 16);
        u4v y0, y1;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f2v a[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) a[t] = unpack2<TYPE>(x[u][4 * q + t]) * inv;
          if (saturate) {
#pragma unroll
            for (int t = 0; t < 4; ++t) a[t] = f2v{saturated(a[t][0]), saturated(a[t][1])};
          }
          y0[q] = codes4(a[0][0], a[1][0], a[2][0], a[3][0]);
          y1[q] = codes4(a[0][1], a[1][1], a[2][1], a[3][1]);
        }
        if (h + 1 < h1) fetch(h + 1, slot0, x[u]);
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
        for (int i = tid; i < (c.page / EV - ng) * c.dim; i += NT) {
          u4v * at = reinterpret_cast<u4v *>(dst + (long)(i < g0 * c.dim ? i : i + ng * c.dim) * 16);
          u4v y = *at;
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = rescale4(y[q], ratio);
          *at = y;
        }
      }
      if (tid == 0) c.vs[w.base + h] = s;
    }
  }
}

// NT: lanes; R: channels of a run of keys; UK, UV: units of keys and 32-byte pieces of values a thread holds of a
// whole page.  A work-group takes `span` heads, for the keys' of which it forms the angles once.
template <int TYPE, int BITS, int NT, int R, int UK, int UV>
__global__ void __launch_bounds__(NT) kv_append_kernel(const AppendParams p, int span)
{
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ float red[4][4];  // of even and uneven heads, in each case a second for pages with infinities
  PageWork w;
  if (!page_work(p.c, blockIdx.x, w)) return;
  const int h0 = blockIdx.y * span, h1 = min(h0 + span, p.c.heads);
  if (blockIdx.z == 0) {
    float * cos = reinterpret_cast<float *>(lds), * sin = cos + p.c.page * AngleTable<R / 4>::pitch_of(p.r.half) * 4;
    append_keys<TYPE, BITS, NT, R, UK>(p, w, h0, h1, red, cos, sin);
  } else {
    append_values<TYPE, BITS, NT, UV>(p, w, h0, h1, red);
  }
}

namespace {

template <int TYPE, int BITS, int NT, int R, int UK, int UV> void launch_append_kernel(const AppendParams & p, hipStream_t s)
{
  const CacheParams & c = p.c;
  auto kern = kv_append_kernel<TYPE, BITS, NT, R, UK, UV>;
  // heads of a work-group: as many as leave four work-groups a CU (20033 tokens of 8 heads: 37 us with
  // 4, 43 with 2, 58 with one each); in 16 bits, where no page's maximum is waited for, one
  const long pages = (long)c.tokens / c.page, wgs = std::max<long>(pages, c.batch) * c.heads * 2;
  const int span = BITS == 16 ? 1 : (int)std::min<long>(c.heads, std::max<long>(1, wgs / 1024));
  const dim3 grid((unsigned)(pages + 2L * c.batch), (c.heads + span - 1) / span, 2);
  const size_t lds = p.r.half ? (size_t)c.page * AngleTable<R / 4>::pitch_of(p.r.half) * 32 : 0;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) throw std::runtime_error(std::string("HIP error: ") + hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, grid, dim3(NT), lds, s, p, span);
}

template <int TYPE> void launch_append(const AppendParams & p, hipStream_t s)
{
  const CacheParams & c = p.c;
  // runs of 16, 8 or 4 channels, as the rotated channels and the others divide
  const int R = p.r.rot % 32 == 0 && c.dim % 32 == 0 ? 16 : p.r.rot % 16 == 0 ? 8 : 4;
  if (c.bits == 16) {  // nothing waits in registers
    if (R >= 8) launch_append_kernel<TYPE, 16, 256, 8, 1, 1>(p, s);
    else launch_append_kernel<TYPE, 16, 256, 4, 1, 1>(p, s);
    return;
  }
  // passes over a page: of the keys, 256 / (dim / 2 R) tokens at once; of the values, 512 / dim
  // granules of 16
  const int tokens = 256 / (c.dim / (2 * R)), uk = (c.page + tokens - 1) / tokens;
  const int gran = 256 / (c.dim / 2), uv = (c.page / 16 + gran - 1) / gran;
  // One wave does a page where the other three would have little to do: pages of 16, or a token or two for
  // each sequence. Registers for four passes cost more than they save while the chip is not full. One
  // wave / four, 8 heads of 128 channels, in us: 60 sequences of a token each, pages of 16, 5.6 / 9.2;
  // 512 of them, pages of 64, 23.0 / 30.5; 8 prompts of 200, pages of 16, 7.5 / 12.1; one token, pages of
  // 64, 6.0 / 4.5 (so not there).
  const bool few = (long)c.tokens <= 4L * c.batch, small = c.page * c.dim <= 64 * 32;
  if (R == 16 && uk <= 1 && uv <= 1 && p.r.half <= 64 && c.dim <= 128 && (few || c.page == 16)) {
    if (small) {
      launch_append_kernel<TYPE, 8, 64, 16, 1, 1>(p, s);
      return;
    }
    if ((long)c.batch * c.heads >= 256) {
      launch_append_kernel<TYPE, 8, 64, 16, 4, 4>(p, s);
      return;
    }
  }
  if (R == 16) {
    if (uk <= 1 && uv <= 1) launch_append_kernel<TYPE, 8, 256, 16, 1, 1>(p, s);
    else if (uk <= 2 && uv <= 2) launch_append_kernel<TYPE, 8, 256, 16, 2, 2>(p, s);
    else launch_append_kernel<TYPE, 8, 256, 16, 4, 4>(p, s);
  } else if (R == 8) {
    if (uk <= 2 && uv <= 1) launch_append_kernel<TYPE, 8, 256, 8, 2, 1>(p, s);
    else launch_append_kernel<TYPE, 8, 256, 8, 8, 4>(p, s);
  } else {
    launch_append_kernel<TYPE, 8, 256, 4, 16, 4>(p, s);
  }
}

}  // namespace

void launch_kv_append(const AppendParams & p, hipStream_t s)
{
  if (p.c.type == kSeqF16) launch_append<kSeqF16>(p, s);
  else launch_append<kSeqBF16>(p, s);
}

}  // namespace ivh
