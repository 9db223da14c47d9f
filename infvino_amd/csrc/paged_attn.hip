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
// e4m3 codes become f16 or bf16 exactly; the key scale multiplies the scores, one factor a lane.  The
// value scale goes into the exponent: with w = exp2(t + log2 vs - M), M the running maximum of t + log2 vs, the output is
// sum w V / sum (w / vs), so no product of a code and its scale can leave the 16-bit range.
// Probabilities are rounded to 16 bits for the second product (half a step relative, as the
// output's own rounding); their sum is taken before that.
//
// Few rows: a work-group's four waves take every fourth step, and further work-groups further keys; the partial
// sums are joined through LDS and by a second kernel.  Many rows: each wave takes rows of its own.
#include <algorithm>
#include <stdexcept>

#include "conv_common.hpp"
#include "seq_common.hpp"

namespace ivh {

namespace {

struct Visible {  // what a query at place i sees
  int full, window, sinks;
  __device__ __forceinline__ bool operator()(int i, int j) const
  {
    return j <= i && j < full && (window == 0 || i - j < window || j < sinks);
  }
};

// the steps of 64 keys that rows at places imin..imax need: `first` of them over the first
// tokens, the others from step `from` on
struct Steps {
  int total, first, from;
};
__device__ __forceinline__ Steps key_steps(int full, int imin, int imax, int window, int sinks)
{
  const int end = imax >= full ? full : imax + 1;
  const int lo = window ? max(0, imin - window + 1) : 0;
  Steps s;
  s.from = min(lo, end) / 64;
  s.first = min((min(sinks, lo) + 63) / 64, s.from);
  s.total = end > 0 ? s.first + (end + 63) / 64 - s.from : 0;
  return s;
}
__device__ __forceinline__ int step_key(const Steps & s, int n) { return 64 * (n < s.first ? n : s.from + n - s.first); }

}  // namespace

// QT: 16-row tiles of a wave; WK: waves that share rows and split the keys, 4 / WK row ranges.
// DP: head size rounded up to 64, 128 or 256.
template <int TYPE, int BITS, int DP, int QT, int WK>
__global__ void __launch_bounds__(256) paged_attn_kernel(const PagedParams p)
{
  using T = St<TYPE>;
  typedef typename T::e E;
  constexpr int EK = BITS == 8 ? 16 : 8;        // channels of a 16-byte key piece
  constexpr int KL = DP / (4 * EK);             // key pieces of a lane and tile
  constexpr int VL = BITS == 8 ? 1 : 2;         // value pieces of a lane and channel block
  constexpr int NB = DP / 16;                   // channel blocks
  constexpr int NS = DP / 32;                   // 32-channel slices
  constexpr int ROWS = 16 * QT * (4 / WK);      // rows of a work-group
  extern __shared__ __attribute__((aligned(16))) float lds[];

  const CacheParams & c = p.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int wk = wave % WK, wr = wave / WK;
  // neighbours share a sequence and key head, and run on one XCD
  int w = xcd_tile(blockIdx.x, gridDim.x);
  const int slot = w % p.row_slots;
  w /= p.row_slots;
  const int part = w % p.parts;
  w /= p.parts;
  const int h = w % c.heads, b = w / c.heads;

  const int c0 = min(max(c.cu[b], 0), c.tokens), c1 = min(max(c.cu[b + 1], c0), c.tokens);
  const int nnew = c1 - c0, rows = nnew * p.group;
  const long len = c.lens[b];
  const int full = (int)min(max(len, 0L), (long)c.width * c.page);
  const int place0 = (int)max(len, 0L) - nnew;  // place of the first new token
  const Visible see = {full, p.window, p.sinks};
  const int32_t * table = c.table + (long)b * c.width;
  const int lp = 31 - __clz(c.page);  // page is a power of two
  const long page_bytes = (long)c.page * c.dim * (BITS / 8);
  const int nblk = c.dim / 16;

  for (int tile = slot; tile * ROWS < rows; tile += p.row_slots) {
    const int row0 = tile * ROWS + wr * 16 * QT;           // this wave's rows
    const int last = min(rows, tile * ROWS + ROWS) - 1;    // the work-group's last row
    const int imin = place0 + tile * ROWS / p.group, imax = place0 + last / p.group;
    const Steps steps = key_steps(full, imin, imax, p.window, p.sinks);
    const int per = max(p.part_steps, (steps.total + p.parts - 1) / p.parts);
    const int n0 = part * per, n1 = min(steps.total, n0 + per);

    // this lane's query of each row tile: token, head, place
    int qtok[QT], qhead[QT], place[QT];
    bool live[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int row = row0 + 16 * t + r;
      live[t] = row < rows;
      qtok[t] = row / p.group;
      qhead[t] = h * p.group + row - qtok[t] * p.group;
      place[t] = live[t] ? place0 + qtok[t] : -1;  // -1 sees nothing
    }
    // Q^T fragments in the order of the key pieces: 8-bit pieces hold 16 channels, two slices
    u4v qf[QT][NS];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const E * q = static_cast<const E *>(p.q) + (long)(c0 + qtok[t]) * p.q_token + (long)qhead[t] * p.q_head;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int ch = BITS == 8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
        qf[t][s] = live[t] && ch < c.dim ? *reinterpret_cast<const u4v *>(q + ch) : u4v{0, 0, 0, 0};
      }
    }

    f4v o[QT][NB];
    float M[QT], L[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      M[t] = kLowest;
      L[t] = 0.0f;
#pragma unroll
      for (int j = 0; j < NB; ++j) o[t][j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // page of the granule that this lane reads keys from (r / 4) and of its own group's
    auto page_of = [&](int n, int gran) {
      const int at = min((step_key(steps, n) + 16 * gran) >> lp, c.width - 1);
      return table[at];
    };
    u4v kf[4][KL], vf[NB][VL];
    float ksc = 1.0f, vsc = 1.0f;
    bool vok = true;
    auto load_k = [&](int n, int id) {
      const bool ok = (unsigned)id < (unsigned)c.pages;
      const uint8_t * base = static_cast<const uint8_t *>(c.kc) + ((long)(ok ? id : 0) * c.heads + h) * page_bytes;
      const int quad = ((step_key(steps, n) + 16 * (r >> 2)) & (c.page - 1)) / 4;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const int ch = 4 * i + g;
          const unsigned off = (unsigned)((quad + t) * (c.dim / EK) + ch) * 64u + (unsigned)(r & 3) * 16u;
          kf[t][i] = ch * EK < c.dim ? *reinterpret_cast<const u4v *>(base + off) : u4v{0, 0, 0, 0};
        }
    };
    auto load_v = [&](int n, int id) {
      vok = (unsigned)id < (unsigned)c.pages;
      const long page = (long)(vok ? id : 0) * c.heads + h;
      const uint8_t * base = static_cast<const uint8_t *>(c.vc) + page * page_bytes;
      const int gran = ((step_key(steps, n) + 16 * g) & (c.page - 1)) / 16;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (j >= nblk) continue;
#pragma unroll
        for (int i = 0; i < VL; ++i)
          vf[j][i] = *reinterpret_cast<const u4v *>(base + ((unsigned)((gran * VL + i) * c.dim) + 16u * j + r) * 16u);
      }
      if (BITS == 8) {
        ksc = c.ks[page];
        vsc = c.vs[page];
      }
    };

    const int nf = n0 + wk;
    if (nf < n1) {
      load_k(nf, page_of(nf, r >> 2));
      load_v(nf, page_of(nf, g));
    }
    for (int n = nf; n < n1; n += WK) {
      const int key0 = step_key(steps, n);
      const int nn = min(n + WK, n1 - 1);  // the next step's pages (the last one's again at the end)
      const int idk = page_of(nn, r >> 2), idv = page_of(nn, g);
      // ---- scores
      f4v s[QT][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int u = 0; u < QT; ++u) s[u][t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          if constexpr (BITS == 8) {
            const u4v x = kf[t][i];
            const u4v lo = {T::fp8_lo(x[0]), T::fp8_hi(x[0]), T::fp8_lo(x[1]), T::fp8_hi(x[1])};
            const u4v hi = {T::fp8_lo(x[2]), T::fp8_hi(x[2]), T::fp8_lo(x[3]), T::fp8_hi(x[3])};
#pragma unroll
            for (int u = 0; u < QT; ++u) {
              s[u][t] = T::mma16(lo, qf[u][2 * i], s[u][t]);
              s[u][t] = T::mma16(hi, qf[u][2 * i + 1], s[u][t]);
            }
          } else {
#pragma unroll
            for (int u = 0; u < QT; ++u) s[u][t] = T::mma16(kf[t][i], qf[u][i], s[u][t]);
          }
        }
      }
      const bool ok = vok;
      const float ks = BITS == 8 ? ksc : 1.0f, vs = BITS == 8 ? fmaxf(vsc, 1e-30f) : 1.0f;
      if (n + WK < n1) load_k(nn, idk);
      // ---- masks: only steps where some row of the work-group does not see every key have them
      const bool inner = key0 + 63 <= imin && key0 + 63 < full &&
                         (p.window == 0 || imax - key0 < p.window || key0 + 63 < p.sinks) && __all(ok);
      const float mul = p.scale_log2 * ks, ev = BITS == 8 ? __builtin_amdgcn_logf(vs) : 0.0f;
      const float unv = BITS == 8 ? __builtin_amdgcn_rcpf(vs) : 1.0f;
      u4v pf[QT][2];
#pragma unroll
      for (int u = 0; u < QT; ++u) {
        float top = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float x = fmaf(s[u][t][v], mul, ev);
            if (!inner && !(ok && see(place[u], key0 + 16 * g + 4 * t + v))) x = -__builtin_inff();
            s[u][t][v] = x;
            top = fmaxf(top, x);
          }
        top = across16(across32(top, MaxOp()), MaxOp());
        // the reference exponent follows the maximum only when that is 2^8 above it: weights up
        // to 2^8 lose nothing in either 16-bit type
        if (__any(top > M[u] + 8.0f)) {
          const float m = fmaxf(M[u], top), a = __builtin_amdgcn_exp2f(M[u] - m);
          M[u] = m;
          L[u] *= a;
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) o[u][j][v] *= a;
        }
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          float e[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            e[v] = __builtin_amdgcn_exp2f(s[u][t][v] - M[u]);
            sum += e[v];
          }
          pf[u][t / 2][2 * (t % 2)] = pack2<TYPE>(e[0], e[1]);
          pf[u][t / 2][2 * (t % 2) + 1] = pack2<TYPE>(e[2], e[3]);
        }
        L[u] = fmaf(sum, unv, L[u]);
      }
      // ---- values that no row sees (behind the last key, outside every window, in no page) may
      // hold anything: zeros in their place.  With several tokens in the tile an infinity or NaN
      // that only some rows see is taken out as well and added to those rows by itself.
      bool odd = false;
      if (!inner) {
        u4v keep[VL];
#pragma unroll
        for (int i = 0; i < VL; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            constexpr int PER = BITS == 8 ? 4 : 2;
            unsigned m = 0;
#pragma unroll
            for (int t = 0; t < PER; ++t) {
              const int j = key0 + 16 * g + (BITS == 8 ? 4 * q + t : 8 * i + 2 * q + t);
              // a key between the first and last row's windows is seen by some row
              const bool any = ok && j < full && j <= imax && (p.window == 0 || imin - j < p.window || j < p.sinks);
              m |= any ? (BITS == 8 ? 0xffu << (8 * t) : 0xffffu << (16 * t)) : 0u;
            }
            keep[i][q] = m;
          }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          if (j >= nblk) continue;
#pragma unroll
          for (int i = 0; i < VL; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              vf[j][i][q] &= keep[i][q];
              if (imax > imin) {
                const unsigned x = vf[j][i][q];
                odd = odd || (BITS == 8 ? (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) : T::odd_bits(x)) != 0;
              }
            }
        }
        if (imax > imin) odd = __any(odd);
      }
      if (odd) {
        // clean the fragments, and add what was taken out to the rows that see it
        for (int j64 = 0; j64 < 64; ++j64) {
          const int key = key0 + j64, at = min(key >> lp, c.width - 1), id = table[at];
          if ((unsigned)id >= (unsigned)c.pages || key >= full) continue;
          const long page = (long)id * c.heads + h;
          const uint8_t * base = static_cast<const uint8_t *>(c.vc) + page * page_bytes;
          const int in = key & (c.page - 1);
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            if (j >= nblk) continue;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const int ch = 16 * j + 4 * g + v;
              float x;
              if (BITS == 8) x = __builtin_amdgcn_cvt_f32_fp8((int)base[((in / 16) * c.dim + ch) * 16 + in % 16], 0);
              else x = (float)reinterpret_cast<const E *>(base)[((in / 8) * c.dim + ch) * 8 + in % 8];
              if (!(fabsf(x) < __builtin_inff()))
#pragma unroll
                for (int u = 0; u < QT; ++u)
                  if (see(place[u], key)) o[u][j][v] += x;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          if (j >= nblk) continue;
#pragma unroll
          for (int i = 0; i < VL; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const unsigned x = vf[j][i][q];
              // top bits of the elements to drop, spread over them
              const unsigned d = BITS == 8 ? (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) : T::odd_bits(x);
              vf[j][i][q] = x & ~(BITS == 8 ? (d >> 7) * 0xffu : (d >> 15) * 0xffffu);
            }
        }
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (j >= nblk) continue;
        u4v v0, v1;
        if constexpr (BITS == 8) {
          const u4v x = vf[j][0];
          v0 = u4v{T::fp8_lo(x[0]), T::fp8_hi(x[0]), T::fp8_lo(x[1]), T::fp8_hi(x[1])};
          v1 = u4v{T::fp8_lo(x[2]), T::fp8_hi(x[2]), T::fp8_lo(x[3]), T::fp8_hi(x[3])};
        } else {
          v0 = vf[j][0];
          v1 = vf[j][1];
        }
#pragma unroll
        for (int u = 0; u < QT; ++u) {
          o[u][j] = T::mma16(v0, pf[u][0], o[u][j]);
          o[u][j] = T::mma16(v1, pf[u][1], o[u][j]);
        }
      }
      if (n + WK < n1) load_v(nn, idv);
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
        if (!live[u]) continue;
        const long row = (long)(c0 + qtok[u]) * p.heads + qhead[u];
        if (p.parts == 1) {
          const float inv = L[u] != 0.0f ? 1.0f / L[u] : 0.0f;  // a row that saw nothing is zero (NaN stays)
          E * out = static_cast<E *>(p.o) + (long)(c0 + qtok[u]) * p.o_token + (long)qhead[u] * p.o_head;
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            if (j >= nblk) continue;
            const u2v y = {pack2<TYPE>(o[u][j][0] * inv, o[u][j][1] * inv), pack2<TYPE>(o[u][j][2] * inv, o[u][j][3] * inv)};
            *reinterpret_cast<u2v *>(out + 16 * j + 4 * g) = y;
          }
        } else {
          const long n = (long)c.tokens * p.heads, at = (long)part * n + row;
          if (n0 < n1) {
            float * out = p.ws + at * c.dim;
#pragma unroll
            for (int j = 0; j < NB; ++j)
              if (j < nblk) *reinterpret_cast<f4v *>(out + 16 * j + 4 * g) = o[u][j];
          }
          if (g == 0) *reinterpret_cast<f2v *>(p.ws + (long)p.parts * n * c.dim + 2 * at) = f2v{M[u], L[u]};
        }
      }
    }
  }
}

// Joins the parts of a row: a lane has 4 channels, dim / 4 lanes a row.  A part that had no keys
// for the row left a sum of zero and is not read.
template <int TYPE>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedParams p)
{
  typedef typename St<TYPE>::e E;
  const CacheParams & c = p.c;
  const int lanes = c.dim / 4, per = 256 / lanes;
  const int sub = threadIdx.x / lanes, ch = 4 * (threadIdx.x - sub * lanes);
  const long n = (long)c.tokens * p.heads;
  const long row = (long)blockIdx.x * per + sub;
  if (sub >= per || row >= n) return;
  const int token = (int)(row / p.heads), head = (int)(row - (long)token * p.heads);
  if (token < c.cu[0] || token >= c.cu[c.batch]) return;  // rows of no sequence stay as they are
  const f2v * ml = reinterpret_cast<const f2v *>(p.ws + (long)p.parts * n * c.dim);
  float M = kLowest;
  for (int i = 0; i < p.parts; ++i) M = fmaxf(M, ml[(long)i * n + row][0]);
  float L = 0.0f;
  f4v o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < p.parts; ++i) {
    const long at = (long)i * n + row;
    const f2v t = ml[at];
    if (t[1] == 0.0f) continue;
    const float e = __builtin_amdgcn_exp2f(t[0] - M);
    L = fmaf(t[1], e, L);
    const f4v x = *reinterpret_cast<const f4v *>(p.ws + at * c.dim + ch);
#pragma unroll
    for (int v = 0; v < 4; ++v) o[v] = fmaf(x[v], e, o[v]);
  }
  const float inv = L != 0.0f ? 1.0f / L : 0.0f;
  const u2v y = {pack2<TYPE>(o[0] * inv, o[1] * inv), pack2<TYPE>(o[2] * inv, o[3] * inv)};
  *reinterpret_cast<u2v *>(static_cast<E *>(p.o) + (long)token * p.o_token + (long)head * p.o_head + ch) = y;
}

size_t paged_split(PagedParams & p, int max_new, int max_len)
{
  const CacheParams & c = p.c;
  const long rows = (long)std::max(1, std::min(max_new, c.tokens)) * p.group;
  p.row_tiles = rows <= 16 ? 1 : 2;
  p.row_waves = rows <= 64 ? 1 : 4;
  const int per_wg = 16 * p.row_tiles * p.row_waves;
  p.row_slots = (int)std::min<long>({(rows + per_wg - 1) / per_wg, 1024, (1L << 24) / ((long)c.batch * c.heads)});
  // keys: enough work-groups to fill the chip four times over, of at least one step a wave; none longer than 32
  // steps a wave, so that one long sequence of a ragged batch does not outlast the others
  long len = std::min<long>(max_len, (long)c.width * c.page);
  if (p.window) len = std::min<long>(len, (long)p.window + p.sinks + max_new + 128);
  const long steps = (len + 63) / 64, waves = 4 / p.row_waves;
  const long wgs = (long)c.batch * c.heads * p.row_slots;
  const long want = std::max<long>((1024 + wgs - 1) / wgs, (steps + 32 * waves - 1) / (32 * waves));
  const long most = std::max<long>(1, (steps + waves - 1) / waves);
  p.parts = (int)std::min<long>({std::max<long>(want, 1), most, 256});
  // a launch holds 2^24 work-groups of 256 lanes
  p.parts = (int)std::min<long>(p.parts, std::max<long>(1, (1L << 24) / wgs));
  p.part_steps = (int)((((steps + p.parts - 1) / p.parts) + waves - 1) / waves * waves);
  p.parts = (int)std::max<long>(1, (steps + p.part_steps - 1) / p.part_steps);
  if (p.parts == 1) return 0;
  return (size_t)p.parts * c.tokens * p.heads * (c.dim + 2) * sizeof(float);
}

namespace {

template <int TYPE, int BITS, int DP, int QT, int WK> void launch_paged(const PagedParams & p, hipStream_t s)
{
  auto kern = paged_attn_kernel<TYPE, BITS, DP, QT, WK>;
  const size_t lds = WK == 1 ? 0 : (size_t)(WK / 2) * (4 / WK) * 16 * QT * (DP + 4 + 2) * sizeof(float);
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) throw std::runtime_error(std::string("HIP error: ") + hipGetErrorString(e));
  }
  const dim3 grid((unsigned)((long)p.c.batch * p.c.heads * p.parts * p.row_slots)), blk(256);
  hipLaunchKernelGGL(kern, grid, blk, lds, s, p);
}

template <int TYPE, int BITS, int DP> void launch_paged_rows(const PagedParams & p, hipStream_t s)
{
  if (p.row_tiles == 1) launch_paged<TYPE, BITS, DP, 1, 4>(p, s);
  else if (p.row_waves == 1) launch_paged<TYPE, BITS, DP, 2, 4>(p, s);
  else launch_paged<TYPE, BITS, DP, 2, 1>(p, s);
}

template <int TYPE, int BITS> void launch_paged_dim(const PagedParams & p, hipStream_t s)
{
  if (p.c.dim <= 64) launch_paged_rows<TYPE, BITS, 64>(p, s);
  else if (p.c.dim <= 128) launch_paged_rows<TYPE, BITS, 128>(p, s);
  else launch_paged_rows<TYPE, BITS, 256>(p, s);
}

}  // namespace

void launch_paged_attention(const PagedParams & p, hipStream_t s)
{
  const bool f16 = p.c.type == kSeqF16;
  if (p.c.bits == 8) f16 ? launch_paged_dim<kSeqF16, 8>(p, s) : launch_paged_dim<kSeqBF16, 8>(p, s);
  else f16 ? launch_paged_dim<kSeqF16, 16>(p, s) : launch_paged_dim<kSeqBF16, 16>(p, s);
  if (p.parts > 1) {
    const int per = 256 / (p.c.dim / 4);
    const dim3 grid((unsigned)(((long)p.c.tokens * p.heads + per - 1) / per)), blk(256);
    if (f16) hipLaunchKernelGGL((paged_join_kernel<kSeqF16>), grid, blk, 0, s, p);
    else hipLaunchKernelGGL((paged_join_kernel<kSeqBF16>), grid, blk, 0, s, p);
  }
}

}  // namespace ivh
