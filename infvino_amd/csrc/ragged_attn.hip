// Attention over ragged contiguous sequences, causal or not, with an optional sliding window and
// first tokens that stay visible, on gfx950 MFMA.
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j] over the keys j that i sees; places count from
//   the end: the last query stands at the last key
//
// Long prompts are bound by the matrix cores: 4 dim operations for a pair of tokens, against
// 4 dim bytes of each key for 128 rows.  A work-group of four waves owns 128 rows of one head, a
// wave 32 of them, and walks the keys 64 at a time with a running maximum and sum in fp32:
//   * keys and values are copied by DMA straight into one of two LDS stages while the other is
//     worked on;
//   * S^T = K Q^T on 32x32x16 MFMA: a lane holds 16 scores of one query of a 32-key block, keys
//     8 (v / 4) + 4 (lane / 32) + v % 4.  As an operand of the second product its scores 8 s ..
//     8 s + 7 are 8 of the 16 keys of slice s, no lane exchange between the products;
//   * O^T = V^T P^T, with V^T read from the row-major stage by the transposing LDS load, 4 keys
//     of one channel a lane, in the order of the scores.
// LDS rows are not padded (DMA writes 64 x 16 bytes in a row); 16-byte pieces are permuted within
// a row by the source address, so that the lanes that are served together lie in distinct banks.
#include <algorithm>
#include <stdexcept>

#include "conv_common.hpp"
#include "seq_common.hpp"

namespace ivh {

namespace {

typedef __attribute__((address_space(3))) void lds_ptr;
typedef short s4v __attribute__((ext_vector_type(4)));

constexpr int kKeys = 64;   // keys of a step
constexpr int kRows = 128;  // rows of a work-group

// position of 16-byte piece c of row r in a row of DP / 8 pieces (its own inverse)
template <int DP> __device__ __forceinline__ int key_piece(int r, int c)
{
  if (DP % 128 == 0) return c ^ ((r & 3) | ((r >> 3 & 3) << 2));
  if (DP % 64 == 0) return c ^ ((r >> 1 & 1) | ((r >> 3 & 3) << 1));
  return c ^ (r >> 3 & 3);
}
template <int DP> __device__ __forceinline__ int value_piece(int r, int c)
{
  if (DP % 128 == 0) return c ^ ((r & 3) << 2);
  if (DP % 64 == 0) return c ^ ((r >> 1 & 1) << 2);
  return c;
}

// 64 x 16 bytes straight into LDS: lane i's from base + its offset (zeros where that is kBufOOB) to lds + 16 i
__device__ __forceinline__ void copy_to_lds(const void * base, unsigned off, void * lds)
{
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, 0x7fffffff, kBufDword3);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr *)lds, 16, (int)off, 0, 0, 0);
}

// 4 x 16 elements of LDS, one 8-byte run a lane (rows of 4 lanes), transposed within 16 lanes: lane
// i gets column i
__device__ __forceinline__ u2v read_transposed(const void * at)
{
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)(at)));
#else
  return u2v{};
#endif
}

// What a query at place i sees: keys lo..hi and the first `sinks`.
struct RaggedMask {
  int nk, causal, window, sinks;  // sinks 0 without a window
  __device__ __forceinline__ int lo(int i) const { return window ? i - window + 1 : 0; }
  __device__ __forceinline__ int hi(int i) const
  {
    const int h = causal ? i : window ? (int)min((long)i + window - 1, (long)nk) : nk;
    return min(h, nk - 1);
  }
  __device__ __forceinline__ bool operator()(int i, int j) const { return (j >= lo(i) && j <= hi(i)) || (j < sinks && (!causal || j <= i) && j < nk); }
  // whether rows imin..imax see all of keys j0..j1, or none of them
  __device__ __forceinline__ bool all(int imin, int imax, int j0, int j1) const
  {
    return j1 <= (causal ? min(imin, nk - 1) : nk - 1) && ((j0 >= lo(imax) && j1 <= hi(imin)) || j1 < sinks);
  }
  __device__ __forceinline__ bool none(int imin, int imax, int j0, int j1) const
  {
    return j0 >= nk || (causal && j0 > imax) || (j0 >= sinks && (j1 < lo(imin) || j0 > hi(imax)));
  }
};

}  // namespace

template <int TYPE, int DP>
__global__ void __launch_bounds__(256, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) ragged_attn_kernel(const RaggedParams p, int slots, int round)
{
  using T = St<TYPE>;
  typedef typename T::e E;
  constexpr int NS = DP / 16;          // 16-channel slices of the first product
  constexpr int NB = DP / 32;          // 32-channel blocks of the second
  constexpr int PR = DP / 8;           // 16-byte pieces of a row
  constexpr int NI = kKeys * PR / 256; // copies of a wave, keys or values of a step
  constexpr int STAGE = kKeys * DP;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_raw[];
  E * const K = reinterpret_cast<E *>(lds_raw);  // [2][64][DP]
  E * const V = K + 2 * STAGE;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 31, hi = lane >> 5;
  // The work-groups of a unit (sequence and key head) run on one XCD, whose L2 they share keys and values in.
  // Units go round the XCDs where that is even, so that each gets its share of long and short
  // sequences; a few units are cut into equal runs of work-groups instead.
  const int unit_wgs = p.group * slots, units = p.batch * (p.heads / p.group);
  int w = blockIdx.x, unit;
  if (round) {
    unit = w / kXcds / unit_wgs * kXcds + w % kXcds;
    w = w / kXcds % unit_wgs;
    if (unit >= units) return;
  } else {
    w = xcd_tile(w, gridDim.x);
    unit = w / unit_wgs;
    w -= unit * unit_wgs;
  }
  const int kv_heads = p.heads / p.group, b = unit / kv_heads, kvh = unit - b * kv_heads;
  const int slot = w % slots, head = kvh * p.group + w / slots;

  const int q0 = min(max(p.cu_q[b], 0), p.tokens_q), q1 = min(max(p.cu_q[b + 1], q0), p.tokens_q);
  const int k0 = min(max(p.cu_k[b], 0), p.tokens_k), k1 = min(max(p.cu_k[b + 1], k0), p.tokens_k);
  const int nq = q1 - q0, nk = k1 - k0;
  const RaggedMask see = {nk, p.causal, p.window, p.window ? p.sinks : 0};
  const E * kp = static_cast<const E *>(p.k) + (long)k0 * p.k_token + (long)kvh * p.k_head;
  const E * vp = static_cast<const E *>(p.v) + (long)k0 * p.v_token + (long)kvh * p.v_head;

  // what this lane copies: position pos of row `row` of the stage holds a piece of the key's row
  unsigned koff[NI], voff[NI];
  int crow[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int s = 64 * (wave + 4 * i) + lane, row = s / PR, pos = s - row * PR;
    const int kc = key_piece<DP>(row, pos), vc = value_piece<DP>(row, pos);
    crow[i] = row;
    koff[i] = kc * 8 < p.dim ? (unsigned)(row * (int)p.k_token + kc * 8) * 2u : kBufOOB;
    voff[i] = vc * 8 < p.dim ? (unsigned)(row * (int)p.v_token + vc * 8) * 2u : kBufOOB;
  }

  // a negative scale turns the queries' signs, so that the largest score has the largest exponent
  const float scale = fmaxf(fabsf(p.scale_log2), 1.2e-38f);  // not 0: masked scores stay -inf
  const unsigned flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;

  const int nqb = (nq + kRows - 1) / kRows;
  for (int t = slot; t < nqb; t += slots) {
    const int qb = nqb - 1 - t;  // the longest first
    const int shift = nk - nq;
    const int imin = qb * kRows + shift, imax = min(nq - 1, qb * kRows + kRows - 1) + shift;
    const int wmin = imin + 32 * wave, wmax = min(imax, wmin + 31);  // this wave's rows (none where wmax < wmin)
    const int row = qb * kRows + 32 * wave + col;
    const bool live = row < nq;
    const int place = live ? row + shift : -(1 << 27);
    const E * q = static_cast<const E *>(p.q) + (long)(q0 + row) * p.q_token + (long)head * p.q_head;
    u4v qf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int ch = 16 * s + 8 * hi;
      qf[s] = live && ch < p.dim ? *reinterpret_cast<const u4v *>(q + ch) ^ flip : u4v{0, 0, 0, 0};
    }

    // steps: `first` over the first tokens, the others from step `from` on
    const int ahead = p.window ? (int)min(max((long)imax + p.window, (long)p.sinks), (long)nk) : nk;
    const int end = p.causal ? min(nk, imax + 1) : ahead;
    const int lo = p.window ? max(0, imin - p.window + 1) : 0;
    const int from = min(lo, max(end, 0)) / kKeys;
    const int first = min((min(p.sinks, lo) + kKeys - 1) / kKeys, from);
    const int total = end > 0 ? first + (end + kKeys - 1) / kKeys - from : 0;
    auto key_of = [&](int n) { return kKeys * (n < first ? n : from + n - first); };

    auto copy = [&](int n) __attribute__((always_inline)) {
      const int key0 = key_of(n), left = nk - key0, st = n & 1;
      const E * ks = kp + (long)key0 * p.k_token, * vs = vp + (long)key0 * p.v_token;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        copy_to_lds(ks, crow[i] < left ? koff[i] : kBufOOB, K + st * STAGE + 512 * (wave + 4 * i));
#pragma unroll
      for (int i = 0; i < NI; ++i)
        copy_to_lds(vs, crow[i] < left ? voff[i] : kBufOOB, V + st * STAGE + 512 * (wave + 4 * i));
    };

    // what this lane's row sees, less the lane's first key of a 32-key block
    const int seen_lo = see.lo(place) - 4 * hi, seen_n = see.hi(place) - see.lo(place);
    const int seen_first = min(see.sinks, see.causal ? place + 1 : see.nk) - 4 * hi;

    f16v o[NB];
    float M, L;
    // An infinity or NaN among the values reaches rows that do not see it, as 0 x inf, and stays in
    // their sums.  So rows are first taken as they come; only if a result is not finite are they taken again
    // with such values left out of the product and added to the rows that do see them.
    for (int careful = 0; careful < 2; ++careful) {
#pragma unroll
    for (int j = 0; j < NB; ++j) o[j] = f16v{};
    M = kLowest;
    L = 0.0f;

    __syncthreads();  // the last rows' stages are no longer read
    if (total > 0) copy(0);
    for (int n = 0; n < total; ++n) {
      __builtin_amdgcn_s_waitcnt(vm_wait(0));
      __syncthreads();
      if (n + 1 < total) copy(n + 1);
      const int key0 = key_of(n);
      if (wmax < wmin || see.none(wmin, wmax, key0, key0 + kKeys - 1)) continue;
      const bool inner = see.all(wmin, wmax, key0, key0 + kKeys - 1);
      const E * Ks = K + (n & 1) * STAGE;
      const E * Vs = V + (n & 1) * STAGE;

      f16v s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        s[kb] = f16v{};
        const int r = 32 * kb + col;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const u4v a = *reinterpret_cast<const u4v *>(Ks + r * DP + key_piece<DP>(r, 2 * i + hi) * 8);
          s[kb] = T::mma32(a, qf[i], s[kb]);
        }
      }
      if (!inner) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int j = key0 + 32 * kb + 8 * (v / 4) + v % 4;
            const bool ok = (seen_n >= 0 && (unsigned)j - (unsigned)seen_lo <= (unsigned)seen_n) || j < seen_first;
            s[kb][v] = ok ? s[kb][v] : -__builtin_inff();
          }
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v) top = fmaxf(top, s[kb][v]);
      top = across32(top, MaxOp()) * scale;
      // the reference exponent follows the maximum only when that is 2^8 above it: weights up to
      // 2^8 lose nothing in either 16-bit type
      if (__any(top > M + 8.0f)) {
        const float m = fmaxf(M, top), a = __builtin_amdgcn_exp2f(M - m);
        M = m;
        L *= a;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[j][v] *= a;
      }
      u4v pf[4];
      float sum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
          const float x = __builtin_amdgcn_exp2f(fmaf(s[kb][v], scale, -M));
          const float y = __builtin_amdgcn_exp2f(fmaf(s[kb][v + 1], scale, -M));
          sum += x + y;
          pf[2 * kb + v / 8][v % 8 / 2] = pack2<TYPE>(x, y);
        }
      L += sum;

      // V^T fragment of 16 keys and 32 channels: two transposing loads of 4 keys each
      auto values = [&](int sl, int j) __attribute__((always_inline)) {
        u4v a;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = 16 * sl + 8 * u + 4 * hi + ((lane & 15) >> 2);
          const int pc = 4 * j + 2 * (lane >> 4 & 1) + ((lane & 3) >> 1);
          const E * at = Vs + r * DP + value_piece<DP>(r, pc) * 8 + (lane & 1) * 4;
          const u2v y = read_transposed(at);
          a[2 * u] = y[0];
          a[2 * u + 1] = y[1];
        }
        return a;
      };
      if (inner || !careful) {
#pragma unroll
        for (int sl = 0; sl < 4; ++sl)
#pragma unroll
          for (int j = 0; j < NB; ++j) o[j] = T::mma32(values(sl, j), pf[sl], o[j]);
      } else {
        unsigned odd = 0;
#pragma unroll
        for (int sl = 0; sl < 4; ++sl)
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            u4v a = values(sl, j);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const unsigned d = T::odd_bits(a[x]);
              odd |= d;
              a[x] &= ~((d >> 15) * 0xffffu);
            }
            o[j] = T::mma32(a, pf[sl], o[j]);
          }
        if (__any(odd != 0)) {
          for (int r = 0; r < kKeys; ++r) {
            const bool mine = see(place, key0 + r);
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int v = 0; v < 16; ++v) {
                const int ch = 32 * j + 8 * (v / 4) + 4 * hi + v % 4;
                const float x = (float)Vs[r * DP + value_piece<DP>(r, ch / 8) * 8 + ch % 8];
                if (mine && !(fabsf(x) < __builtin_inff())) o[j][v] += x;
              }
          }
        }
      }
    }

    L = across32(L, SumOp());
    bool odd = false;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) odd = odd || !(fabsf(o[j][v]) < __builtin_inff());
    if (!__syncthreads_or(odd)) break;
    }
    if (live) {
      const float inv = L != 0.0f ? 1.0f / L : 0.0f;  // a row that saw nothing is zero (NaN stays)
      E * out = static_cast<E *>(p.o) + (long)(q0 + row) * p.o_token + (long)head * p.o_head;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 4) {
          const int ch = 32 * j + 2 * v + 4 * hi;
          if (ch >= p.dim) continue;
          const u2v y = {pack2<TYPE>(o[j][v] * inv, o[j][v + 1] * inv), pack2<TYPE>(o[j][v + 2] * inv, o[j][v + 3] * inv)};
          *reinterpret_cast<u2v *>(out + ch) = y;
        }
    }
  }
}

namespace {

template <int TYPE, int DP> void launch_ragged(const RaggedParams & p, hipStream_t s)
{
  auto kern = ragged_attn_kernel<TYPE, DP>;
  const size_t lds = (size_t)4 * kKeys * DP * 2;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) throw std::runtime_error(std::string("HIP error: ") + hipGetErrorString(e));
  }
  // max_q only sizes the grid: a work-group takes every slots-th row block of its sequence.  A
  // launch holds 2^24 work-groups of 256 lanes.
  const long heads = (long)p.batch * p.heads;
  const int slots = (int)std::min<long>((std::max(1, std::min(p.max_q, p.tokens_q)) + kRows - 1) / kRows, (1L << 24) / (heads + kXcds * p.group));
  const long units = heads / p.group;
  const int round = units % kXcds == 0 || units >= 4 * kXcds;
  const long wgs = (round ? (units + kXcds - 1) / kXcds * kXcds : units) * p.group * slots;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(256), lds, s, p, slots, round);
}

template <int TYPE> void launch_ragged_dim(const RaggedParams & p, hipStream_t s)
{
  if (p.dim <= 32) launch_ragged<TYPE, 32>(p, s);
  else if (p.dim <= 64) launch_ragged<TYPE, 64>(p, s);
  else if (p.dim <= 96) launch_ragged<TYPE, 96>(p, s);
  else if (p.dim <= 128) launch_ragged<TYPE, 128>(p, s);
  else if (p.dim <= 192) launch_ragged<TYPE, 192>(p, s);
  else launch_ragged<TYPE, 256>(p, s);
}

}  // namespace

void launch_ragged_attention(const RaggedParams & p, hipStream_t s)
{
  if (p.type == kSeqF16) launch_ragged_dim<kSeqF16>(p, s);
  else launch_ragged_dim<kSeqBF16>(p, s);
}

}  // namespace ivh
