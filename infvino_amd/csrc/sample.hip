// The next token of each row of logits: temperature, top-k, top-p, min-p, and the inverse of what is left
// at a given random number, on gfx950.
//
// Weights w = exp((x - max) / T) are whole multiples of 2^-44: their sums over up to 2^19 tokens fit in
// 63 bits and are the same in any order, so cuts and draws do not depend on how a row is split, and no atomic's
// order can change a token.  A weight below 2^-45 of the largest is 0.  The exponential is formed in 64 bits to 2^-50.
#include <cmath>
#include <stdexcept>

#include "conv_common.hpp"
#include "seq_common.hpp"

namespace ivh {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr double kOne = 17592186044416.0;  // 2^44, the largest weight
constexpr u64 kAll = 1ull << 63;           // no sum is larger

template <int TYPE> struct Logit;
template <> struct Logit<kSeqF16> { typedef _Float16 e; };
template <> struct Logit<kSeqBF16> { typedef __bf16 e; };
template <> struct Logit<kSeqF32> { typedef float e; };

// an order-preserving code of x: NaN as -infinity, -0 as 0
__device__ __forceinline__ unsigned code_of(float x)
{
  if (!(x == x)) x = -__builtin_inff();
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned code) { return __builtin_bit_cast(float, code & 0x80000000u ? code & 0x7fffffffu : ~code); }
constexpr unsigned kNone = 0x007fffffu;  // of -infinity

// the weight of a token in units of 2^-44; scale: log2 e / T in 64 bits
__device__ __forceinline__ u64 weight_of(unsigned code, unsigned top, double scale)
{
  if (code == top) return (u64)kOne;
  if (code <= kNone) return 0;
  const double z = ((double)value_of(code) - (double)value_of(top)) * scale;
  if (!(z > -46.0)) return 0;
  return (u64)rint(exp2(z) * kOne);
}

struct Cut {
  unsigned code;  // kept: codes above, and the first `ties` of this one
  unsigned ties;
  u64 sum;        // of what is kept
};

}  // namespace

template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p)
{
  typedef typename Logit<TYPE>::e E;
  __shared__ unsigned count[256];
  __shared__ u64 sums[256];
  __shared__ unsigned wave_u[16], sh_need_n;
  __shared__ u64 wave_s[16], sh_need_s, sh_above_s;
  __shared__ unsigned sh_above_n;
  __shared__ int sh_at;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
  const E * x = static_cast<const E *>(p.x) + (long)row * p.row;
  const int n = p.vocab;

  // the largest and its first place
  unsigned top = 0;
  int at = n;
  for (int i = tid; i < n; i += kThreads) {
    const unsigned c = code_of((float)x[i]);
    if (c > top) {
      top = c;
      at = i;
    }
  }
  for (int d = 32; d >= 1; d /= 2) {
    const unsigned c = __shfl_xor(top, d);
    const int j = __shfl_xor(at, d);
    if (c > top || (c == top && j < at)) {
      top = c;
      at = j;
    }
  }
  if (lane == 0) {
    wave_u[wave] = top;
    wave_s[wave] = (u64)at;
  }
  __syncthreads();
  for (int i = 0; i < 16; ++i) {
    const unsigned c = wave_u[i];
    const int j = (int)wave_s[i];
    if (c > top || (c == top && j < at)) {
      top = c;
      at = j;
    }
  }
  __syncthreads();
  const float t = p.temperature ? p.temperature[row] : 1.0f;
  if (top <= kNone || !(t > 0.0f)) {
    if (tid == 0) p.token[row] = top <= kNone ? -1 : at;
    return;
  }
  const double scale = 1.4426950408889634 / (double)t;

  // the shortest prefix of the descending order that has need_n tokens or a sum of need_s, by digits of the code
  auto descend = [&](unsigned need_n, u64 need_s) {
    unsigned prefix = 0, above_n = 0;
    u64 above_s = 0;
    Cut cut = {0, 0, 0};
    for (int digit = 3; digit >= 0; --digit) {
      for (int i = tid; i < 256; i += kThreads) {
        count[i] = 0;
        sums[i] = 0;
      }
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const unsigned c = code_of((float)x[i]);
        if (digit < 3 && c >> (8 * digit + 8) != prefix) continue;
        const u64 w = weight_of(c, top, scale);
        if (w == 0) continue;
        atomicAdd(&count[c >> (8 * digit) & 255], 1u);
        atomicAdd(&sums[c >> (8 * digit) & 255], w);
      }
      __syncthreads();
      if (tid == 0) {
        int found = -1;
        for (int i = 255; i >= 0; --i) {
          if (count[i] == 0) continue;
          found = i;
          if (above_n + count[i] >= need_n || above_s + sums[i] >= need_s) break;
          above_n += count[i];
          above_s += sums[i];
          found = -1;
        }
        sh_at = found;
        sh_above_n = above_n;
        sh_above_s = above_s;
        if (found >= 0) {
          sh_need_n = count[found];
          sh_need_s = sums[found];
        }
      }
      __syncthreads();
      above_n = sh_above_n;
      above_s = sh_above_s;
      const int found = sh_at;
      if (found < 0) return Cut{0, 0, above_s};  // all are kept
      prefix = prefix << 8 | (unsigned)found;
      if (digit == 0) {
        const u64 w = weight_of(prefix, top, scale);
        u64 ties = sh_need_n;
        ties = min(ties, (u64)(need_n - above_n));
        if (need_s > above_s) ties = min(ties, (need_s - above_s + w - 1) / w);
        cut = Cut{prefix, (unsigned)ties, above_s + ties * w};
      }
      __syncthreads();
    }
    return cut;
  };
  const int k = p.top_k ? p.top_k[row] : 0;
  Cut cut = descend(k > 0 ? (unsigned)k : 0xffffffffu, kAll);
  const float tp = p.top_p ? p.top_p[row] : 1.0f, mp = p.min_p ? p.min_p[row] : 0.0f;
  if (tp < 1.0f) {
    const double need = ceil(fmax((double)tp, 0.0) * (double)cut.sum);
    cut = descend(0xffffffffu, max((u64)need, (u64)1));
  }
  const u64 least = mp > 0.0f ? (u64)ceil((double)fminf(mp, 1.0f) * kOne) : 1;

  // the kept weights in the order of the vocabulary: their sum, then the token at u of it
  const float u = p.u[row];
  u64 total = 0, goal = 0;
  for (int pass = 0; pass < 2; ++pass) {
    u64 before_s = 0;
    unsigned before_n = 0;
    if (tid == 0) sh_at = -1;
    for (int base = 0; base < n; base += kThreads) {
      const int i = base + tid;
      const unsigned c = i < n ? code_of((float)x[i]) : 0;
      u64 w = weight_of(c, top, scale);
      if (w < least || c < cut.code) w = 0;
      const bool tie = w != 0 && c == cut.code;
      const unsigned long long ties = __ballot(tie);
      if (lane == 0) wave_u[wave] = __popcll(ties);
      __syncthreads();
      unsigned rank = before_n + __popcll(ties & ((1ull << lane) - 1));
      for (int j = 0; j < 16; ++j) {
        if (j < wave) rank += wave_u[j];
        before_n += wave_u[j];
      }
      if (tie && rank >= cut.ties) w = 0;
      u64 run = w;
      for (int d = 1; d < 64; d *= 2) {
        const u64 y = __shfl_up(run, d);
        if (lane >= d) run += y;
      }
      if (lane == 63) wave_s[wave] = run;
      __syncthreads();
      u64 mine = before_s + run;
      for (int j = 0; j < 16; ++j) {
        if (j < wave) mine += wave_s[j];
        before_s += wave_s[j];
      }
      if (pass == 1 && w != 0 && mine > goal && mine - w <= goal) p.token[row] = i;
      __syncthreads();
    }
    if (pass == 0) {
      total = before_s;
      goal = u > 0.0f ? (u < 1.0f ? min((u64)((double)u * (double)total), total - 1) : total - 1) : 0;
    }
  }
}

void launch_sample(const SampleParams & p, hipStream_t s)
{
  const dim3 grid((unsigned)p.rows), blk(kThreads);
  if (p.type == kSeqF16) hipLaunchKernelGGL((sample_kernel<kSeqF16>), grid, blk, 0, s, p);
  else if (p.type == kSeqBF16) hipLaunchKernelGGL((sample_kernel<kSeqBF16>), grid, blk, 0, s, p);
  else hipLaunchKernelGGL((sample_kernel<kSeqF32>), grid, blk, 0, s, p);
}

}  // namespace ivh
