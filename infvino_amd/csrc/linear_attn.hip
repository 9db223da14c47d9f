// Linear attention with a decay for each head, on gfx950.
//
//   S <- a_t S + k_t^T v_t,  o_t = scale q_t S,  a_t = exp(g_t)
//
// Few new tokens (the recurrence): a state is read, taken through its tokens in registers, and
// written, 8 key_dim dim bytes of HBM for 4 key_dim dim operations a token: HBM bounds it.  A
// work-group has `DV` value channels of one head: a thread 4 of them and every (1024 / DV)-th key channel.  The sums
// over the key channels meet by lane exchanges and through LDS, which two copies of keep at one barrier a
// token.
#include <algorithm>
#include <cmath>
#include <stdexcept>

#include "conv_common.hpp"
#include "seq_common.hpp"

namespace ivh {

namespace {

constexpr int kStepThreads = 256;

// exp(g) of a decay's logarithm
__device__ __forceinline__ float decay_of(float g) { return __builtin_amdgcn_exp2f(g * kLog2E); }

}  // namespace

// DV: value channels of a work-group, NR: key channels of a thread
template <int TYPE, int DV, int NR>
__global__ void __launch_bounds__(kStepThreads) linear_step_kernel(const LinearParams p, int blocks)
{
  typedef typename St<TYPE>::e E;
  constexpr int LANES = DV / 4, ROWS = kStepThreads / LANES;  // threads side by side, key channels at a time
  __shared__ __attribute__((aligned(16))) float qs[2][256], ks[2][256];
  __shared__ __attribute__((aligned(16))) float part[2][4 * DV];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = tid % LANES, r = tid / LANES;
  const int block = blockIdx.x % blocks, w = blockIdx.x / blocks, h = w % p.heads, b = w / p.heads;
  const int c0 = min(max(p.cu[b], 0), p.tokens), n = min(max(p.cu[b + 1], c0), p.tokens) - c0;
  const int in = p.from ? p.from[b] : -1, out = p.to ? p.to[b] : -1;
  const bool has = (unsigned)in < (unsigned)p.slots, keep = (unsigned)out < (unsigned)p.slots;
  const int ch = block * DV + 4 * c;  // this thread's value channels
  const bool live = ch < p.dim;
  const int kh = h / p.group;

  const long one = (long)p.key_dim * p.dim;
  f4v s[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int d = r + ROWS * i;
    s[i] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
    if (has && live && d < p.key_dim) s[i] = *reinterpret_cast<const f4v *>(p.state + ((long)in * p.heads + h) * one + (long)d * p.dim + ch);
  }
  const E * q = static_cast<const E *>(p.q) + (long)c0 * p.q_token + (long)kh * p.q_head;
  const E * k = static_cast<const E *>(p.k) + (long)c0 * p.k_token + (long)kh * p.k_head;
  const E * v = static_cast<const E *>(p.v) + (long)c0 * p.v_token + (long)h * p.v_head + ch;
  const float * g = p.g + (long)c0 * p.g_token + (long)h * p.g_head;
  E * o = static_cast<E *>(p.o) + (long)c0 * p.o_token + (long)h * p.o_head + ch;
  for (int t = 0; t < n; ++t) {
    const int at = t & 1;
    if (tid < p.key_dim) {
      qs[at][tid] = (float)q[(long)t * p.q_token + tid];
      ks[at][tid] = (float)k[(long)t * p.k_token + tid];
    }
    const float a = decay_of(g[(long)t * p.g_token]);
    f4v x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
      const u2v y = *reinterpret_cast<const u2v *>(v + (long)t * p.v_token);
      const f2v lo = unpack2<TYPE>(y[0]), hi = unpack2<TYPE>(y[1]);
      x = f4v{lo[0], lo[1], hi[0], hi[1]};
    }
    __syncthreads();
    f4v sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int d = r + ROWS * i;
      if (d >= p.key_dim) continue;
      const float kd = ks[at][d], qd = qs[at][d];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = fmaf(kd, x[j], a * s[i][j]);
        sum[j] = fmaf(qd, s[i][j], sum[j]);
      }
    }
#pragma unroll
    for (int step = LANES; step < 64; step *= 2)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += __shfl_xor(sum[j], step);
    if (lane < LANES) *reinterpret_cast<f4v *>(&part[at][wave * DV + 4 * c]) = sum;
    __syncthreads();
    if (tid < LANES && live) {
#pragma unroll
      for (int i = 1; i < 4; ++i) sum += *reinterpret_cast<const f4v *>(&part[at][i * DV + 4 * c]);
      sum *= p.scale;
      *reinterpret_cast<u2v *>(o + (long)t * p.o_token) = u2v{pack2<TYPE>(sum[0], sum[1]), pack2<TYPE>(sum[2], sum[3])};
    }
  }
  if (!keep || !live) return;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int d = r + ROWS * i;
    if (d < p.key_dim) *reinterpret_cast<f4v *>(p.state + ((long)out * p.heads + h) * one + (long)d * p.dim + ch) = s[i];
  }
}

namespace {

template <int TYPE> void launch_linear_type(const LinearParams & p, hipStream_t s)
{
  const int blocks = (p.dim + 31) / 32;
  const dim3 grid((unsigned)((long)p.batch * p.heads * blocks)), blk(kStepThreads);
  if (p.key_dim <= 64) hipLaunchKernelGGL((linear_step_kernel<TYPE, 32, 2>), grid, blk, 0, s, p, blocks);
  else if (p.key_dim <= 128) hipLaunchKernelGGL((linear_step_kernel<TYPE, 32, 4>), grid, blk, 0, s, p, blocks);
  else hipLaunchKernelGGL((linear_step_kernel<TYPE, 32, 8>), grid, blk, 0, s, p, blocks);
}

}  // namespace

void launch_linear_attention(const LinearParams & p, hipStream_t s)
{
  if (p.type == kSeqF16) launch_linear_type<kSeqF16>(p, s);
  else launch_linear_type<kSeqBF16>(p, s);
}

}  // namespace ivh
