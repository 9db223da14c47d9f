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
#include <type_traits>

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

// ------------------------------------------------------------------ prompts, 64 tokens at a time
namespace {

typedef short s4v __attribute__((ext_vector_type(4)));

constexpr int kChunk = 64;
constexpr int kMaxSeg = 1 << 27;  // longer than any sequence: one segment each

// bits 2 and 3 swapped: with rows m of a product's first operand taken from channel (or token) turned(m), the 16 values
// of a lane in a 32 x 32 result are 8 (lane / 32) + 0 .. 7 and 16 more: two runs of 8, which are operands of the
// next product as they are
__device__ __forceinline__ int turned(int m) { return (m & 0x13) | (m & 4) << 1 | (m & 8) >> 1; }
// row of value v of a lane in such a result
__device__ __forceinline__ int result_row(int v, int half) { return (v & 7) + 8 * half + 2 * (v & 8); }

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

// The products x[i] y[i] in fp32 as sums of N 16-bit values each.
template <int TYPE, int N> __device__ __forceinline__ void split(f2v x, f2v y, unsigned (&part)[N])
{
  float a = x[0] * y[0], b = x[1] * y[1];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    part[i] = pack2<TYPE>(a, b);
    // what is left is taken from these very bits: the compiler would round the product a second time for it, in one
    // step from the unrounded one, which is now and then another value
    asm("" : "+v"(part[i]));
    const f2v z = unpack2<TYPE>(part[i]);
    a = a - z[0];
    b = b - z[1];
  }
}

// Segment `s` of the `n` of a sequence: its rows, and where its first state stands in the workspace.
struct Segment {
  int b, s, n, row, rows;
};
__device__ __forceinline__ Segment segment_of(const LinearParams & p, int u)
{
  auto first = [&](int i) { return (long)(min(max(p.cu[i], 0), p.tokens) / p.seg) + i; };
  const int b = find_seq(p.batch, u, first);
  const int c0 = min(max(p.cu[b], 0), p.tokens), rows = min(max(p.cu[b + 1], c0), p.tokens) - c0;
  const int s = u - (int)first(b), n = max(1, (rows + p.seg - 1) / p.seg);
  return Segment{b, s, n, c0 + s * p.seg, min(p.seg, rows - s * p.seg)};
}

}  // namespace

// DK: key channels rounded up to 64, 128 or 256.  OUT: outputs and the last state; else the state that each
// segment but the last adds to nothing, for linear_join_kernel.
template <int TYPE, int DK, bool OUT>
__global__ void __launch_bounds__(256, DK <= 128 ? 2 : 1) linear_chunk_kernel(const LinearParams p, int units, int blocks)
{
  using T = St<TYPE>;
  typedef typename T::e E;
  constexpr int ND = DK / 32;                              // 32-channel tiles of the state
  constexpr int QP = DK + 8, KP = DK + 16, VP = 128 + 16, PP = kChunk + 8;  // LDS rows, in elements
  constexpr int QI = kChunk * DK / 8 / 256, VI = kChunk * 128 / 8 / 256;     // 16-byte pieces of a thread
  constexpr int PARTS = TYPE == kSeqBF16 ? 3 : 2;          // 16-bit parts of a value with its decay: 24 and 22 bits
  __shared__ __attribute__((aligned(16))) E Q[OUT ? kChunk * QP : 8], K[kChunk * KP], V[kChunk * VP], P[OUT ? kChunk * PP : 8];
  __shared__ __attribute__((aligned(16))) f2v age[2][kChunk];             // log2 of the decay since the chunk's start, as a sum of two
  __shared__ float since[2][kChunk], left[2][kChunk], whole[2];  // that decay, from the row to the chunk's end, of all of it
  __shared__ float unit[2][kChunk];          // fp16: what a row's scores were divided by, for each half of the keys

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  // the work-groups of a segment's key head share an XCD, and its keys in that one's L2; key heads go round the XCDs
  const int each = p.group * blocks, w = blockIdx.x / kXcds, key = w / each * kXcds + blockIdx.x % kXcds;
  const int block = w % blocks, key_heads = p.heads / p.group, u = key / key_heads, kh = key - u * key_heads;
  const int h = kh * p.group + w % each / blocks;
  if (u >= units) return;
  const Segment seg = segment_of(p, u);
  if (seg.s < 0 || seg.s >= seg.n || (!OUT && seg.s == seg.n - 1)) return;
  const int in = p.from ? p.from[seg.b] : -1, out = p.to ? p.to[seg.b] : -1;
  const int n = seg.rows;
  const long one = (long)p.key_dim * p.dim;
  const int ch0 = block * 128 + 32 * wave;      // this wave's value channels
  const bool on = ch0 < p.dim;
  const int dv = ch0 + turned(col);             // this lane's column of the state
  float * first = p.ws + ((long)u * p.heads + h) * one;

  f16v s[ND];
  auto state_io = [&](float * at, auto store) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int dk = 32 * d + result_row(v, half);
        if (store) {
          if (dk < p.key_dim && dv < p.dim) at[(unsigned)(dk * p.dim + dv)] = s[d][v];
        } else {
          const float x = at[(unsigned)(min(dk, p.key_dim - 1) * p.dim + min(dv, p.dim - 1))];
          s[d][v] = dk < p.key_dim && dv < p.dim ? x : 0.0f;
        }
      }
  };
  constexpr std::integral_constant<bool, true> store{};
  constexpr std::integral_constant<bool, false> load{};
  auto begin = [&]() __attribute__((always_inline)) {
    if (OUT && seg.n > 1) {
      state_io(first, load);
    } else if (seg.s == 0 && (unsigned)in < (unsigned)p.slots) {
      state_io(p.state + ((long)in * p.heads + h) * one, load);
    } else {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[d][v] = 0.0f;
    }
  };
  if (on) begin();
  if (!OUT && seg.s == 0 && on) state_io(first, store);  // the slot may be written while other segments run

  const E * q = static_cast<const E *>(p.q) + (long)seg.row * p.q_token + (long)kh * p.q_head;
  const E * k = static_cast<const E *>(p.k) + (long)seg.row * p.k_token + (long)kh * p.k_head;
  const E * v = static_cast<const E *>(p.v) + (long)seg.row * p.v_token + (long)h * p.v_head + block * 128;
  const float * g = p.g + (long)seg.row * p.g_token + (long)h * p.g_head;
  E * o = static_cast<E *>(p.o) + (long)seg.row * p.o_token + (long)h * p.o_head + ch0;
  const int chunks = (n + kChunk - 1) / kChunk;

  u4v qr[QI], kr[QI], vr[VI];
  auto ask = [&](int c) __attribute__((always_inline)) {  // rows that are not there read the last one
#pragma unroll
    for (int i = 0; i < QI; ++i) {
      const int piece = tid + 256 * i, row = min(c * kChunk + piece / (DK / 8), n - 1), ch = min(piece % (DK / 8) * 8, p.key_dim - 8);
      if (OUT) qr[i] = *reinterpret_cast<const u4v *>(q + (long)row * p.q_token + ch);
      kr[i] = *reinterpret_cast<const u4v *>(k + (long)row * p.k_token + ch);
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int piece = tid + 256 * i, row = min(c * kChunk + piece / 16, n - 1), ch = min(piece % 16 * 8, p.dim - 8 - block * 128);
      vr[i] = *reinterpret_cast<const u4v *>(v + (long)row * p.v_token + ch);
    }
  };
  auto put = [&](int c) __attribute__((always_inline)) {
    const u4v zero = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < QI; ++i) {
      const int piece = tid + 256 * i, row = piece / (DK / 8), ch = piece % (DK / 8) * 8;
      const bool there = c * kChunk + row < n && ch < p.key_dim;
      if (OUT) *reinterpret_cast<u4v *>(Q + row * QP + ch) = there ? qr[i] : zero;
      *reinterpret_cast<u4v *>(K + row * KP + ch) = there ? kr[i] : zero;
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int piece = tid + 256 * i, row = piece / 16, ch = piece % 16 * 8;
      *reinterpret_cast<u4v *>(V + row * VP + ch) = c * kChunk + row < n && block * 128 + ch < p.dim ? vr[i] : zero;
    }
  };
  // Decays of chunk c, by one wave, a row a lane: sums of logarithms in 64 bits, since slow decays add up over thousands
  // of tokens and differences are taken.  A decay below 2^-256 is 0 whatever it multiplies.
  double total = 0.0;
  auto ask_decay = [&](int c) { return g[(long)min(c * kChunk + lane, n - 1) * p.g_token]; };
  auto decays = [&](int c, float its) __attribute__((always_inline)) {
    double x = c * kChunk + lane < n ? (double)its * 1.4426950408889634 : 0.0;
    x = x < -256.0 ? -256.0 : x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    const double end = __shfl(x, 63);
    const float hi = (float)x;
    age[c & 1][lane] = f2v{hi, (float)(x - (double)hi)};
    since[c & 1][lane] = (float)exp2(x);
    left[c & 1][lane] = (float)exp2(end - x);
    if (lane == 0) whole[c & 1] = (float)exp2(end);
    total += end;
  };

  // LDS offsets of this lane's pieces of transposed operands: 4 rows of 16 lanes, runs in the order of turned()
  const int run = 16 * (lane >> 4 & 1) + 4 * ((lane & 1) << 1 | (lane >> 1 & 1)), tr = 8 * half + (lane >> 2 & 3);
  const E * kt = K + tr * KP + run;
  const E * vt = V + tr * VP + 32 * wave + run;

  // of the chunk after next, asked for before the next one's rows: they are there when those are
  float next_decay = 0.0f;
  if (chunks > 0) {
    if (wave == 3) {
      const float its = ask_decay(0);
      next_decay = ask_decay(1);
      decays(0, its);
    }
    ask(0);
  }
  for (int c = 0; c < chunks; ++c) {
    put(c);
    __syncthreads();
    const float its_decay = next_decay;
    if (c + 1 < chunks) {
      if (wave == 3) next_decay = ask_decay(c + 2);
      ask(c + 1);
    }
    f16v acc[2];
    float fit = 1.0f;  // fp16: the state's power of two
    auto from_state = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[t][x] = 0.0f;
#pragma unroll
      for (int i = 0; i < 2 * ND; ++i) {
        u4v hi, lo;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          unsigned y[2];
          split<TYPE>(f2v{s[i / 2][8 * (i % 2) + 2 * x], s[i / 2][8 * (i % 2) + 2 * x + 1]}, f2v{fit, fit}, y);
          hi[x] = y[0];
          lo[x] = y[1];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const u4v y = *reinterpret_cast<const u4v *>(Q + (32 * t + col) * QP + 16 * i + 8 * half);
          acc[t] = T::mma32(hi, y, acc[t]);
          acc[t] = T::mma32(lo, y, acc[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float f = since[c & 1][32 * t + col] / fit;
#pragma unroll
        for (int x = 0; x < 16; ++x) acc[t][x] *= f;
      }
    };
    if constexpr (OUT) {
      // scores of a 32 x 32 part, keys in rows; of those above the diagonal none
      if (wave < 3) {
        const int t0 = wave ? 32 : 0, s0 = wave == 2 ? 32 : 0;
        f16v x;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i)
          x = T::mma32(*reinterpret_cast<const u4v *>(K + (s0 + turned(col)) * KP + 16 * i + 8 * half),
                       *reinterpret_cast<const u4v *>(Q + (t0 + col) * QP + 16 * i + 8 * half), x);
        const f2v mine = age[c & 1][t0 + col];
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const int row = s0 + result_row(i, half);
          const f4v its = *reinterpret_cast<const f4v *>(&age[c & 1][row]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool seen = row + e <= t0 + col;
            const float decay = __builtin_amdgcn_exp2f(seen ? (mine[0] - its[2 * e]) + (mine[1] - its[2 * e + 1]) : -200.0f);
            x[i + e] = (seen ? x[i + e] : 0.0f) * decay;
            if (TYPE == kSeqF16) most = fmaxf(most, fabsf(x[i + e]));
          }
        }
        if constexpr (TYPE == kSeqF16) {  // the largest of a row's to about 2^14, so that none overflows and small ones count
          most = across32(most, MaxOp());
          const int e = min(max(__builtin_amdgcn_frexp_expf(most) - 14, -40), 60);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = __builtin_ldexpf(x[i], -e);
          if (half == 0) unit[s0 / 32][t0 + col] = __builtin_ldexpf(1.0f, e);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<u4v *>(P + (t0 + col) * PP + s0 + 16 * i + 8 * half) =
              u4v{pack2<TYPE>(x[8 * i], x[8 * i + 1]), pack2<TYPE>(x[8 * i + 2], x[8 * i + 3]), pack2<TYPE>(x[8 * i + 4], x[8 * i + 5]),
                  pack2<TYPE>(x[8 * i + 6], x[8 * i + 7])};
      }
    }
    if (wave == 3 && c + 1 < chunks) decays(c + 1, its_decay);
    if constexpr (OUT) {
      if (on) {
        if constexpr (TYPE == kSeqF16) {
          float most = 0.0f;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int x = 0; x < 16; ++x) most = fmaxf(most, fabsf(s[d][x]));
#pragma unroll
          for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
          fit = __builtin_ldexpf(1.0f, min(max(14 - __builtin_amdgcn_frexp_expf(most), -100), 100));
        }
        from_state();
      }
      __syncthreads();
    }
    u4v vf[4];
    if (on) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u2v a = read_transposed(vt + 16 * j * VP), b = read_transposed(vt + (16 * j + 4) * VP);
        vf[j] = u4v{a[0], a[1], b[0], b[1]};
      }
    }
    if constexpr (OUT) {
      if (on) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float back = 1.0f;
#pragma unroll
          for (int y = 0; y <= t; ++y) {  // halves of the keys
            if constexpr (TYPE == kSeqF16) {
              const float mine = unit[y][32 * t + col], f = back / mine;
#pragma unroll
              for (int x = 0; x < 16; ++x) acc[t][x] *= f;
              back = mine;
            }
#pragma unroll
            for (int j = 2 * y; j < 2 * y + 2; ++j)
              acc[t] = T::mma32(vf[j], *reinterpret_cast<const u4v *>(P + (32 * t + col) * PP + 16 * j + 8 * half), acc[t]);
          }
          if constexpr (TYPE == kSeqF16)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[t][x] *= back;
        }
        // An infinity or NaN among the values reaches earlier rows of the chunk as 0 times it.  If a result is not
        // finite, the chunk's part is summed again over the keys that a row sees.
        bool odd = false;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 16; ++x) odd = odd || !(fabsf(acc[t][x]) < __builtin_inff());
        if (__any(odd)) {
          from_state();
#pragma unroll
          for (int t = 0; t < 2; ++t)
            for (int y = 0; y <= 32 * t + col; ++y) {
              float z = (float)P[(32 * t + col) * PP + y];
              if (TYPE == kSeqF16) z *= unit[y / 32][32 * t + col];
#pragma unroll
              for (int x = 0; x < 16; ++x) acc[t][x] = fmaf(z, (float)V[y * VP + 32 * wave + result_row(x, half)], acc[t][x]);
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int row = c * kChunk + 32 * t + col;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (row >= n || ch0 + 16 * i + 8 * half >= p.dim) continue;
            float y[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) y[x] = acc[t][8 * i + x] * p.scale;
            *reinterpret_cast<u4v *>(o + (long)row * p.o_token + 16 * i + 8 * half) =
                u4v{pack2<TYPE>(y[0], y[1]), pack2<TYPE>(y[2], y[3]), pack2<TYPE>(y[4], y[5]), pack2<TYPE>(y[6], y[7])};
          }
        }
      }
    }
    // the state: values with their decays to the chunk's end in parts of 16 bits, which together have fp32's precision
    if (on) {
      const float a = whole[c & 1];
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int x = 0; x < 16; ++x) s[d][x] *= a;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u4v part[PARTS];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = 16 * j + 8 * half + 2 * x;
          unsigned y[PARTS];
          split<TYPE>(unpack2<TYPE>(vf[j][x]), f2v{left[c & 1][row], left[c & 1][row + 1]}, y);
#pragma unroll
          for (int i = 0; i < PARTS; ++i) part[i][x] = y[i];
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const u2v a = read_transposed(kt + 16 * j * KP + 32 * d), b = read_transposed(kt + (16 * j + 4) * KP + 32 * d);
          const u4v x = {a[0], a[1], b[0], b[1]};
#pragma unroll
          for (int i = 0; i < PARTS; ++i) s[d] = T::mma32(x, part[i], s[d]);
        }
      }
    }
    __syncthreads();
  }
  if (!on) {
    if (!OUT && wave == 3 && lane == 0 && block == 0) p.decay[(long)u * p.heads + h] = (float)exp2(total);
    return;
  }
  if constexpr (OUT) {
    if (seg.s == seg.n - 1 && (unsigned)out < (unsigned)p.slots) state_io(p.state + ((long)out * p.heads + h) * one, store);
  } else {
    state_io(first + (long)p.heads * one, store);
    if (wave == 3 && lane == 0 && block == 0) p.decay[(long)u * p.heads + h] = (float)exp2(total);
  }
}

// The first states of a sequence's segments from those that the segments add: four elements a thread.
__global__ void __launch_bounds__(256) linear_join_kernel(const LinearParams p, int blocks)
{
  const long one = (long)p.key_dim * p.dim;
  const int block = blockIdx.x % blocks, h = blockIdx.x / blocks % p.heads, b = blockIdx.x / blocks / p.heads;
  const int c0 = min(max(p.cu[b], 0), p.tokens), rows = min(max(p.cu[b + 1], c0), p.tokens) - c0;
  const int n = (rows + p.seg - 1) / p.seg;
  const long u = (long)(c0 / p.seg) + b, i = 4L * (block * 256 + threadIdx.x);
  if (n < 3 || i >= one) return;
  float * at = p.ws + (u * p.heads + h) * one + i;
  f4v x = *reinterpret_cast<const f4v *>(at + p.heads * one);
#pragma unroll 4
  for (int s = 2; s < n; ++s) {
    const float a = p.decay[(u + s - 1) * p.heads + h];
    f4v y = *reinterpret_cast<const f4v *>(at + s * p.heads * one);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = fmaf(a, x[j], y[j]);
    *reinterpret_cast<f4v *>(at + s * p.heads * one) = x;
  }
}

namespace {

template <int TYPE, int DK> void launch_linear_chunks(const LinearParams & p, hipStream_t s)
{
  const int blocks = (p.dim + 127) / 128;
  const int units = p.tokens / p.seg + p.batch;
  const long keys = (long)units * (p.heads / p.group);
  const dim3 grid((unsigned)((keys + kXcds - 1) / kXcds * kXcds * p.group * blocks)), blk(256);
  if (p.ws) {
    hipLaunchKernelGGL((linear_chunk_kernel<TYPE, DK, false>), grid, blk, 0, s, p, units, blocks);
    const int parts = (p.key_dim * p.dim + 1023) / 1024;
    hipLaunchKernelGGL(linear_join_kernel, dim3((unsigned)((long)p.batch * p.heads * parts)), blk, 0, s, p, parts);
  }
  hipLaunchKernelGGL((linear_chunk_kernel<TYPE, DK, true>), grid, blk, 0, s, p, units, blocks);
}

template <int TYPE> void launch_linear_type(const LinearParams & p, hipStream_t s)
{
  if (p.seg > 0) {
    if (p.key_dim <= 64) launch_linear_chunks<TYPE, 64>(p, s);
    else if (p.key_dim <= 128) launch_linear_chunks<TYPE, 128>(p, s);
    else launch_linear_chunks<TYPE, 256>(p, s);
    return;
  }
  const int blocks = (p.dim + 31) / 32;
  const dim3 grid((unsigned)((long)p.batch * p.heads * blocks)), blk(kStepThreads);
  if (p.key_dim <= 64) hipLaunchKernelGGL((linear_step_kernel<TYPE, 32, 2>), grid, blk, 0, s, p, blocks);
  else if (p.key_dim <= 128) hipLaunchKernelGGL((linear_step_kernel<TYPE, 32, 4>), grid, blk, 0, s, p, blocks);
  else hipLaunchKernelGGL((linear_step_kernel<TYPE, 32, 8>), grid, blk, 0, s, p, blocks);
}

}  // namespace

size_t linear_split(LinearParams & p, int max_new)
{
  p.seg = 0;
  if (max_new <= 16) return 0;
  const long blocks = (p.dim + 127) / 128;
  const long each = (long)p.tokens * p.heads * blocks / 512;
  p.seg = (int)((std::max<long>(each, 512) + kChunk - 1) / kChunk * kChunk);
  if (max_new <= 2 * p.seg) {
    p.seg = (max_new + kChunk - 1) / kChunk * kChunk;
    p.seg = kMaxSeg;
    return 0;
  }
  return ((size_t)p.tokens / p.seg + p.batch) * p.heads * ((size_t)p.key_dim * p.dim + 1) * sizeof(float);
}

void launch_linear_attention(const LinearParams & p, hipStream_t s)
{
  if (p.type == kSeqF16) launch_linear_type<kSeqF16>(p, s);
  else launch_linear_type<kSeqBF16>(p, s);
}

}  // namespace ivh
