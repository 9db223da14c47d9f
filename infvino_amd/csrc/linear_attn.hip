// Linear attention with a decay for each head, on gfx950.
//
//   S <- a_t S + k_t^T v_t,  o_t = scale q_t S,  a_t = exp(g_t)
//
// Few new tokens (the recurrence): a state is read, taken through its tokens in registers, and
// written, 8 key_dim dim bytes of HBM for 4 key_dim dim operations a token: HBM bounds it.  A
// work-group has `DV` value channels of one head: a thread 4 of them and every (1024 / DV)-th key channel.  The sums
// over the key channels meet by lane exchanges and through LDS, two barriers a token; two copies of what LDS holds keep the next token's
// rows from waiting for the last one's sums.  96 sequences of 32 heads of 128 x 128, a token each: 84 us, 4.8 TB/s.
//
// Many (chunks of 64 rows): with b_t the sum of the chunk's g up to t,
//
//   o_t = scale (e^(b_t) q_t S0 + sum_{s <= t} e^(b_t - b_s) (q_t k_s) v_s),  S' = e^(b_63) S0 + sum_s e^(b_63 - b_s) k_s^T v_s
//
// are matrix products.  A work-group has up to 128 value channels of a head, a wave 32 of them and all key channels: the state
// stays in a wave's accumulators, and values with their decays enter the last in three bf16 or two fp16 parts, so that states, which
// hand their errors on, keep the precision of fp32 products.  What only an output sees is held to fewer bits: S0 enters the first
// product in two 16-bit parts (16 bits in bf16, off by 2^-17, a 512th of half a step of the output; a third part would be half of that
// product's matrix work again), and scores are rounded to the storage type once, as the weights of the softmax
// attention are (off by half a step each, independently, where the output's own rounding is half a step of the sum): an operand
// of the matrix cores has 16 bits.  fp16's range is too small for states, values with decays and scores: columns of the first two and
// rows of the last are held times powers of two, which follow what they meet.  Chunks follow one another, which leaves
// little to hide latency behind: the next chunk's rows come by LDS DMA while this one is worked on, over barriers that do not
// wait for them.  A long sequence is cut into segments: what each adds to a state that begins with
// nothing, the first states from those, then the outputs of all at once.  It costs a second pass over keys and
// values and pays where sequences do not fill the chip.  Ragged prompts of 16 heads of 64 x 96 in fp16 93 us (in a trace the median of
// states is 28.6, of the join 5.4, of outputs 65.5), a long one of 32 heads of 128 x 128 225 (at best 70, 10 and 136; in a trace, whose calls
// follow one another less closely, medians of 87, 12 and 176); by single tokens 4240 and 17160.
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
typedef __attribute__((address_space(3))) void lds_ptr;

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

// Rows of LDS hold no padding, since copies write 64 x 16 bytes one behind the other; 16-byte pieces are permuted within a
// row instead, piece c of row r to c ^ order(r), so that the lanes that are served together lie in distinct banks:
// queries are read a row a lane, values four rows of 16 lanes, keys both ways.
__device__ __forceinline__ int query_order(int r) { return r & 15; }
__device__ __forceinline__ int key_order(int r) { return (r & 3) << 1 | (r >> 3 & 1) | (r >> 2 & 1) << 3; }
__device__ __forceinline__ int value_order(int r) { return (r & 3) << 1; }

// 64 x 16 bytes straight into LDS: lane i's from the buffer r at its offset, zeros outside it, to `to` + 16 i.  In
// assembler, and with barriers that wait for no copy, so that copies stay in flight: the compiler would wait for all of
// them at a barrier and before each transposing read.  Five wait states, which it does not count in assembler: r may have been
// written by the vector unit just before.
__device__ __forceinline__ void copy_to_lds(u4v r, unsigned off, void * to)
{
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(off), "s"(r), "s"((unsigned)(unsigned long)(lds_ptr *)to)
               : "memory", "m0");
#endif
}
__device__ __forceinline__ void wait_for_copies()
{
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(vm_wait(0));  // the compiler's own: it knows by it that its loads are there too
  asm volatile("" ::: "memory");
#endif
}
__device__ __forceinline__ void lds_barrier()
{
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#endif
}

// DK: key channels rounded up to 64, 128 or 256.  OUT: outputs and the last state; else the state that each
// segment but the last adds to nothing, for linear_join_kernel.
template <int TYPE, int DK, bool OUT>
__global__ void __launch_bounds__(256, DK <= 128 ? 2 : 1) linear_chunk_kernel(const LinearParams p, int units, int blocks)
{
  using T = St<TYPE>;
  typedef typename T::e E;
  constexpr int ND = DK / 32;                      // 32-channel tiles of the state
  constexpr int PK = DK / 8, MK = PK < 16 ? PK - 1 : 15;  // 16-byte pieces of a key row, and those that are permuted among themselves
  constexpr int PP = kChunk + 8;                   // elements of a row of scores
  constexpr int PARTS = TYPE == kSeqBF16 ? 3 : 2;  // 16-bit parts of a value with its decay: 24 and 22 bits
  // Arrays of their own, so that the compiler sees which copy a read waits for.  Keys are read to the end of a chunk and
  // have two; queries are done with, and values in registers, in the middle of it, when the next ones are asked for.
  __shared__ __attribute__((aligned(16))) unsigned char K0[kChunk * DK * 2], K1[kChunk * DK * 2], V0[kChunk * 256];
  __shared__ __attribute__((aligned(16))) unsigned char Q[OUT ? kChunk * DK * 2 : 16], V1[OUT ? 16 : kChunk * 256];
  __shared__ __attribute__((aligned(16))) E P[OUT ? kChunk * PP : 8];
  struct Decays {
    f2v age[2][kChunk];     // log2 of the decay since the chunk's start, as a sum of two
    float left[2][kChunk];  // the decay from the row to the chunk's end,
    float since[2][kChunk], whole[2];  // since its start, and of all of it
    float unit[2][kChunk];  // fp16: what a row's scores were divided by, for each half of the keys
  };
  __shared__ __attribute__((aligned(16))) Decays its;

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
  const int n = __builtin_amdgcn_readfirstlane(seg.rows), row0 = __builtin_amdgcn_readfirstlane(seg.row);
  const long one = (long)p.key_dim * p.dim;
  const int ch0 = block * 128 + 32 * wave;      // this wave's value channels
  const bool on = ch0 < p.dim;
  const int dv = ch0 + turned(col);             // this lane's column of the state
  float * first = p.ws + ((long)u * p.heads + h) * one;

  f16v s[ND];
  int held = 0;  // fp16: the column is held times 2^held, so that the parts below are normal numbers
  auto state_io = [&](float * at, auto store) __attribute__((always_inline)) {  // channels that are not there: zeros, nowhere
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(at, (short)0, (int)(one * 4), kBufDword3);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int dk = 32 * d + result_row(v, half);
        const unsigned off = dv < p.dim ? (unsigned)(dk * p.dim + dv) * 4u : kBufOOB;  // rows from key_dim on lie behind the end
        const float x = TYPE == kSeqF16 ? __builtin_ldexpf(s[d][v], -held) : s[d][v];  // by itself: a bit cast of an element is one of the vector's start
        if (store) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), r, (int)off, 0, 0);
        else s[d][v] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0));
      }
  };
  constexpr std::integral_constant<bool, true> store{};
  constexpr std::integral_constant<bool, false> load{};
  constexpr std::integral_constant<int, 0> even{};
  constexpr std::integral_constant<int, 1> odd_one{};

  const E * q = static_cast<const E *>(p.q) + (long)row0 * p.q_token + (long)kh * p.q_head;
  const E * k = static_cast<const E *>(p.k) + (long)row0 * p.k_token + (long)kh * p.k_head;
  const E * v = static_cast<const E *>(p.v) + (long)row0 * p.v_token + (long)h * p.v_head + block * 128;
  const float * g = p.g + (long)row0 * p.g_token + (long)h * p.g_head;
  E * o = static_cast<E *>(p.o) + (long)row0 * p.o_token + (long)h * p.o_head + ch0;
  const int chunks = (n + kChunk - 1) / kChunk, width = min(128, p.dim - block * 128);

  // what this lane copies: position pos of a row holds a piece of it; channels and rows that are not there become zeros (rows
  // may lie on top of one another: the buffer's end alone would let in parts of others)
  auto copy = [&](const E * at, long token, int channels, int c, auto pieces, auto order, unsigned char * to) __attribute__((always_inline)) {
    const int rows = min(n - c * kChunk, kChunk);
    const unsigned bytes = (unsigned)((rows - 1) * (int)token + channels) * 2u;
    const unsigned long base = reinterpret_cast<unsigned long>(at + (long)c * kChunk * token);
    const u4v r = {(unsigned)__builtin_amdgcn_readfirstlane((int)base), (unsigned)__builtin_amdgcn_readfirstlane((int)(base >> 32)),
                   (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), (unsigned)kBufDword3};
#pragma unroll
    for (int i = 0; i < pieces / 4; ++i) {
      const int at16 = 64 * (wave + 4 * i) + lane, row = at16 / pieces, ch = (at16 % pieces ^ order(row)) * 8;
      const unsigned off = ch < channels && row < rows ? (unsigned)(row * (int)token + ch) * 2u : kBufOOB;
      copy_to_lds(r, off, to + 1024 * (wave + 4 * i));
    }
  };
  constexpr std::integral_constant<int, PK> key_pieces{};
  constexpr std::integral_constant<int, 16> value_pieces{};
  auto copy_q = [&](int c) __attribute__((always_inline)) { copy(q, p.q_token, p.key_dim, c, key_pieces, [](int r) { return query_order(r) & MK; }, Q); };
  auto copy_k = [&](int c, auto side) __attribute__((always_inline)) {
    copy(k, p.k_token, p.key_dim, c, key_pieces, [](int r) { return key_order(r) & MK; }, side == 0 ? K0 : K1);
  };
  auto copy_v = [&](int c, auto side) __attribute__((always_inline)) {
    copy(v, p.v_token, width, c, value_pieces, [](int r) { return value_order(r); }, side == 0 ? V0 : V1);
  };

  // Decays of chunk c, by one wave, a row a lane: sums of logarithms in 64 bits, since slow decays add up over thousands
  // of tokens and differences are taken.  A decay below 2^-4096 is held as that: 0 whatever it multiplies, also after 64 tokens
  // whose decays are above 1.
  double total = 0.0;
  auto ask_decay = [&](int c) { return g[(long)min(c * kChunk + lane, n - 1) * p.g_token]; };
  auto decays = [&](int c, float log_decay) __attribute__((always_inline)) {
    double x = c * kChunk + lane < n ? (double)log_decay * 1.4426950408889634 : 0.0;
    x = x < -4096.0 ? -4096.0 : x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    const double end = __shfl(x, 63);
    const float hi = (float)x;
    its.age[c & 1][lane] = f2v{hi, (float)(x - (double)hi)};
    its.since[c & 1][lane] = (float)exp2(x);
    its.left[c & 1][lane] = (float)exp2(end - x);
    if (lane == 0) its.whole[c & 1] = (float)exp2(end);
    total += end;
  };

  // LDS byte offsets of this lane's fragments: of channels 16 i + 8 half of a row, whose permuted bits an exclusive or
  // sets, and of transposed operands: 4 rows of 16 lanes, runs in the order of turned()
  const int krow = turned(col), run = (lane & 1) << 1 | (lane >> 1 & 1), tr = lane >> 2 & 3, side16 = lane >> 4 & 1;
  const unsigned qat = (unsigned)(col * DK * 2 + ((half ^ query_order(col)) & MK) * 16);
  const unsigned kat = (unsigned)(krow * DK * 2 + ((half ^ key_order(krow)) & MK) * 16);
  const unsigned ktr = (unsigned)((8 * half + tr) * DK * 2 + (((2 * side16 + (run >> 1)) ^ key_order(8 * half + tr)) & MK) * 16 + (run & 1) * 8);
  const unsigned vtr = (unsigned)((8 * half + tr) * 256 + ((4 * wave + 2 * side16 + (run >> 1)) ^ value_order(tr)) * 16 + (run & 1) * 8);
  auto piece = [&](const unsigned char * rows, unsigned at, int i) __attribute__((always_inline)) {  // i: 32-byte steps
    return *reinterpret_cast<const u4v *>(rows + (at ^ (unsigned)(2 * i & MK) * 16u) + (unsigned)(2 * i & ~MK) * 16u);
  };
  // 16 tokens from 16 j on of channels 32 d ..
  auto keys_of = [&](const unsigned char * rows, int j, int d) __attribute__((always_inline)) {
    const unsigned low = (unsigned)(4 * d & MK) * 16u, high = (unsigned)(4 * d & ~MK) * 16u, flip = (unsigned)(8 & MK) * 16u;
    const u2v x = read_transposed(rows + (ktr ^ low) + high + 16 * j * DK * 2), y = read_transposed(rows + (ktr ^ low ^ flip) + high + (16 * j + 4) * DK * 2);
    return u4v{x[0], x[1], y[0], y[1]};
  };
  auto values_of = [&](const unsigned char * rows, int j) __attribute__((always_inline)) {
    const u2v x = read_transposed(rows + vtr + 16 * j * 256), y = read_transposed(rows + vtr + (16 * j + 4) * 256);
    return u4v{x[0], x[1], y[0], y[1]};
  };

  // of the chunk after next, asked for before the next one's rows: they are there when those are
  float next_decay = 0.0f;
  if (chunks > 0) {
    float log_decay = 0.0f;
    if (wave == 3) {
      log_decay = ask_decay(0);
      next_decay = ask_decay(1);
    }
    copy_k(0, even);
    if (OUT) copy_q(0);
    copy_v(0, even);
    if (wave == 3) decays(0, log_decay);
  }
  if (on) {
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
    if (!OUT && seg.s == 0) state_io(first, store);  // the slot may be written while other segments run
  }
  wait_for_copies();
  lds_barrier();

  auto chunk = [&](int c, auto side) __attribute__((always_inline)) {
    constexpr int SIDE = decltype(side)::value;
    constexpr std::integral_constant<int, 1 - SIDE> other{};
    const unsigned char * K = SIDE == 0 ? K0 : K1;
    const bool more = c + 1 < chunks;
    const float decay_then = next_decay;
    if (more) {
      if (wave == 3) next_decay = ask_decay(c + 2);
      copy_k(c + 1, other);
      if (!OUT) copy_v(c + 1, other);
    }
    f16v acc[2];
    float fit = 1.0f, back = 1.0f;  // fp16: what brings this lane's column of the state to about 2^14, and what it comes back by
    float top = 0.0f;               // fp16: the column's largest, as it is held
    auto from_state = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) acc[t] = f16v{};
#pragma unroll
      for (int i = 0; i < 2 * ND; ++i) {
        u4v part[2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          unsigned y[2];
          split<TYPE>(f2v{s[i / 2][8 * (i % 2) + 2 * x], s[i / 2][8 * (i % 2) + 2 * x + 1]}, f2v{fit, fit}, y);
          part[0][x] = y[0];
          part[1][x] = y[1];
        }
        const u4v y0 = piece(Q, qat, i), y1 = piece(Q + 32 * DK * 2, qat, i);
        acc[0] = T::mma32(part[0], y0, acc[0]);
        acc[1] = T::mma32(part[0], y1, acc[1]);
        acc[0] = T::mma32(part[1], y0, acc[0]);
        acc[1] = T::mma32(part[1], y1, acc[1]);
      }
      const float f0 = its.since[SIDE][col], f1 = its.since[SIDE][32 + col];
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float y = TYPE == kSeqF16 ? __shfl(back, turned(result_row(x, half))) : 1.0f;
        acc[0][x] *= f0 * y;
        acc[1][x] *= f1 * y;
      }
    };
    u4v vf[4], y[4];
    unsigned odd_row = kChunk;
    bool odd = false;
    if constexpr (OUT) {
      // scores of a 32 x 32 part, keys in rows; of those above the diagonal none
      if (wave < 3) {
        const int t0 = wave ? 32 : 0, s0 = wave == 2 ? 32 : 0;
        f16v x = {};
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i) x = T::mma32(piece(K + s0 * DK * 2, kat, i), piece(Q + t0 * DK * 2, qat, i), x);
        const f2v mine = its.age[SIDE][t0 + col];
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const int row = s0 + result_row(i, half);
          const f4v key = *reinterpret_cast<const f4v *>(&its.age[SIDE][row]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool seen = row + e <= t0 + col;
            const float decay = __builtin_amdgcn_exp2f(seen ? (mine[0] - key[2 * e]) + (mine[1] - key[2 * e + 1]) : -200.0f);
            x[i + e] = (seen ? x[i + e] : 0.0f) * decay;
            if (TYPE == kSeqF16) most = fmaxf(most, fabsf(x[i + e]));
          }
        }
        if constexpr (TYPE == kSeqF16) {  // the largest of a row's to about 2^14, so that none overflows and small ones count
          most = across32(most, MaxOp());
          const int e = max(__builtin_amdgcn_frexp_expf(most) - 14, -100);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = __builtin_ldexpf(x[i], -e);
          if (half == 0) its.unit[s0 / 32][t0 + col] = __builtin_ldexpf(1.0f, e);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<u4v *>(P + (t0 + col) * PP + s0 + 16 * i + 8 * half) =
              u4v{pack2<TYPE>(x[8 * i], x[8 * i + 1]), pack2<TYPE>(x[8 * i + 2], x[8 * i + 3]), pack2<TYPE>(x[8 * i + 4], x[8 * i + 5]),
                  pack2<TYPE>(x[8 * i + 6], x[8 * i + 7])};
      }
    }
    if (wave == 3 && more) decays(c + 1, decay_then);
    if (on) {
      if constexpr (TYPE == kSeqF16) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int x = 0; x < 16; ++x) top = fmaxf(top, fabsf(s[d][x]));
        top = across32(top, MaxOp());
      }
      if constexpr (OUT) {
        if constexpr (TYPE == kSeqF16) {
          const int e = min(14 - __builtin_amdgcn_frexp_expf(top), 100);
          fit = __builtin_ldexpf(1.0f, e);
          back = __builtin_ldexpf(1.0f, -e - held);
        }
        from_state();
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) vf[j] = values_of(SIDE && !OUT ? V1 : V0, j);
    }
    if constexpr (OUT) {
      // An infinity or NaN among the values would reach earlier rows of the chunk as 0 times it: left out of the product
      // it makes NaN of its channel from its row on, and of the state's.
      if (on) {
        typedef unsigned short us2 __attribute__((ext_vector_type(2)));
        us2 most = {0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) most = __builtin_elementwise_max(most, __builtin_bit_cast(us2, vf[j][x] & 0x7fff7fffu));
        if (__any(T::odd_bits(__builtin_bit_cast(unsigned, most)) != 0)) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const unsigned bad = T::odd_bits(vf[j][x]), at = 16 * j + 8 * half + 2 * x;
              if (bad) odd_row = min(odd_row, bad & 0x8000u ? at : at + 1);
              vf[j][x] &= ~((bad >> 15) * 0xffffu);
            }
          odd_row = min(odd_row, (unsigned)__shfl_xor((int)odd_row, 32));
          odd = true;
        }
      }
      lds_barrier();
      if (on) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int z = 0; z <= t; ++z) {  // halves of the keys
            // fp16: by itself, since neither half's units need hold the state's part or the other half's
            f16v sum = {};
#pragma unroll
            for (int j = 2 * z; j < 2 * z + 2; ++j) {
              const u4v x = *reinterpret_cast<const u4v *>(P + (32 * t + col) * PP + 16 * j + 8 * half);
              if constexpr (TYPE == kSeqF16) sum = T::mma32(vf[j], x, sum);
              else acc[t] = T::mma32(vf[j], x, acc[t]);
            }
            if constexpr (TYPE == kSeqF16) {
              const float unit = its.unit[z][32 * t + col];
#pragma unroll
              for (int x = 0; x < 16; ++x) acc[t][x] = fmaf(sum[x], unit, acc[t][x]);
            }
          }
      }
      if (odd) {
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const unsigned from = (unsigned)__shfl((int)odd_row, turned(result_row(x, half)));
#pragma unroll
          for (int t = 0; t < 2; ++t) acc[t][x] = 32u * t + col >= from ? __builtin_nanf("") : acc[t][x];
        }
      }
      if (more) {
        copy_q(c + 1);
        copy_v(c + 1, even);
      }
      if (on) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) y[2 * t + i][x] = pack2<TYPE>(acc[t][8 * i + 2 * x] * p.scale, acc[t][8 * i + 2 * x + 1] * p.scale);
      }
    }
    // the state: values with their decays to the chunk's end in parts of 16 bits, which together have fp32's precision
    if (on) {
      float a = its.whole[SIDE], hold = 1.0f;
      int by = 0;  // fp16: the state is multiplied by a 2^by
      if constexpr (TYPE == kSeqF16) {
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const f2v y = unpack2<TYPE>(vf[j][x]), z = *reinterpret_cast<const f2v *>(&its.left[SIDE][16 * j + 8 * half + 2 * x]);
            most = fmaxf(most, fmaxf(fabsf(y[0] * z[0]), fabsf(y[1] * z[1])));
          }
        most = fminf(across32(most, MaxOp()), 3.0e38f);
        asm volatile("" ::: "memory");  // the decays are read again below: kept, they cost registers that spill
        // Values with their decays to about 2^14, whether decays are below 1 or above, as far as what the column held before
        // stays below 2^125: an infinity where it need not be would be a NaN in the second part, or a state that is lost.
        const int grows = __builtin_amdgcn_frexp_expf(a);
        int next = min(most > 0.0f ? 14 - __builtin_amdgcn_frexp_expf(most) : 40, 40);
        if (top > 0.0f) next = min(next, 125 + held - __builtin_amdgcn_frexp_expf(top) - grows);
        by = grows + next - held;
        a = __builtin_amdgcn_frexp_mantf(a);
        held = next;
        hold = __builtin_ldexpf(1.0f, next);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int x = 0; x < 16; ++x) s[d][x] = TYPE == kSeqF16 ? __builtin_ldexpf(s[d][x] * a, by) : s[d][x] * a;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u4v part[PARTS];
        const f4v l0 = *reinterpret_cast<const f4v *>(&its.left[SIDE][16 * j + 8 * half]), l1 = *reinterpret_cast<const f4v *>(&its.left[SIDE][16 * j + 8 * half + 4]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          unsigned z[PARTS];
          f2v left = x < 2 ? f2v{l0[2 * x], l0[2 * x + 1]} : f2v{l1[2 * x - 4], l1[2 * x - 3]};
          // finite, since it may meet a value of zero
          if (TYPE == kSeqF16) left = f2v{fminf(left[0] * hold, 3.0e38f), fminf(left[1] * hold, 3.0e38f)};
          split<TYPE>(unpack2<TYPE>(vf[j][x]), left, z);
#pragma unroll
          for (int i = 0; i < PARTS; ++i) part[i][x] = z[i];
        }
        u4v kf[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) kf[d] = keys_of(K, j, d);
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
#pragma unroll
          for (int d = 0; d < ND; ++d) s[d] = T::mma32(kf[d], part[i], s[d]);
      }
      if (OUT && odd && odd_row < (unsigned)kChunk)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int x = 0; x < 16; ++x) s[d][x] = __builtin_nanf("");
    }
    wait_for_copies();  // the next chunk's rows; outputs go behind them and are waited for a chunk later
    if (OUT && on) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int row = c * kChunk + 32 * t + col;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (row < n && ch0 + 16 * i + 8 * half < p.dim) *reinterpret_cast<u4v *>(o + (long)row * p.o_token + 16 * i + 8 * half) = y[2 * t + i];
      }
    }
    lds_barrier();
  };
  for (int c = 0; c < chunks; c += 2) {
    chunk(c, even);
    if (c + 1 < chunks) chunk(c + 1, odd_one);
  }
  if (!OUT && wave == 3 && lane == 0 && block == 0) {
    // the decay of thousands of tokens need not be one of fp32's numbers, where what it makes of a state is: 2^e m
    const double e = fmin(fmax(floor(total), -300.0), 250.0);
    reinterpret_cast<f2v *>(p.decay)[(long)u * p.heads + h] = f2v{(float)exp2(total - e), (float)e};
  }
  if (!on) return;
  if constexpr (OUT) {
    if (seg.s == seg.n - 1 && (unsigned)out < (unsigned)p.slots) state_io(p.state + ((long)out * p.heads + h) * one, store);
  } else {
    state_io(first + (long)p.heads * one, store);
  }
}

// The first states of a sequence's segments from those that the segments add: four elements a thread.
__global__ void __launch_bounds__(256) linear_join_kernel(const LinearParams p)
{
  const long one = (long)p.key_dim * p.dim;
  const int h = blockIdx.x % p.heads, b = blockIdx.x / p.heads;
  const int c0 = min(max(p.cu[b], 0), p.tokens), rows = min(max(p.cu[b + 1], c0), p.tokens) - c0;
  const int n = (rows + p.seg - 1) / p.seg;
  const long u = (long)(c0 / p.seg) + b, i = 4L * (blockIdx.y * 256 + threadIdx.x);
  if (n < 3 || i >= one) return;
  float * at = p.ws + (u * p.heads + h) * one + i;
  f4v x = *reinterpret_cast<const f4v *>(at + p.heads * one);
#pragma unroll 4
  for (int s = 2; s < n; ++s) {
    // in two factors, of which each is finite: a state of zeros stays one
    const f2v decay = reinterpret_cast<const f2v *>(p.decay)[(u + s - 1) * p.heads + h];
    const int e = (int)decay[1], e0 = e / 2;
    const float a0 = __builtin_ldexpf(decay[0], e0), a1 = __builtin_ldexpf(1.0f, e - e0);
    f4v y = *reinterpret_cast<const f4v *>(at + s * p.heads * one);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = fmaf(a1, a0 * x[j], y[j]);
    *reinterpret_cast<f4v *>(at + s * p.heads * one) = x;
  }
}

namespace {

template <int TYPE, int DK> void launch_linear_chunks(const LinearParams & p, hipStream_t s)
{
  const int blocks = (p.dim + 127) / 128;
  const int units = p.tokens / p.seg + p.batch;
  const dim3 grid((unsigned)linear_wgs(p)), blk(256);
  if (p.ws) {
    hipLaunchKernelGGL((linear_chunk_kernel<TYPE, DK, false>), grid, blk, 0, s, p, units, blocks);
    const int parts = (p.key_dim * p.dim + 1023) / 1024;
    hipLaunchKernelGGL(linear_join_kernel, dim3((unsigned)(p.batch * p.heads), (unsigned)parts), blk, 0, s, p);
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
  const dim3 grid((unsigned)linear_wgs(p)), blk(kStepThreads);
  if (p.key_dim <= 64) hipLaunchKernelGGL((linear_step_kernel<TYPE, 32, 2>), grid, blk, 0, s, p, blocks);
  else if (p.key_dim <= 128) hipLaunchKernelGGL((linear_step_kernel<TYPE, 32, 4>), grid, blk, 0, s, p, blocks);
  else hipLaunchKernelGGL((linear_step_kernel<TYPE, 32, 8>), grid, blk, 0, s, p, blocks);
}

}  // namespace

size_t linear_split(LinearParams & p, int max_new)
{
  // Token by token a state is read and written once as well, and a few tokens of it cost less than a chunk's start, whose
  // products take 64 rows whatever there is.  The sides meet between 3 and 10 tokens, by sizes of states (96 sequences, us, token by token
  // and in a chunk: 32 heads of 128 x 128 4 tokens 94 and 97, 6 111 and 99, 8 132 and 99, 16 207 and 104; 48 heads of
  // 128 x 64 6 85 and 109, 10 114 and 109; 8 heads of 256 x 64 6 43 and 49, 8 52 and 49; 16 heads of 256 x 256 3 303 and 240;
  // one sequence of 32 heads of 128 x 128 8 10.4 and 11.2, 16 16.5 and 11.2).
  p.seg = 0;
  if (max_new <= 6) return 0;
  // Rounds of work-groups, two a CU (one above 128 key channels), times the tokens of each, for sequences of the same length
  // or the longest one.
  const long cap = p.key_dim <= 128 ? 512 : 256, wgs = (long)p.heads * ((p.dim + 127) / 128), mean = std::max(1, p.tokens / p.batch);
  auto rounds = [&](long units) { return (units * wgs + cap - 1) / cap; };
  long best = 0, cost = std::max(rounds(p.batch) * mean, (long)max_new);
  // a launch holds fewer than 2^24 work-groups
  const long least = std::max<long>(256, ((long)p.tokens * wgs >> 22) / kChunk * kChunk + kChunk);
  for (long seg = least; seg < max_new; seg += std::max<long>(kChunk, seg / 16 / kChunk * kChunk)) {
    const long c = rounds(p.batch * ((mean + seg - 1) / seg)) * seg;
    if (c < cost || (best > 0 && c == cost)) {
      best = seg;
      cost = c;
    }
    if (seg > cost) break;
  }
  // Segments cost a second pass over keys and values, and their first states: 0.7 of the outputs' time.  A second work-group on a
  // CU takes 0.72 of another's time where it shares one, so whole sequences that give each CU one are left whole (32
  // heads of 128 x 128, us, whole and in segments: 8 of 4096 tokens 325 and 385, 8 of 2048 167 and 207, 4 of 4096 283 and 212, one
  // of 4096 281 and 82, of 512 42 and 41, of 300 28 and 40; 16 ragged ones of 16 heads of 64 x 96, 301 to 4099 tokens, 208 and 189).
  auto busy = [&](long units) { return cap == 512 ? std::max(1.0, 0.86 * (double)(units * wgs) / 256.0) : (double)rounds(units); };
  if (best && 1.7 * busy(p.batch * ((mean + best - 1) / best)) * (double)best >= std::max(busy(p.batch) * (double)mean, (double)max_new)) best = 0;
  p.seg = best ? (int)best : kMaxSeg;
  return best ? ((size_t)p.tokens / p.seg + p.batch) * p.heads * ((size_t)p.key_dim * p.dim + 2) * sizeof(float) : 0;
}

long linear_wgs(const LinearParams & p)
{
  if (p.seg == 0) return (long)p.batch * p.heads * ((p.dim + 31) / 32);
  const long keys = ((long)p.tokens / p.seg + p.batch) * (p.heads / p.group);
  return (keys + kXcds - 1) / kXcds * kXcds * p.group * ((p.dim + 127) / 128);
}

void launch_linear_attention(const LinearParams & p, hipStream_t s)
{
  if (p.type == kSeqF16) launch_linear_type<kSeqF16>(p, s);
  else launch_linear_type<kSeqBF16>(p, s);
}

}  // namespace ivh
