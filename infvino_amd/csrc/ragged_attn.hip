// Attention over ragged contiguous sequences, causal or not, with an optional sliding window and
// first tokens that stay visible, on gfx950 MFMA.
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j] over the keys j that i sees; places count from
//   the end: the last query stands at the last key
//
// Long prompts are bound by the matrix cores: 4 dim operations for a pair of tokens, against
// 4 dim bytes of each key for 128 rows.  A work-group of four waves owns 128 rows of one head, a
// wave 32 of them, and walks the keys 64 at a time with a running maximum and sum in fp32:
//   * keys and values are copied by DMA straight into LDS while earlier ones are worked on: keys in
//     a ring of four 32-key blocks, since a block's scores are formed while the block before it is
//     weighed, values in two stages of 64;
//   * S^T = K Q^T on 32x32x16 MFMA: a lane holds 16 scores of one query of a 32-key block, keys
//     8 (v / 4) + 4 (lane / 32) + v % 4.  As an operand of the second product its scores 8 s ..
//     8 s + 7 are 8 of the 16 keys of slice s, no lane exchange between the products;
//   * O^T = V^T P^T, with V^T read from the row-major stage by the transposing LDS load, 4 keys
//     of one channel a lane, in the order of the scores.
//   * a block is a fixed order of slots, each a matrix instruction of the next block's scores or of
//     this one's second product, the exponentials beside the former; fragments are read from LDS
//     four slots before their use, so that the matrix cores do not wait for them;
//   * the running maximum moves only when a score exceeds it by 8 (in powers of two): until then
//     the accumulators need no rescaling.  fp16 weights hold 2^7 more, so that thousands of small ones
//     are not lost: those below 2^-21 of the largest are off by 2^-32 of it at most;
//   * a second, careful pass over the keys runs for rows whose result is not finite: there 0 times an
//     infinity or NaN of a key that the row does not see may be the reason.
// LDS rows are not padded (DMA writes 64 x 16 bytes in a row); 16-byte pieces are permuted within
// a row by the source address, so that the lanes that are served together lie in distinct banks.
// Probabilities are rounded to 16 bits for the second product, and their sum is that of the rounded
// ones, so a row's weights add up to 1.
//
// Measured (a bf16 product of 8192^3 reaches 1.23 PFLOP/s here): a prompt of 16384 tokens, 16 heads
// of 128 channels on 4, causal: 1000 to 1080 us by card, 1.10 to 1.02 PFLOP/s.  The matrix cores are busy half the cycles and
// the vector unit most of the others: work of one wave hides little of another's, with or without
// copies, exponentials or LDS reads (each taken out alone changes 3 to 10 %), and zeros for data run
// a fifth faster, which is power.  Five prompts of up to 6007 in a window of 1024: 186 to 194 us, 0.73 to
// 0.70 PFLOP/s, the same and the last of 4.6 rounds of work-groups.  64 x 16 images of up to 400 tokens, 72
// channels: 100 us, 0.35 PFLOP/s (0.43 with the products on 80 and 96 channels that it runs), 5 to 7
// steps a work-group behind 3 us of its start.  Operations are those of the pairs that are seen.
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

// 64 x 16 bytes straight into LDS: lane i's from base + its offset, zeros from `bytes` on, to lds + 16 i
__device__ __forceinline__ void copy_to_lds(const void * base, unsigned bytes, unsigned off, void * lds)
{
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, kBufDword3);
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

// LDS byte offsets of a lane's fragment pieces: of channels 16 i + 8 (lane / 32) of a key row, and
// of channel block j of a value row.  The permuted bits lie below a row's, so pieces differ by an
// exclusive or of those and a constant.
template <int DP> __device__ __forceinline__ unsigned key_at(unsigned base, int i)
{
  constexpr int BITS = DP % 128 == 0 ? 4 : DP % 64 == 0 ? 3 : 2;
  return (base ^ (32u * (i & ((1 << (BITS - 1)) - 1)))) + (unsigned)(2 * i >> BITS) * (16u << BITS);
}
template <int DP> __device__ __forceinline__ unsigned value_at(unsigned base, int j)
{
  constexpr int BITS = DP % 128 == 0 ? 2 : DP % 64 == 0 ? 1 : 0;
  return (base ^ (64u * (j & ((1 << BITS) - 1)))) + (unsigned)(j >> BITS) * (64u << BITS);
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
  // whether rows imin..imax see all of keys j0..j1
  __device__ __forceinline__ bool all(int imin, int imax, int j0, int j1) const
  {
    return j1 <= (causal ? min(imin, nk - 1) : nk - 1) && ((j0 >= lo(imax) && j1 <= hi(imin)) || j1 < sinks);
  }
};

}  // namespace

// NS: 16-channel slices of the head size, DP: that rounded up to a build's rows.
template <int TYPE, int DP, int NS>
__global__ void __launch_bounds__(256, DP <= 96 ? 3 : DP <= 128 ? 2 : 1) ragged_attn_kernel(const RaggedParams p, int slots, int side)
{
  using T = St<TYPE>;
  typedef typename T::e E;
  constexpr int NB = DP / 32;          // 32-channel blocks of the second
  constexpr int PR = DP / 8;           // 16-byte pieces of a row
  constexpr int VI = kKeys * PR / 256; // copies of a wave: values of a step,
  constexpr int KC = 32 * PR / 64, KI = (KC + 3) / 4;  // keys of a block (KC in all)
  constexpr int STAGE = kKeys * DP, BLOCK = 32 * DP;
  constexpr int UP = TYPE == kSeqF16 ? 7 : 0;  // weights of 2^-21 of the largest are normal fp16 numbers, the largest is below 2^15
  // keys: a ring of four 32-key blocks; values: two stages of 64.  Arrays of their own, so that the
  // compiler sees that a copy into one does not touch the others and leaves it in flight.
  __shared__ __attribute__((aligned(16))) unsigned char K0[BLOCK * 2], K1[BLOCK * 2], K2[BLOCK * 2], K3[BLOCK * 2];
  __shared__ __attribute__((aligned(16))) unsigned char V0[STAGE * 2], V1[STAGE * 2];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hi = lane >> 5;
  // The work-groups of a unit (sequence and key head) run on one XCD, whose L2 they share keys and
  // values in: a row block of each of its heads, then the next block of each, since those want the
  // same keys at the same time (16384 tokens, 32 heads on 8, window 4096: 934 us, 968 head by head; 8 of 4096
  // without a window 1130, 1162).  Units go round the XCDs where that is even, so that each gets its
  // share of long and short sequences; few units are cut into `side` heads for each XCD, or else
  // into equal runs of work-groups, head by head (block by block the first run would be the long ones).
  const int unit_wgs = p.group * slots, units = p.batch * (p.heads / p.group);
  int w = blockIdx.x, unit, slot, g;
  if (side < 0) {
    unit = w / kXcds / unit_wgs * kXcds + w % kXcds;
    w = w / kXcds % unit_wgs;
    if (unit >= units) return;
    slot = w / p.group;
    g = w - slot * p.group;
  } else if (side > 0) {
    slot = w / kXcds / side;
    g = w % kXcds * side + w / kXcds % side;
    unit = g / p.group;
    g -= unit * p.group;
  } else {
    w = xcd_tile(w, gridDim.x);
    unit = w / unit_wgs;
    w -= unit * unit_wgs;
    g = w / slots;
    slot = w - g * slots;
  }
  const int kv_heads = p.heads / p.group, b = unit / kv_heads, kvh = unit - b * kv_heads, head = kvh * p.group + g;

  const int q0 = min(max(p.cu_q[b], 0), p.tokens_q), q1 = min(max(p.cu_q[b + 1], q0), p.tokens_q);
  const int k0 = min(max(p.cu_k[b], 0), p.tokens_k), k1 = min(max(p.cu_k[b + 1], k0), p.tokens_k);
  const int nq = q1 - q0, nk = k1 - k0;
  const RaggedMask see = {nk, p.causal, p.window, p.window ? p.sinks : 0};
  const E * kp = static_cast<const E *>(p.k) + (long)k0 * p.k_token + (long)kvh * p.k_head;
  const E * vp = static_cast<const E *>(p.v) + (long)k0 * p.v_token + (long)kvh * p.v_head;

  // what this lane copies: position pos of row `row` of the stage holds a piece of the key's row
  unsigned koff[KI], voff[VI];
#pragma unroll
  for (int i = 0; i < KI; ++i) {
    const int s = 64 * (wave + 4 * i) + lane, row = s / PR, c = key_piece<DP>(row, s - row * PR);
    koff[i] = c * 8 < p.dim ? (unsigned)(row * (int)p.k_token + c * 8) * 2u : kBufOOB;
  }
#pragma unroll
  for (int i = 0; i < VI; ++i) {
    const int s = 64 * (wave + 4 * i) + lane, row = s / PR, c = value_piece<DP>(row, s - row * PR);
    voff[i] = c * 8 < p.dim ? (unsigned)(row * (int)p.v_token + c * 8) * 2u : kBufOOB;
  }
  // a negative scale turns the queries' signs, so that the largest score has the largest exponent
  const float scale = fmaxf(fabsf(p.scale_log2), 1.2e-38f);  // not 0: masked scores stay -inf
  const unsigned flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;

  const unsigned kaddr = (unsigned)(col * DP + key_piece<DP>(col, hi) * 8) * 2u;
  const int tr = (lane & 15) >> 2;
  const unsigned vaddr =
      (unsigned)((4 * hi + tr) * DP + value_piece<DP>(tr, 2 * (lane >> 4 & 1) + ((lane & 3) >> 1)) * 8 + (lane & 1) * 4) * 2u;

  const int nqb = (nq + kRows - 1) / kRows;
  for (int t = slot; t < nqb; t += slots) {
    const int qb = nqb - 1 - t;  // the longest first
    const int shift = nk - nq;
    const int imin = qb * kRows + shift, imax = min(nq - 1, qb * kRows + kRows - 1) + shift;
    const int wmin = imin + 32 * wave, wmax = min(imax, wmin + 31);  // this wave's rows (none where wmax < wmin)
    const int row = qb * kRows + 32 * wave + col;
    // rows and channels that are not there read some that are, without a branch that would make each
    // load wait for the one before
    const E * q = static_cast<const E *>(p.q) + (long)(q0 + min(row, nq - 1)) * p.q_token + (long)head * p.q_head;
    u4v qf[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int ch = 16 * i + 8 * hi;
      qf[i] = *reinterpret_cast<const u4v *>(q + (ch < p.dim ? ch : 0));
    }

    // steps: `first` over the first tokens, the others from step `from` on
    const int ahead = p.window ? (int)min(max((long)imax + p.window, (long)p.sinks), (long)nk) : nk;
    const int end = p.causal ? min(nk, imax + 1) : ahead;
    const int lo = p.window ? max(0, imin - p.window + 1) : 0;
    const int from = min(lo, max(end, 0)) / kKeys;
    const int first = min((min(p.sinks, lo) + kKeys - 1) / kKeys, from);
    const int total = end > 0 ? first + (end + kKeys - 1) / kKeys - from : 0;
    auto key_of = [&](int n) { return kKeys * (n < first ? n : from + n - first); };

    constexpr std::integral_constant<int, 0> c0{};
    constexpr std::integral_constant<int, 1> c1{};
    constexpr std::integral_constant<int, 2> c2{};
    constexpr std::integral_constant<int, 3> c3{};
    // keys of block g (32 of step g / 2) into slot sl of the ring; values of step n into stage st
    auto copy_keys = [&](int g, auto sl) __attribute__((always_inline)) {
      if (g >= 2 * total) return;
      const int key = key_of(g >> 1) + 32 * (g & 1), left = min(nk - key, 32);
      const unsigned bytes = left > 0 ? (unsigned)((left - 1) * (int)p.k_token + p.dim) * 2u : 0u;  // none behind the last key
      const E * at = kp + (long)key * p.k_token;
      unsigned char * to = sl == 0 ? K0 : sl == 1 ? K1 : sl == 2 ? K2 : K3;
#pragma unroll
      for (int i = 0; i < KI; ++i)
        if (4 * i + 3 < KC || wave + 4 * i < KC) copy_to_lds(at, bytes, koff[i], to + 1024 * (wave + 4 * i));
    };
    auto copy_values = [&](int n, auto st) __attribute__((always_inline)) {
      if (n >= total) return;
      const unsigned bytes = (unsigned)((min(nk - key_of(n), kKeys) - 1) * (int)p.v_token + p.dim) * 2u;
      const E * at = vp + (long)key_of(n) * p.v_token;
#pragma unroll
      for (int i = 0; i < VI; ++i)
        copy_to_lds(at, bytes, voff[i], (st ? V1 : V0) + 1024 * (wave + 4 * i));
    };
    auto copy_step = [&](int n) __attribute__((always_inline)) {  // the whole of step n, alone
      __syncthreads();
      copy_keys(2 * n, c0);
      copy_keys(2 * n + 1, c1);
      copy_values(n, c0);
      __builtin_amdgcn_s_waitcnt(vm_wait(0));
      __syncthreads();
    };
    // what this lane's row sees, less the lane's first key of a 32-key block
    const int place = row < nq ? row + shift : -(1 << 26);  // a row that is not there: as low as one can be
    const int seen_lo = see.lo(place) - 4 * hi, seen_n = see.hi(place) - see.lo(place);
    const int seen_first = min(see.sinks, see.causal ? place + 1 : see.nk) - 4 * hi;

    f16v o[NB], s0, s1;
    float M, L;
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NB; ++j) o[j] = f16v{};
      M = kLowest;
      L = 0.0f;
    };
    // fragment of channels 16 i .. of the keys in ring slot sl; of the values of keys 16 q .. and channels
    // 32 j .. in stage st, two transposing loads of 4 keys each
    auto key_piece_of = [&](auto sl, int i) __attribute__((always_inline)) {
      return *reinterpret_cast<const u4v *>((sl == 0 ? K0 : sl == 1 ? K1 : sl == 2 ? K2 : K3) + key_at<DP>(kaddr, i));
    };
    auto value_piece_of = [&](auto st, int q, int j) __attribute__((always_inline)) {
      const unsigned char * at = (st ? V1 : V0) + value_at<DP>(vaddr, j) + 32 * q * DP;
      const u2v x = read_transposed(at), y = read_transposed(at + 16 * DP);
      return u4v{x[0], x[1], y[0], y[1]};
    };
    // S^T of the 32 keys in slot sl
    auto scores = [&](auto sl, f16v & s) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NS; ++i) s = T::mma32(key_piece_of(sl, i), qf[i], i ? s : f16v{});
    };
    // scores of keys (from key0 on) that a row does not see become -inf; the reference exponent lies UP
    // below a maximum and follows it only when that is 2^8 above: weights that are larger by that lose nothing
    // in either 16-bit type
    auto settle = [&](int key0, bool inner, f16v & s) __attribute__((always_inline)) {
      if (!inner) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int j = key0 + 8 * (v / 4) + v % 4;
          const bool ok = (seen_n >= 0 && (unsigned)j - (unsigned)seen_lo <= (unsigned)seen_n) || j < seen_first;
          s[v] = ok ? s[v] : -__builtin_inff();
        }
      }
      float a = s[0], b = s[1];
#pragma unroll
      for (int v = 2; v < 16; v += 4) {
        a = top_of(a, s[v], s[v + 1]);
        if (v + 2 < 16) b = top_of(b, s[v + 2], s[v + 3]);
      }
      const float top = across32(top_of(a, b, b), MaxOp()) * scale;
      if (__any(top > M + (8.0f + UP))) {
        const float m = fmaxf(M, top - UP), e = __builtin_amdgcn_exp2f(M - m);
        M = m;
        L *= e;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[j][v] *= e;
      }
    };
    // weights of score pairs [from, to) of 8, two 16-bit values a pair; their sum is of the rounded
    // ones, which are what the values get
    auto weights = [&](const f16v & s, u4v (&pf)[2], int from, int to) __attribute__((always_inline)) {
#pragma unroll
      for (int i = from; i < to; ++i) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * i], scale, -M));
        const float y = __builtin_amdgcn_exp2f(fmaf(s[2 * i + 1], scale, -M));
        const unsigned w = pack2<TYPE>(x, y);
        L = T::add2(w, L);
        pf[i / 4][i % 4] = w;
      }
    };
    // 32 keys, half kb of the step in stage st.  The matrix cores form the scores of the next 32 (in
    // slot nsl) while the vector unit turns these into weights, then take the values.  The order is
    // pinned slot by slot, with fragments read ahead.
    auto block = [&](auto st, auto kb, auto nsl, int key0, bool inner, f16v & s, f16v & next) __attribute__((always_inline)) {
      // slots: the next keys' products, then the values'; fragment i is read R - 1 slots before its slot
      constexpr int Q = NS, W = 2 * NB, R = 5;
      u4v pf[2], f[R];
      auto read = [&](auto i) __attribute__((always_inline)) {
        if constexpr (i < Q) f[i % R] = key_piece_of(nsl, i);
        else if constexpr (i < Q + W) f[i % R] = value_piece_of(st, 2 * kb + (i - Q) / NB, (i - Q) % NB);
      };
      static_for<0, R - 1>(read);
      settle(key0, inner, s);
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, Q>([&](auto i) __attribute__((always_inline)) {
        read(std::integral_constant<int, i + R - 1>{});
        next = T::mma32(f[i % R], qf[i], i ? next : f16v{});
        weights(s, pf, i * 8 / Q, (i + 1) * 8 / Q);
        __builtin_amdgcn_sched_barrier(0);
      });
      static_for<0, W>([&](auto i) __attribute__((always_inline)) {
        read(std::integral_constant<int, Q + i + R - 1>{});
        o[i % NB] = T::mma32(f[(Q + i) % R], pf[i / NB], o[i % NB]);
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    // Step n in value stage st, whose first 32 scores are there; x, y: ring slots of the two key blocks
    // it multiplies, behind the ones it weighs; z, w: the slots that take the two after those.
    auto step = [&](int n, auto st, auto nst, auto x, auto y, auto z, auto w) __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(vm_wait(0));
      __syncthreads();
      copy_keys(2 * n + 3, z);
      copy_keys(2 * n + 4, w);
      copy_values(n + 1, nst);
      const int key0 = key_of(n);
      const bool inner = see.all(wmin, wmax, key0, key0 + kKeys - 1);
      block(st, c0, x, key0, inner, s0, s1);
      block(st, c1, y, key0 + 32, inner, s1, s0);  // after the last step s0 is of no use (whatever the slot holds)
    };

    // a step of which this wave's rows see no key: its share of the copies
    auto idle = [&](int n) __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(vm_wait(0));
      __syncthreads();
      if (n & 1) {
        copy_keys(2 * n + 3, c1);
        copy_keys(2 * n + 4, c2);
        copy_values(n + 1, c0);
      } else {
        copy_keys(2 * n + 3, c3);
        copy_keys(2 * n + 4, c0);
        copy_values(n + 1, c1);
      }
    };

    __syncthreads();  // the last rows' stages are no longer read
    if (total > 0) {
      copy_keys(0, c0);
      copy_keys(1, c1);
      copy_keys(2, c2);
      copy_values(0, c0);
      __builtin_amdgcn_s_waitcnt(vm_wait(0));
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) qf[i] = row < nq && 16 * i + 8 * hi < p.dim ? qf[i] ^ flip : u4v{0, 0, 0, 0};
    if (wmax < wmin) {  // no rows: this wave's share of the copies, up to the same barriers as the others
      for (int n = 0; n < total; ++n) idle(n);
      if (__syncthreads_or(0))
        for (int n = 0; n < total; ++n) copy_step(n);
      continue;
    }
    clear();
    if (total > 0) {
      // the wave's last key may lie steps before the work-group's
      const int wend = p.causal ? max(0, min(total, first + (wmax + kKeys) / kKeys - from)) : total;
      scores(c0, s0);
      for (int n = 0; n < wend; n += 2) {
        step(n, c0, c1, c1, c2, c3, c0);
        if (n + 1 < wend) step(n + 1, c1, c0, c3, c0, c1, c2);
      }
      for (int n = wend; n < total; ++n) idle(n);
    }

    // An infinity or NaN among the values reaches rows that do not see it, as 0 x inf, and stays
    // in their sums.  If a result is not finite the rows are taken again, one step at a time, with such
    // values left out of the product and added to the rows that do see them.
    bool odd = false;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) odd = odd || !(fabsf(o[j][v]) < __builtin_inff());
    if (__syncthreads_or(odd)) {
      clear();
      for (int n = 0; n < total; ++n) {
        copy_step(n);
        const bool inner = see.all(wmin, wmax, key_of(n), key_of(n) + kKeys - 1);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          u4v pf[2];
          if (kb) scores(c1, s0);
          else scores(c0, s0);
          settle(key_of(n) + 32 * kb, inner, s0);
          weights(s0, pf, 0, 8);
#pragma unroll
          for (int sl = 0; sl < 2; ++sl)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
              u4v a = value_piece_of(c0, 2 * kb + sl, j);
#pragma unroll
              for (int x = 0; x < 4; ++x) a[x] &= ~((T::odd_bits(a[x]) >> 15) * 0xffffu);
              o[j] = T::mma32(a, pf[sl], o[j]);
            }
        }
        const E * Vs = reinterpret_cast<const E *>(V0);
        for (int r = 0; r < kKeys; ++r) {
          const bool mine = row < nq && see(place, key_of(n) + r);
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

    const float sum = across32(L, SumOp());
    {
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;  // a row that saw nothing is zero (NaN stays)
      E * const out = static_cast<E *>(p.o) + (long)(q0 + row) * p.o_token + (long)head * p.o_head;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int v = 0; v < 16; v += 8) {
          // a lane has channels 4 hi .. of both 8-channel groups; the two halves of the wave exchange
          // theirs, so that a lane writes all 8 of group v / 4 + hi
          u4v y;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const unsigned g0 = pack2<TYPE>(o[j][v + 2 * x] * inv, o[j][v + 2 * x + 1] * inv);
            const unsigned g1 = pack2<TYPE>(o[j][v + 4 + 2 * x] * inv, o[j][v + 5 + 2 * x] * inv);
            const auto r = __builtin_amdgcn_permlane32_swap(g0, g1, false, false);
            y[x] = r[0];
            y[2 + x] = r[1];
          }
          const int ch = 32 * j + 2 * v + 8 * hi;
          if (row < nq && ch < p.dim) *reinterpret_cast<u4v *>(out + ch) = y;
        }
    }
  }
}

namespace {

template <int TYPE, int DP, int NS> void launch_ragged(const RaggedParams & p, hipStream_t s)
{
  // max_q only sizes the grid: a work-group takes every slots-th row block of its sequence.  A
  // launch holds 2^24 work-groups of 256 lanes.
  const long heads = (long)p.batch * p.heads;
  const int slots = (int)std::min<long>((std::max(1, std::min(p.max_q, p.tokens_q)) + kRows - 1) / kRows, (1L << 24) / (heads + kXcds * p.group));
  const long units = heads / p.group;
  const bool round = units % kXcds == 0 || units >= 4 * kXcds;
  const long share = heads / kXcds;  // heads of an XCD
  const int side = round ? -1 : heads % kXcds == 0 && p.group % share == 0 ? (int)share : 0;
  const long wgs = (round ? (units + kXcds - 1) / kXcds * kXcds : units) * p.group * slots;
  hipLaunchKernelGGL((ragged_attn_kernel<TYPE, DP, NS>), dim3((unsigned)wgs), dim3(256), 0, s, p, slots, side);
}

template <int TYPE> void launch_ragged_dim(const RaggedParams & p, hipStream_t s)
{
  if (p.dim <= 32) launch_ragged<TYPE, 32, 2>(p, s);
  else if (p.dim <= 64) launch_ragged<TYPE, 64, 4>(p, s);
  else if (p.dim <= 80) launch_ragged<TYPE, 96, 5>(p, s);
  else if (p.dim <= 96) launch_ragged<TYPE, 96, 6>(p, s);
  else if (p.dim <= 128) launch_ragged<TYPE, 128, 8>(p, s);
  else if (p.dim <= 192) launch_ragged<TYPE, 192, 12>(p, s);
  else launch_ragged<TYPE, 256, 16>(p, s);
}

}  // namespace

void launch_ragged_attention(const RaggedParams & p, hipStream_t s)
{
  if (p.type == kSeqF16) launch_ragged_dim<kSeqF16>(p, s);
  else launch_ragged_dim<kSeqBF16>(p, s);
}

}  // namespace ivh
