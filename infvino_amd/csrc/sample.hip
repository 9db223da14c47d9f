// The next token of each row of logits: temperature, top-k, top-p, min-p, and the inverse of what is left
// at a given random number, on gfx950.
//
// Weights w = 2^z, z = (x - max) log2 e / T, are whole multiples of 2^-44: their sums over up to 2^19 tokens fit in
// 63 bits and are the same in any order, so cuts and draws do not depend on how a row is split, and no atomic's
// order can change a token.  What lies 45 powers of two below the largest is out.  Exponentials are formed in 64 bits.
//
// Every filter keeps a leading part of the descending order (equal logits by index), so that all of them together are one
// cut, a code of a logit and how many of those that equal it are in, and nothing is sorted.  Rows of up to 8192 tokens
// are left to one work-group.  Longer ones are read three times in pieces of 4096 tokens, by as many
// work-groups as fill the chip:
//   1. the largest logit of each part;
//   2. counts and sums of weights in 256 bins of z, 8 to a power of two down to 2^-28 (rows with top-k or top-p alone);
//   3. the bins say in which of them the cut lies: sums of what is surely kept for each piece, and a list
//      of the tokens of those bins;
// and a last kernel, a work-group a row, finds the cut among the listed ones by digits of their codes, adds
// them to their pieces' sums, and reads the one piece that u falls in.  Where more than 8192 tokens fall into those
// bins, as in rows of equal logits, it reads the row itself instead.
//
// One row of 131072 fp32 logits: 42 us, four kernels of 26 in all and the gaps between them; a sort of the row in one work-group takes
// 855.  96 rows 70 us (list 27, bins 21, last 17, top 6), 320 rows of 200000 fp32 logits 269 us (106, 87, 36, 40), of which the
// bytes are 150 at three passes: the exponentials in 64 bits and the vector unit bound the others.
#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <type_traits>

#include "conv_common.hpp"
#include "seq_common.hpp"

namespace ivh {

namespace {

typedef unsigned long long u64;

constexpr int kPiece = 4096;      // tokens of a piece
constexpr int kMaxPieces = 128;   // of a row
constexpr int kList = 8192;       // listed tokens of a row, and tokens of a row that is left to one work-group
constexpr int kBins = 256;
constexpr int kThreads = 256;     // of the kernels over pieces
constexpr int kLast = 512;        // of the last kernel, two work-groups a CU,
constexpr int kLastWaves = kLast / 64;
constexpr u64 kOne = 1ull << 44;  // the largest weight
constexpr u64 kAll = 1ull << 63;  // no sum is larger
constexpr unsigned kNone = 0x007fffffu;  // code of -infinity

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

// z of a logit x (NaN where none can be formed): above -45 if it has a weight.  x may be NaN or infinite
__device__ __forceinline__ double power_of(float x, float top, double scale)
{
  return x == top ? 0.0 : ((double)x - (double)top) * scale;
}
// 2^z in units of 2^-44, z in (-45, 0]: Taylor's polynomial of e^t, |t| <= log 2 / 2, off by 2^-47 before rounding; adding
// 2^52 leaves the nearest whole number in a double's low bits
__device__ __forceinline__ u64 weight_at(double z)
{
  const double n = rint(z), t = (z - n) * 0.693147180559945309;
  double y = 1.0 / 39916800.0;
  constexpr double c[] = {1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0,
                          1.0 / 720.0, 1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
  for (int i = 0; i < 11; ++i) y = fma(y, t, c[i]);
  const double w = __builtin_amdgcn_ldexp(y, (int)n + 44) + 4503599627370496.0;
  return max(__builtin_bit_cast(u64, w) & 0xfffffffffffffull, 1ull);
}
__device__ __forceinline__ u64 weight_of(float x, float top, double scale)
{
  const double z = power_of(x, top, scale);
  return z > -45.0 ? weight_at(z) : 0;
}
// bin of a power in (-45, 0], the largest first; does not decrease as z falls
__device__ __forceinline__ int bin_of(double z)
{
  const float a = -(float)z;
  return a < 28.0f ? (int)(a * 8.0f) : min(224 + (int)((a - 28.0f) * 1.9f), kBins - 1);
}

// What a row asks for.
struct Filters {
  float t;
  int k;
  float p;
  u64 least;  // the smallest weight that min-p keeps
  bool has_k, has_p;
};
__device__ __forceinline__ Filters filters_of(const SampleParams & s, int row)
{
  Filters f;
  f.t = s.temperature ? s.temperature[row] : 1.0f;
  f.k = s.top_k ? s.top_k[row] : 0;
  f.p = s.top_p ? s.top_p[row] : 1.0f;
  const float m = s.min_p ? s.min_p[row] : 0.0f;
  f.least = m > 0.0f ? max((u64)ceil((double)fminf(m, 1.0f) * (double)kOne), 1ull) : 1;
  f.has_k = f.k > 0 && f.k < s.vocab;
  f.has_p = f.p < 1.0f;
  return f;
}
__device__ __forceinline__ double scale_of(float t) { return 1.4426950408889634 / (double)t; }
// the fewest units that reach p of a sum
__device__ __forceinline__ u64 share_of(float p, u64 sum) { return max((u64)ceil(fmax((double)p, 0.0) * (double)sum), 1ull); }

// What the kernels over pieces leave for the last one.
struct RowHead {
  unsigned listed;    // tokens in the list
  unsigned mode;
  unsigned deep;      // the sum of the top k is known from the listed tokens alone
  unsigned sure;      // codes from here on are kept, whatever is listed
  u64 before_n, before_s, need_s;  // of the surely kept; the sum that top-p asks for, unless deep
};
enum Mode : unsigned { kNoCut, kCutListed, kCutLong };

// A row's part of the workspace.
struct RowSpace {
  uint2 * list;     // [kList] codes and indexes
  u64 * bin_sum;    // [parts][kBins]
  u64 * piece;      // [pieces] sums of what is surely kept
  RowHead * head;
  uint2 * top;      // [parts] largest code and its first index
  unsigned * bin_n; // [parts][kBins]
};
__device__ __host__ __forceinline__ size_t row_bytes(int parts, int pieces)
{
  return ((size_t)kList * 8 + (size_t)parts * (12 * kBins + 8) + (size_t)pieces * 8 + sizeof(RowHead) + 255) / 256 * 256;
}
__device__ __forceinline__ RowSpace space_of(const SampleParams & s, int row)
{
  RowSpace r;
  r.list = reinterpret_cast<uint2 *>(static_cast<char *>(s.ws) + (size_t)row * row_bytes(s.parts, s.pieces));
  r.bin_sum = reinterpret_cast<u64 *>(r.list + kList);
  r.piece = r.bin_sum + s.parts * kBins;
  r.head = reinterpret_cast<RowHead *>(r.piece + s.pieces);
  r.top = reinterpret_cast<uint2 *>(r.head + 1);
  r.bin_n = reinterpret_cast<unsigned *>(r.top + s.parts);
  return r;
}

// the largest code with its first index, over a wave
__device__ __forceinline__ void wave_top(unsigned & code, unsigned & at)
{
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) {
    const unsigned c = __shfl_xor(code, d), j = __shfl_xor(at, d);
    if (c > code || (c == code && j < at)) {
      code = c;
      at = j;
    }
  }
}
__device__ __forceinline__ void row_top(const RowSpace & r, int parts, unsigned & code, unsigned & at)
{
  code = 0;
  at = 0xffffffffu;
  for (int i = threadIdx.x & 63; i < parts; i += 64) {
    const uint2 x = r.top[i];
    if (x.x > code || (x.x == code && x.y < at)) {
      code = x.x;
      at = x.y;
    }
  }
  wave_top(code, at);
}

// The smallest code whose token lies in a bin before `bin`, by a 64-wide search of one wave.
__device__ __forceinline__ unsigned code_before(int bin, unsigned top, double scale)
{
  const unsigned lane = threadIdx.x & 63;
  unsigned low = 0, width = top;  // the code is in [low, low + width]: that of the largest is in bin 0
  if (bin <= 0) return 0xffffffffu;
  while (width > 0) {
    const unsigned step = width / 64 + 1, c = low + min(step * lane, width);
    const double z = power_of(value_of(c), value_of(top), scale);
    const u64 in = __ballot(c > kNone && z > -45.0 && bin_of(z) < bin);  // codes up to that of -infinity are NaN's
    const unsigned i = in ? __builtin_ctzll(in) : 64;  // the first of them
    const unsigned from = i ? min(step * (i - 1) + 1, width) : 0;
    width = (i < 64 ? min(step * i, width) : width) - from;
    low += from;
  }
  return __builtin_amdgcn_readfirstlane(low);
}

template <class T> __device__ __forceinline__ T wave_scan(T x)  // inclusive
{
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

typedef u4v u4v_of_halves __attribute__((aligned(2)));
typedef u4v u4v_of_floats __attribute__((aligned(4)));
template <class E> __device__ __forceinline__ u4v load_any(const E * x)
{
  if constexpr (sizeof(E) == 2) return *reinterpret_cast<const u4v_of_halves *>(x);
  else return *reinterpret_cast<const u4v_of_floats *>(x);
}

// The 16 tokens of a piece that a thread has, in runs of 16 bytes at any alignment, 256 threads side by side; -infinity
// behind the row's end.
template <int TYPE> struct Piece {
  typedef typename Logit<TYPE>::e E;
  static constexpr int RUN = 16 / sizeof(E), RUNS = 16 / RUN;
  u4v run[RUNS];
  static __device__ __forceinline__ int first(int i) { return (i * kThreads + (int)threadIdx.x) * RUN; }
  // place of token j of a thread
  static __device__ __forceinline__ int place(int j) { return first(j / RUN) + j % RUN; }
  __device__ __forceinline__ void load(const E * x, int base, int n)
  {
    constexpr unsigned NONE = TYPE == kSeqF32 ? 0xff800000u : TYPE == kSeqF16 ? 0xfc00u : 0xff80u;  // -infinity
    if (base + kPiece <= n) {
#pragma unroll
      for (int i = 0; i < RUNS; ++i) run[i] = load_any(x + base + first(i));
    } else {
#pragma unroll
      for (int i = 0; i < RUNS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = base + first(i) + j * (RUN / 4);
          if constexpr (TYPE == kSeqF32) {
            const E y = x[min(at, n - 1)];
            run[i][j] = at < n ? __builtin_bit_cast(unsigned, y) : NONE;
          } else {
            const E y = x[min(at, n - 1)], z = x[min(at + 1, n - 1)];
            run[i][j] = (at < n ? __builtin_bit_cast(unsigned short, y) : NONE) | (at + 1 < n ? (unsigned)__builtin_bit_cast(unsigned short, z) : NONE) << 16;
          }
        }
    }
  }
  template <class Fn> __device__ __forceinline__ void each(Fn && fn) const  // fn(j, logit)
  {
#pragma unroll
    for (int i = 0; i < RUNS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned y = run[i][j];
        if constexpr (TYPE == kSeqF32) {
          fn(i * RUN + j, __builtin_bit_cast(float, y));
        } else {
          const f2v z = unpack2<TYPE>(y);
          fn(i * RUN + 2 * j, z[0]);
          fn(i * RUN + 2 * j + 1, z[1]);
        }
      }
  }
};

// The pieces of a part, the next one on its way while one is worked on: fn(piece, first token), the first
// from `ahead`, which is asked for before what the work needs is known.
template <int TYPE, class Fn> __device__ __forceinline__ void each_piece(Piece<TYPE> & ahead, const typename Logit<TYPE>::e * x, int from, int to, int n, Fn && fn)
{
  for (int i = from; i < to; ++i) {
    const Piece<TYPE> now = ahead;
    if (i + 1 < to) ahead.load(x, (i + 1) * kPiece, n);
    fn(now, i);
  }
}

}  // namespace

// 1. The largest logit of each part.
template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_top_kernel(const SampleParams p)
{
  typedef typename Logit<TYPE>::e E;
  __shared__ unsigned code[4], at[4];
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const E * x = static_cast<const E *>(p.x) + (long)row * p.row;
  const RowSpace r = space_of(p, row);
  if (part == 0 && threadIdx.x == 0) r.head->listed = 0;
  float most = -__builtin_inff();
  unsigned first = 0xffffffffu;
  const int from = part * p.per, to = min(p.pieces, from + p.per);
  Piece<TYPE> ahead;
  ahead.load(x, from * kPiece, p.vocab);
  each_piece<TYPE>(ahead, x, from, to, p.vocab, [&](const Piece<TYPE> & now, int i) {
    now.each([&](int j, float y) {
      if (y > most) {  // a thread's indexes grow
        most = y;
        first = (unsigned)(i * kPiece + Piece<TYPE>::place(j));
      }
    });
  });
  unsigned top = code_of(most);
  wave_top(top, first);
  if ((threadIdx.x & 63) == 0) {
    code[threadIdx.x / 64] = top;
    at[threadIdx.x / 64] = first;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 4; ++i)
      if (code[i] > top || (code[i] == top && at[i] < first)) {
        top = code[i];
        first = at[i];
      }
    r.top[part] = uint2{top, first};
  }
}

// 2. Counts and sums of each part's bins.
template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_bins_kernel(const SampleParams p)
{
  typedef typename Logit<TYPE>::e E;
  constexpr int COPIES = 4;  // of the bins, for lanes side by side
  __shared__ u64 sum[COPIES * (kBins + 1)];
  __shared__ unsigned count[COPIES * (kBins + 1)];
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const Filters f = filters_of(p, row);
  if (!(f.has_k || f.has_p) || !(f.t > 0.0f)) return;
  const E * x = static_cast<const E *>(p.x) + (long)row * p.row;
  const RowSpace r = space_of(p, row);
  const int from = part * p.per, to = min(p.pieces, from + p.per);
  Piece<TYPE> ahead;
  ahead.load(x, from * kPiece, p.vocab);
  for (int i = threadIdx.x; i < COPIES * (kBins + 1); i += kThreads) {
    sum[i] = 0;
    count[i] = 0;
  }
  unsigned top, at;
  row_top(r, p.parts, top, at);
  const double scale = scale_of(f.t);
  const float most = value_of(top);
  const int mine = (threadIdx.x & (COPIES - 1)) * (kBins + 1);
  if (top <= kNone) return;
  __syncthreads();
  each_piece<TYPE>(ahead, x, from, to, p.vocab, [&](const Piece<TYPE> & now, int) {
    now.each([&](int, float y) {
      const double z = power_of(y, most, scale);
      if (!(z > -45.0)) return;
      const int b = mine + bin_of(z);
      atomicAdd(&count[b], 1u);
      if (f.has_p) atomicAdd(&sum[b], weight_at(z));
    });
  });
  __syncthreads();
  const int b = threadIdx.x;
  u64 s = 0;
  unsigned n = 0;
#pragma unroll
  for (int i = 0; i < COPIES; ++i) {
    s += sum[i * (kBins + 1) + b];
    n += count[i * (kBins + 1) + b];
  }
  r.bin_sum[part * kBins + b] = s;
  r.bin_n[part * kBins + b] = n;
}

// 3. Where the cut lies; each piece's sum of what is surely kept; the tokens among which the cut is.
template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_list_kernel(const SampleParams p)
{
  typedef typename Logit<TYPE>::e E;
  __shared__ u64 wave_s[4];
  __shared__ unsigned wave_n[4], lowest[4][3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
  const Filters f = filters_of(p, row);
  if (!(f.t > 0.0f)) return;
  const E * x = static_cast<const E *>(p.x) + (long)row * p.row;
  const RowSpace r = space_of(p, row);
  const int from = part * p.per, to = min(p.pieces, from + p.per);
  Piece<TYPE> ahead;
  ahead.load(x, from * kPiece, p.vocab);
  unsigned top, at;
  row_top(r, p.parts, top, at);
  if (top <= kNone) return;
  const double scale = scale_of(f.t);
  const float most = value_of(top);
  int first = kBins, end = kBins;  // bins of the cut
  bool listed = false, inside = false, none = false;
  float kept = -__builtin_inff(), maybe = 0.0f;  // logits that are surely kept, and listed, from here on; none: none surely
  if (f.has_k || f.has_p) {
    u64 own_s = 0;
    unsigned own_n = 0;
#pragma unroll 16
    for (int i = 0; i < p.parts; ++i) {
      own_s += r.bin_sum[i * kBins + tid];
      own_n += r.bin_n[i * kBins + tid];
    }
    u64 s = wave_scan(own_s);
    unsigned n = wave_scan(own_n);
    if (lane == 63) {
      wave_s[wave] = s;
      wave_n[wave] = n;
    }
    __syncthreads();
    for (int i = 0; i < wave; ++i) {
      s += wave_s[i];
      n += wave_n[i];
    }
    const u64 all_s = wave_s[0] + wave_s[1] + wave_s[2] + wave_s[3];
    const unsigned all_n = wave_n[0] + wave_n[1] + wave_n[2] + wave_n[3];
    // the first bin for which a condition holds, of those that rise with the bin
    auto first_bin = [&](bool holds, int slot) {
      const u64 m = __ballot(holds);
      if (lane == 0) lowest[wave][slot] = m ? wave * 64 + __builtin_ctzll(m) : kBins;
    };
    __shared__ u64 kept_s[2];
    __shared__ unsigned kept_n;
    const bool cut_k = f.has_k && all_n > (unsigned)f.k;
    if (cut_k) {  // sums of the top k lie between those of the bins before its last one and with it
      first_bin(n >= (unsigned)f.k, 0);
      __syncthreads();
      const int b = (int)min(min(lowest[0][0], lowest[1][0]), min(lowest[2][0], lowest[3][0]));
      if (tid == b) {
        kept_s[0] = n == (unsigned)f.k ? s : s - own_s;
        kept_s[1] = s;
        kept_n = n;
      }
      __syncthreads();
      inside = kept_n != (unsigned)f.k;  // else the bin's end is the cut
      end = b + 1;
      first = inside ? b : end;
    } else if (tid == 0) {
      kept_s[0] = kept_s[1] = all_s;
    }
    if (f.has_p) {
      __syncthreads();
      first_bin(s >= share_of(f.p, kept_s[0]), 1);
      first_bin(s >= share_of(f.p, kept_s[1]), 2);
      __syncthreads();
      const int lo = (int)min(min(lowest[0][1], lowest[1][1]), min(lowest[2][1], lowest[3][1]));
      const int hi = (int)min(min(lowest[0][2], lowest[1][2]), min(lowest[2][2], lowest[3][2]));
      first = lo;
      if (!inside) end = hi + 1;  // else the sum of the top k needs its last bin's tokens
    }
    __shared__ unsigned span_n[2];
    __shared__ u64 before_s;
    __syncthreads();
    if (tid == 0) {
      span_n[0] = 0;
      before_s = 0;
    }
    __syncthreads();
    if (tid == first - 1) {
      span_n[0] = n;
      before_s = s;
    }
    if (tid == end - 1) span_n[1] = n;
    __syncthreads();
    const unsigned many = first < end ? span_n[1] - span_n[0] : 0;
    listed = many > 0 && many <= (unsigned)kList;
    const unsigned sure = code_before(first, top, scale);
    if (part == 0 && tid == 0) {
      r.head->mode = first >= end ? kNoCut : listed ? kCutListed : kCutLong;
      r.head->deep = inside;
      r.head->sure = sure;
      r.head->before_n = span_n[0];
      r.head->before_s = before_s;
      r.head->need_s = f.has_p ? share_of(f.p, kept_s[0]) : kAll;
    }
    if (first < end && !listed) return;
    kept = first > 0 ? value_of(sure) : __builtin_inff();
    none = first == 0;
    if (listed) maybe = value_of(code_before(end, top, scale));
  }
  each_piece<TYPE>(ahead, x, from, to, p.vocab, [&](const Piece<TYPE> & now, int i) {
    u64 sum = 0;
    unsigned mask = 0;
    now.each([&](int j, float y) {
      if (y >= kept && !none) {
        const u64 w = weight_of(y, most, scale);
        sum += w >= f.least ? w : 0;
      } else if (listed && y >= maybe) {
        mask |= 1u << j;
      }
    });
    if (listed) {
      const unsigned mine = __popc(mask), upto = wave_scan(mine), all = __shfl(upto, 63);
      if (all) {
        unsigned base = 0;
        if (lane == 0) base = atomicAdd(&r.head->listed, all);
        base = __shfl(base, 0) + upto - mine;
        now.each([&](int j, float y) {
          if (!(mask >> j & 1)) return;
          if (base < (unsigned)kList) r.list[base] = uint2{code_of(y), (unsigned)(i * kPiece + Piece<TYPE>::place(j))};
          ++base;
        });
      }
    }
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) sum += __shfl_xor(sum, d);
    __syncthreads();
    if (lane == 0) wave_s[wave] = sum;
    __syncthreads();
    if (tid == 0) r.piece[i] = wave_s[0] + wave_s[1] + wave_s[2] + wave_s[3];
  });
}

namespace {

struct Cut {
  unsigned code;  // kept: codes above, and the first `ties` of this one
  unsigned ties;
  u64 sum;        // of what is kept
};

constexpr int kDigit = 11, kDigits = 1 << kDigit;  // of a code

struct LastSpace {
  u64 sum[kDigits], piece[kMaxPieces], wave_s[kLastWaves], found_s, before_s;
  unsigned count[kDigits], tie[kMaxPieces], wave_n[kLastWaves], found_n, before_n;
  int at;
};

// sum over a work-group's lower threads; all: over all
template <class T> __device__ __forceinline__ T block_before(T x, T (&wave_x)[kLastWaves], T & all)
{
  const int wave = threadIdx.x >> 6;
  const T upto = wave_scan(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) wave_x[wave] = upto;
  __syncthreads();
  T before = upto - x;
  all = 0;
#pragma unroll
  for (int i = 0; i < kLastWaves; ++i) {
    const T y = wave_x[i];
    before += i < wave ? y : 0;
    all += y;
  }
  return before;
}

// The shortest leading part of the descending order of some tokens that has need_n of them or a sum of need_s, by digits of their
// codes of up to 11 bits.  each(fn): fn(code, weight) for every token of this thread that has a weight; of them all, codes
// agree with `same` from bit `shift` on and below bit `low`.  All are kept if neither is reached.
template <class Each> __device__ __forceinline__ Cut descend(LastSpace & l, unsigned need_n, u64 need_s, unsigned same, int shift, int low, Each && each)
{
  constexpr int OWN = kDigits / kLast;
  const int tid = threadIdx.x;
  unsigned before_n = 0, prefix = shift < 32 ? same >> shift : 0;
  u64 before_s = 0;
  for (;;) {
    const int next = max(shift - kDigit, low), width = shift - next;
    const unsigned mask = (1u << width) - 1;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      l.count[tid * OWN + i] = 0;
      l.sum[tid * OWN + i] = 0;
    }
    if (tid == 0) l.at = -1;
    __syncthreads();
    each([&](unsigned c, u64 w) {
      if (shift < 32 && c >> shift != prefix) return;
      const unsigned b = mask - ((c >> next) & mask);  // the largest first
      atomicAdd(&l.count[b], 1u);
      atomicAdd(&l.sum[b], w);
    });
    __syncthreads();
    unsigned own_n = 0, all_n;
    u64 own_s = 0, all_s;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      own_n += l.count[tid * OWN + i];
      own_s += l.sum[tid * OWN + i];
    }
    unsigned n = before_n + block_before(own_n, l.wave_n, all_n);
    u64 s = before_s + block_before(own_s, l.wave_s, all_s);
    if (!(n >= need_n || s >= need_s)) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const unsigned here_n = l.count[tid * OWN + i];
        const u64 here_s = l.sum[tid * OWN + i];
        if (n + here_n >= need_n || s + here_s >= need_s) {
          l.at = tid * OWN + i;
          l.found_n = here_n;
          l.found_s = here_s;
          l.before_n = n;
          l.before_s = s;
          break;
        }
        n += here_n;
        s += here_s;
      }
    }
    __syncthreads();
    const int at = l.at;
    if (at < 0) return Cut{0, 0, before_s + all_s};
    before_n = l.before_n;
    before_s = l.before_s;
    const unsigned found_n = l.found_n;
    const u64 found_s = l.found_s;
    prefix = (shift < 32 ? prefix << width : 0) | (mask - at);
    shift = next;
    __syncthreads();
    if (shift == low) {
      const u64 w = found_s / found_n;  // of each: they are equal
      u64 ties = min((u64)found_n, (u64)(need_n - before_n));
      if (need_s > before_s) ties = min(ties, (need_s - before_s + w - 1) / w);
      return Cut{prefix << low | (same & ((1u << low) - 1)), (unsigned)ties, before_s + ties * w};
    }
  }
}

// floor(u times a sum), so that a larger sum lies beyond u of it
__device__ __forceinline__ u64 goal_of(float u, u64 sum)
{
  return u > 0.0f ? u < 1.0f ? min((u64)((double)u * (double)sum), sum - 1) : sum - 1 : 0;
}

}  // namespace

// 4. The token.  ROW: of a row of up to kList tokens; else by what the kernels above found.
template <int TYPE, bool ROW>
__global__ void __launch_bounds__(kLast, 4) sample_last_kernel(const SampleParams p)
{
  typedef typename Logit<TYPE>::e E;
  __shared__ LastSpace l;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
  const E * x = static_cast<const E *>(p.x) + (long)row * p.row;
  const int n = p.vocab;
  const Filters f = filters_of(p, row);
  const float u = p.u[row];
  RowSpace r = {};
  unsigned top = 0, at = 0xffffffffu;
  if constexpr (ROW) {
    for (int i = tid; i < n; i += kLast) {
      const unsigned c = code_of((float)x[i]);
      if (c > top) {
        top = c;
        at = i;
      }
    }
    wave_top(top, at);
    if (lane == 0) {
      l.wave_n[wave] = top;
      l.count[wave] = at;
    }
    __syncthreads();
    top = l.wave_n[lane & (kLastWaves - 1)];
    at = l.count[lane & (kLastWaves - 1)];
    wave_top(top, at);
    __syncthreads();
  } else {
    r = space_of(p, row);
    row_top(r, p.parts, top, at);
  }
  if (top <= kNone || !(f.t > 0.0f)) {
    if (tid == 0) p.token[row] = top <= kNone ? -1 : (int)at;
    return;
  }
  const double scale = scale_of(f.t);
  const float most = value_of(top);
  auto kept_weight = [&](unsigned c) {
    const u64 w = c > kNone ? weight_of(value_of(c), most, scale) : 0;
    return w >= f.least ? w : 0;
  };

  // ---- the cut
  const bool filtered = f.has_k || f.has_p;
  RowHead head = {0, filtered ? (unsigned)(ROW ? kCutLong : kCutListed) : (unsigned)kNoCut, f.has_k, 0, 0, 0, kAll};
  if (!ROW && filtered) head = *r.head;
  head.listed = min(head.listed, (unsigned)kList);
  Cut cut = {head.mode == kNoCut ? 0xffffffffu : 0u, 0, 0};  // none: codes from head.sure on
  if (head.mode == kCutListed) {
    auto each = [&](auto fn) {
      for (unsigned i = tid; i < head.listed; i += kLast) {
        const unsigned c = r.list[i].x;
        fn(c, weight_of(value_of(c), most, scale));
      }
    };
    unsigned differ = 0;  // bits in which codes differ from the largest
    for (unsigned i = tid; i < head.listed; i += kLast) differ |= r.list[i].x ^ top;
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) differ |= __shfl_xor(differ, d);
    if (lane == 0) l.wave_n[wave] = differ;
    __syncthreads();
    differ = 0;
    for (int i = 0; i < kLastWaves; ++i) differ |= l.wave_n[i];
    __syncthreads();
    const int shift = differ ? 32 - __clz(differ) : 1, low = differ ? __ffs(differ) - 1 : 0;
    if (f.has_k && head.deep) cut = descend(l, (unsigned)f.k - (unsigned)head.before_n, kAll, top, shift, low, each);
    if (f.has_p) {
      const u64 need = head.deep ? share_of(f.p, head.before_s + cut.sum) : head.need_s;
      cut = descend(l, 0xffffffffu, need - head.before_s, top, shift, low, each);
    }
  } else if (head.mode == kCutLong) {
    auto each = [&](auto fn) {
      for (int i = tid; i < n; i += kLast) {
        const float y = (float)x[i];
        const u64 w = weight_of(y, most, scale);
        if (w) fn(code_of(y), w);
      }
    };
    // without top-k the sum of all
    cut = descend(l, f.has_k ? (unsigned)f.k : 0xffffffffu, kAll, 0, 32, 0, each);
    if (f.has_p) cut = descend(l, 0xffffffffu, share_of(f.p, cut.sum), 0, 32, 0, each);
  }

  // ---- the piece that u falls in
  constexpr int HERE = ROW ? kList / kLast : kPiece / kLast;  // tokens of a thread below
  u64 goal = 0;
  unsigned ties = cut.ties;
  int base = 0;
  if constexpr (!ROW) {
    const u64 tied = kept_weight(cut.code);  // of a token that equals the cut
    if (tid < kMaxPieces) {
      l.piece[tid] = head.mode != kCutLong && tid < p.pieces ? r.piece[tid] : 0;
      l.tie[tid] = 0;
    }
    if (tid == 0) {
      l.at = 0;
      l.before_n = 0;
      l.before_s = 0;
    }
    __syncthreads();
    auto add = [&](unsigned c, unsigned i) {
      if (c == cut.code) atomicAdd(&l.tie[i / kPiece], 1u);
      else if (c > cut.code) atomicAdd(&l.piece[i / kPiece], kept_weight(c));
    };
    if (head.mode == kCutListed) {
      for (unsigned i = tid; i < head.listed; i += kLast) add(r.list[i].x, r.list[i].y);
    } else if (head.mode == kCutLong) {
      for (int i = tid; i < n; i += kLast) add(code_of((float)x[i]), (unsigned)i);
    }
    __syncthreads();
    const unsigned mine = tid < kMaxPieces ? l.tie[tid] : 0;
    unsigned all_n;
    const unsigned before_n = block_before(mine, l.wave_n, all_n), in = min(mine, ties - min(ties, before_n));
    const u64 own = tid < kMaxPieces ? l.piece[tid] + in * tied : 0;
    u64 all_s;
    const u64 before_s = block_before(own, l.wave_s, all_s);
    goal = goal_of(u, all_s);
    if (before_s <= goal && goal - before_s < own) {
      l.at = tid;
      l.before_n = before_n;
      l.before_s = before_s;
    }
    __syncthreads();
    base = l.at * kPiece;
    ties -= min(ties, l.before_n);
    goal -= l.before_s;
  }

  // ---- the token: a thread's in order of the vocabulary
  unsigned code[HERE], equal = 0;
#pragma unroll
  for (int i = 0; i < HERE; ++i) {
    const int j = base + tid * HERE + i;
    code[i] = code_of((float)x[min(j, n - 1)]);
    if (j >= n) code[i] = 0;
    equal += code[i] == cut.code;
  }
  unsigned all_n, rank = block_before(equal, l.wave_n, all_n);
  auto weight_here = [&](int i) {  // in order: ties count up
    const bool tie = code[i] == cut.code, in = code[i] > cut.code || (tie && rank < ties) || (head.mode == kNoCut && code[i] >= head.sure);
    rank += tie;
    return in ? kept_weight(code[i]) : 0;
  };
  u64 own = 0, all_s;
  const unsigned first = rank;
#pragma unroll
  for (int i = 0; i < HERE; ++i) own += weight_here(i);
  u64 before = block_before(own, l.wave_s, all_s);
  if (ROW) goal = goal_of(u, all_s);
  if (before <= goal && goal - before < own) {
    rank = first;
#pragma unroll
    for (int i = 0; i < HERE; ++i) {
      const u64 w = weight_here(i);
      if (before <= goal && goal - before < w) p.token[row] = base + tid * HERE + i;
      before += w;
    }
  }
}

namespace {

template <int TYPE> void launch_sample_type(const SampleParams & p, hipStream_t s)
{
  if (p.parts == 0) {
    hipLaunchKernelGGL((sample_last_kernel<TYPE, true>), dim3((unsigned)p.rows), dim3(kLast), 0, s, p);
    return;
  }
  const dim3 grid((unsigned)p.rows * (unsigned)p.parts), blk(kThreads);
  hipLaunchKernelGGL((sample_top_kernel<TYPE>), grid, blk, 0, s, p);
  if (p.top_k || p.top_p) hipLaunchKernelGGL((sample_bins_kernel<TYPE>), grid, blk, 0, s, p);
  hipLaunchKernelGGL((sample_list_kernel<TYPE>), grid, blk, 0, s, p);
  hipLaunchKernelGGL((sample_last_kernel<TYPE, false>), dim3((unsigned)p.rows), dim3(kLast), 0, s, p);
}

}  // namespace

size_t sample_split(SampleParams & p)
{
  p.pieces = (p.vocab + kPiece - 1) / kPiece;
  p.parts = p.per = 0;
  if (p.vocab <= kList || p.rows == 0) return 0;
  // eight work-groups a CU, of whole pieces (320 rows of 200000: 269 us, four 322, sixteen 264; 96 rows 70, 70, 72)
  const int want = std::min(p.pieces, (2048 + p.rows - 1) / p.rows);
  p.per = (p.pieces + want - 1) / want;
  p.parts = (p.pieces + p.per - 1) / p.per;
  return (size_t)p.rows * row_bytes(p.parts, p.pieces);
}

void launch_sample(const SampleParams & p, hipStream_t s)
{
  if (p.type == kSeqF16) launch_sample_type<kSeqF16>(p, s);
  else if (p.type == kSeqBF16) launch_sample_type<kSeqBF16>(p, s);
  else launch_sample_type<kSeqF32>(p, s);
}

}  // namespace ivh
