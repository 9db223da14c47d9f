// Device-side pieces of the sequence operators: the two 16-bit types behind one interface, MFMA
// shapes, cross-lane exchanges and rotation angles.
#pragma once

#include "seq_ops.hpp"

namespace ivh {

typedef float f2v __attribute__((ext_vector_type(2)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef unsigned u2v __attribute__((ext_vector_type(2)));
typedef unsigned u4v __attribute__((ext_vector_type(4)));

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLowest = -3.0e38f;  // running maximum before any key: finite, so that no inf - inf arises

template <int TYPE> struct St;
template <> struct St<kSeqF16> {
  typedef _Float16 e;
  typedef _Float16 e2 __attribute__((ext_vector_type(2)));
  typedef _Float16 e8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f4v mma16(u4v a, u4v b, f4v c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(e8, a), __builtin_bit_cast(e8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f16v mma32(u4v a, u4v b, f16v c)
  {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(e8, a), __builtin_bit_cast(e8, b), c, 0, 0, 0);
  }
  // four e4m3 codes as two pairs: exact, e4m3 is a subset of both types
  static __device__ __forceinline__ unsigned fp8_lo(unsigned x)
  {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false));
  }
  static __device__ __forceinline__ unsigned fp8_hi(unsigned x)
  {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true));
  }
  static __device__ __forceinline__ float add2(unsigned x, float c)  // c + both halves
  {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(e2, x), __builtin_bit_cast(e2, 0x3c003c00u), c, false);
  }
  // which halves of x are infinite or NaN: their top bits
  static __device__ __forceinline__ unsigned odd_bits(unsigned x) { return ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }
};
template <> struct St<kSeqBF16> {
  typedef __bf16 e;
  typedef __bf16 e2 __attribute__((ext_vector_type(2)));
  typedef __bf16 e8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f4v mma16(u4v a, u4v b, f4v c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(e8, a), __builtin_bit_cast(e8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f16v mma32(u4v a, u4v b, f16v c)
  {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(e8, a), __builtin_bit_cast(e8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned fp8_lo(unsigned x)
  {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false));
  }
  static __device__ __forceinline__ unsigned fp8_hi(unsigned x)
  {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true));
  }
  static __device__ __forceinline__ float add2(unsigned x, float c)
  {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(e2, x), __builtin_bit_cast(e2, 0x3f803f80u), c, false);
  }
  static __device__ __forceinline__ unsigned odd_bits(unsigned x) { return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
};

// two fp32 values rounded to a pair of 16-bit ones (nearest, ties to even)
template <int TYPE> __device__ __forceinline__ unsigned pack2(float a, float b)
{
  typename St<TYPE>::e2 v;
  v[0] = (typename St<TYPE>::e)a;
  v[1] = (typename St<TYPE>::e)b;
  return __builtin_bit_cast(unsigned, v);
}

template <int TYPE> __device__ __forceinline__ f2v unpack2(unsigned x)
{
  const typename St<TYPE>::e2 v = __builtin_bit_cast(typename St<TYPE>::e2, x);
  return f2v{(float)v[0], (float)v[1]};
}

// the largest of three, NaN if one is: one instruction
__device__ __forceinline__ float top_of(float a, float b, float c)
{
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// x of the lane 16 and 32 away, combined: swaps of lane rows on the vector unit
template <class Op> __device__ __forceinline__ float across16(float x, Op op)
{
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return op(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
template <class Op> __device__ __forceinline__ float across32(float x, Op op)
{
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return op(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
struct MaxOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct SumOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// Axis of frequency f.
__device__ __forceinline__ int rot_axis(const RotParams & r, int f)
{
  if (r.axes == 1) return 0;
  if (r.dealt) {  // frequency f is axis f mod axes' while that axis has some left; the first axis takes the rest
    const int a = f % r.axes;
    const int n = a == 1 ? r.sec[1] : a == 2 ? r.sec[2] : r.sec[3];
    return a != 0 && f / r.axes < n ? a : 0;
  }
  const int e0 = r.sec[0], e1 = e0 + r.sec[1], e2 = e1 + r.sec[2];
  return (f >= e0) + (f >= e1) + (f >= e2);
}

// A frequency in turns (radians / 2 pi) as the sum of two fp32 values.
__device__ __forceinline__ f2v rot_turns(float freq)
{
  const double t = (double)freq * 0.15915494309189535;
  const float h = (float)t;
  return f2v{h, (float)(t - (double)h)};
}

// cos and sin of pos * freq; turns: rot_turns(freq).  At position 10^6 an angle of 32 bits would be off by
// 0.03 radians: the product is formed in two parts, off by 2^-48 of it, of which the whole turns and then
// the quadrant are dropped before the parts are added; positions from 2^22 on take 64 bits.  Taylor's polynomials up
// to a quarter of pi are off by 2^-28 before rounding.
__device__ __forceinline__ f2v rot_cossin(int pos, float freq, f2v turns)
{
#pragma clang fp contract(off)  // the product and its remainder are two values
  const float x = (float)pos, a = x * turns[0];
  float e = fmaf(x, turns[1], fmaf(x, turns[0], -a)), t = a - rintf(a);
  if (pos >= 1 << 22 || pos <= -(1 << 22)) {
    const double d = (double)pos * (double)freq * 0.15915494309189535, f = d - rint(d);
    t = (float)f;
    e = (float)(f - (double)t);
  }
  const float q = rintf(4.0f * (t + e)), r = 2.0f * (fmaf(q, -0.25f, t) + e), r2 = r * r;  // half turns, in [-1/4, 1/4]
  constexpr double pi = 3.14159265358979323846, pi2 = pi * pi;
  constexpr float s1 = (float)pi, s1l = (float)(pi - (double)(float)pi), s3 = (float)(-pi * pi2 / 6), s5 = (float)(pi * pi2 * pi2 / 120),
                  s7 = (float)(-pi * pi2 * pi2 * pi2 / 5040), s9 = (float)(pi * pi2 * pi2 * pi2 * pi2 / 362880);
  constexpr float c2 = (float)(-pi2 / 2), c4 = (float)(pi2 * pi2 / 24), c6 = (float)(-pi2 * pi2 * pi2 / 720),
                  c8 = (float)(pi2 * pi2 * pi2 * pi2 / 40320), c10 = (float)(-pi2 * pi2 * pi2 * pi2 * pi2 / 3628800);
  const float sp = fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, s9, s7), s5), s3), s1l);
  const float s = fmaf(r, s1, r * sp);
  const float c = fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, c10, c8), c6), c4), c2), 1.0f);
  const unsigned n = (unsigned)(int)q;
  const unsigned us = __builtin_bit_cast(unsigned, n & 1 ? c : s), uc = __builtin_bit_cast(unsigned, n & 1 ? s : c);
  return f2v{__builtin_bit_cast(float, uc ^ ((n + 1) << 30 & 0x80000000u)), __builtin_bit_cast(float, us ^ (n << 30 & 0x80000000u))};
}

// The sequence whose start start(b) is the largest not above w, by a 64-wide search of one wave:
// start must not decrease over [0, n).  Any values keep the answer within [0, n).
template <class Fn> __device__ __forceinline__ int find_seq(int n, long w, Fn && start)
{
  const int lane = threadIdx.x & 63;
  int b0 = 0;
  while (n > 1) {
    const int stride = (n + 63) / 64;
    const int off = lane * stride;
    const bool below = off < n && start(b0 + off) <= w;
    const unsigned long long m = __ballot(below);
    const int i = m ? 63 - __clzll(m) : 0;
    const int left = n - i * stride;
    b0 += i * stride;
    n = left < stride ? left : stride;
  }
  return b0;
}

}  // namespace ivh
