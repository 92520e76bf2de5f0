// Rows held in 8 bits: the values of a row in groups of 32, a group as one power of two s = 2^(e - 127), held as the byte e,
// and a whole number c of -127 .. 127 per value; the value is c * s. e is the smallest with max|x| / s < 127.5, kept within
// 1 .. 248, so that s and 1 / s are normal numbers; c = x / s rounded to nearest, ties to even: off by at most s / 2, at most
// 2^-7 of the group's largest value. Seven bits and a power of two are exact in fp32 and in bf16. A group with a value that
// is not finite has e = 255 and c = 0: 2^128 is read as infinity, and zero times it is NaN, with no test where rows are read.
//
// In memory: codes [rows + 1][pitch] bytes c + 128 (which saves every reader a flip of the sign), pitch = width in whole groups of
// 32, zeros (128) behind the width; scales [rows + 1][pitch / 32] bytes. The last row is of zeros: what ids outside the rows
// stand for. (One scale per group and not per
// row: activations behind a ReLU differ by orders of magnitude along a row. Scales in an array of their own: rows of codes
// then start on whole sectors, and the scales of a million rows of 128 stay in L2.)
#pragma once
#include "common.cuh"

namespace cxg {

// Pairs of fp32 values for the packed instructions, which round each half like the scalar ones.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1,%2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(Pair p) {
  float2 r;
  asm("mov.b64 {%0,%1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float sum2(Pair a) {
  const float2 t = halves(a);
  return t.x + t.y;
}

namespace rows8 {

constexpr int kGroup = 32;
constexpr uint32_t kNotFinite = 255;

inline int groups_of(int width) { return (width + kGroup - 1) / kGroup; }

// The byte of the scale, from the largest absolute value's bit pattern. A mantissa of 127.5 / 64 and more would round to 128
// and carries into the exponent instead.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top_bits) {
  if (top_bits >= 0x7f800000u) return kNotFinite;
  const int e = static_cast<int>((top_bits + 0x10000u) >> 23) - 6;
  return static_cast<uint32_t>(min(max(e, 1), 248));
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// x / s of finite groups: the product with 2^(254 - e - 127) is exact, or so small that it rounds to zero either way
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// c + 128 as the low byte of the result: adding 1.5 * 2^23 to x / s (exact in front of the addition) rounds to whole numbers,
// ties to even, and leaves them in the low bits.
__device__ __forceinline__ uint32_t code_bits(float x, float inv) { return __float_as_uint(fmaf(x, inv, 12582912.f + 128.f)); }
constexpr uint32_t kZeroCodes = 0x80808080u;

__device__ __forceinline__ uint32_t pack_codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// The codes of N values of a group, four to a word. At the top of the range of fp32, where e is kept at 248, a code is limited.
template <int N>
__device__ __forceinline__ void codes_of(uint32_t (&w)[N / 4], const float (&v)[N], uint32_t e) {
  const float inv = inverse_scale(e);
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    const float *f = v + 4 * j;
    w[j] = pack_codes(code_bits(f[0], inv), code_bits(f[1], inv), code_bits(f[2], inv), code_bits(f[3], inv));
  }
  if (e >= 248) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = code_bits(fminf(fmaxf(v[4 * j + i] * inverse_scale(248), -127.f), 127.f), 1.f);
      w[j] = e == kNotFinite ? kZeroCodes : pack_codes(c[0], c[1], c[2], c[3]);
    }
  }
}

// Code i of a word as fp32: as the low byte of 2^23 it is 2^23 + 128 + c.
template <int I>
__device__ __forceinline__ float code_value(uint32_t word) {
  return __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7440 | I)) - 8388736.f;
}
__device__ __forceinline__ void code_values(float *f, uint32_t word) {
  f[0] = code_value<0>(word), f[1] = code_value<1>(word), f[2] = code_value<2>(word), f[3] = code_value<3>(word);
}

// The scale times an edge's value may leave the range of fp32 where both are finite (scales reach 2^121): every term of the group that
// is not zero overflows then, and zeros, which an infinite factor would make NaN, have to stay zeros. The codes become -127, 0 or
// 127, and the scale (returned as its byte) is one with which the factor lies between 2^126 and 2^127. Values below kSafeValue
// cannot get there.
constexpr float kSafeValue = 128.f;
template <int N>
__device__ __forceinline__ uint32_t keep_zeros(uint32_t (&w)[N], uint32_t byte, float value) {
  const uint32_t value_exponent = (__float_as_uint(value) >> 23) & 255;
  if (byte == kNotFinite || value_exponent == 255 || (__float_as_uint(scale_of(byte) * value) & 0x7fffffffu) != 0x7f800000u) return byte;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t below = __vcmpltu4(w[i], kZeroCodes), above = __vcmpgtu4(w[i], kZeroCodes);
    w[i] = above | (below & 0x01010101u) | (kZeroCodes & ~(above | below));
  }
  return 127 + 253 - value_exponent;
}

}  // namespace rows8

// The weight gradient for a dy of few columns, one row behind the other (rows8_wgrad_narrow.cu); scales and dy 16-byte aligned. Its
// sums: [parts][columns][128] and [parts][n].
struct Rows8Narrow {
  const uint8_t *codes, *scales;
  const void *dy;
  int64_t m;
  int k, n, pitch, groups;
  uint32_t inverse;  // floor(2^32 / n)
  float *partial, *partial_db;
};
struct Rows8NarrowPlan {
  int columns, parts;  // columns 0: not for these sizes
};
Rows8NarrowPlan rows8_narrow_plan(int64_t m, int k, int n);
cudaError_t rows8_narrow_run(const Rows8Narrow &a, const Rows8NarrowPlan &plan, int dtype, cudaStream_t st);

}  // namespace cxg
