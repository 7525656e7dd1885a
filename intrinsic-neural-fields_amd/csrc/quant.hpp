// Rows in 8-bit whole numbers with a scale each: the arithmetic that csrc/rows8.hip,
// linear8.hip and ckpt.hip share.
//
//   a_m = max_k |x_mk|    s_m = fl(a_m fl(1 / 127))    q_mk = nearest whole number to 127 x_mk / a_m
//
// q goes by the ratio itself (ties to even), not by a rounded quotient: the same numbers
// whichever kernel makes them.  A row of zeros has s = 0 and q = 0; a row with an infinity
// or a NaN has s = NaN and q = 0, so that whatever is made of it is NaN.
#pragma once

#include "common.hpp"

namespace inf {
namespace q8 {

constexpr int Q_MAX = 127;
// q rows start on 16 bytes, so that 16 of their values are one load
constexpr int64_t Q_ALIGN = 16;
// packed weight rows are zero up to a multiple of this: a product may run past a row's end
// on the other side (csrc/linear8.hip)
constexpr int64_t W_ALIGN = 128;
// bytes behind the last q row that a product may read
constexpr int64_t Q_SLACK = 128;

// |x| as an unsigned number: orders like |x|, infinities and NaNs above everything finite,
// so that a maximum keeps them (fmaxf drops a NaN)
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct RowScale {
  float s;     // the row's scale (NaN where the row is not finite)
  float a;     // its maximum, times up
  float r;     // about 127 / a; 0 where every q is 0
  float up;    // 2^64 for a row below 2^-90, whose 127 / a would overflow; 1 otherwise
};

__device__ __forceinline__ RowScale row_scale(unsigned amax_bits) {
  RowScale o;
  const float a = __uint_as_float(amax_bits);
  const bool finite = amax_bits < 0x7f800000u;
  o.s = finite ? a * (1.f / 127.f) : __uint_as_float(0x7fc00000u);
  o.up = a < 0x1p-90f ? 0x1p64f : 1.f;
  o.a = a * o.up;
  o.r = finite && amax_bits != 0 ? 127.f / o.a : 0.f;
  return o;
}

// The nearest whole number to 127 x / a.  t is off by at most 127 (2^-23 + 2^-24) < 3e-5;
// where that could matter (t within 1e-4 of a half) the ratio is compared with the half in
// 64 bits, 254 |x| against (2 n + 1) a, both exact there.
__device__ __forceinline__ int quantize(float x, const RowScale& rs) {
  const float t = rs.r == 0.f ? 0.f : (x * rs.up) * rs.r;
  const float n = rintf(t);
  int q = (int)n;
  if (fabsf(t - n) > 0.4999f) {
    const float f = floorf(fabsf(t));
    const double twice = 254.0 * (double)fabsf(x * rs.up), half = (2.0 * (double)f + 1.0) * (double)rs.a;
    const int m = (int)f + (twice > half || (twice == half && ((int)f & 1)) ? 1 : 0);
    q = t < 0.f ? -m : m;
  }
  return q;
}

// four values as the bytes of a word
__device__ __forceinline__ uint32_t quantize4(float x0, float x1, float x2, float x3, const RowScale& rs) {
  return (uint32_t)(uint8_t)quantize(x0, rs) | (uint32_t)(uint8_t)quantize(x1, rs) << 8 |
         (uint32_t)(uint8_t)quantize(x2, rs) << 16 | (uint32_t)quantize(x3, rs) << 24;
}

// relu keeps a NaN (fmaxf would make it 0); sigmoid as csrc/dense.hip
__device__ __forceinline__ float activate(float v, int act) {
  if (act == 1) return v > 0.f ? v : (v != v ? v : 0.f);
  if (act == 2) return 1.f / (1.f + expf(-v));
  return v;
}

}  // namespace q8

int launch_quantize_rows(const void* x, int dtype, int64_t rows, int k, int64_t ldx, int8_t* q, int64_t ldq,
                         float* scale, hipStream_t stream);

}  // namespace inf
