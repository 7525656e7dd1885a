// Rows in 8-bit whole numbers with a scale each: the arithmetic that csrc/rows8.hip,
// linear8.hip and ckpt.hip share.
//
//   a_m = max_k |x_mk|    s_m = fl(a_m fl(1 / 127))    q_mk = nearest whole number to 127 x_mk / a_m
//
// q goes by the ratio itself (ties to even), not by a rounded quotient: the same numbers
// whichever kernel makes them.  A row of zeros has s = 0 and q = 0; a row with an infinity
// or a NaN has s = NaN and q = 0, so that whatever is made of it is NaN.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace inf {
namespace q8 {

template <int N> using Const = std::integral_constant<int, N>;

constexpr int Q_MAX = 127;
// q rows start on 16 bytes, so that 16 of their values are one load
constexpr int64_t Q_ALIGN = 16;
// packed weight rows are zero up to a multiple of this: a product may run past a row's end
// on the other side (csrc/linear8.hip)
constexpr int64_t W_ALIGN = 128;
// bytes behind the last q row that a product may read
constexpr int64_t Q_SLACK = 128;

// A launch holds fewer than 2^32 threads.  These kernels take up to 256 of them a row and one for 16 results:
// rows beyond that go in turns of about equal size.
template <class F>
int in_turns(int64_t rows, int64_t width, const F& f) {
  const int64_t most = std::min<int64_t>((int64_t)1 << 23, std::max<int64_t>(((int64_t)1 << 35) / width, 1));
  const int64_t each = ceil_div(rows, std::max<int64_t>(ceil_div(rows, most), 1));
  for (int64_t r = 0; r < rows; r += each) {
    const int rc = f(r, std::min(each, rows - r));
    if (rc != INF_OK) return rc;
  }
  return INF_OK;
}

// |x| as an unsigned number: orders like |x|, infinities and NaNs above everything finite,
// so that a maximum keeps them (fmaxf drops a NaN)
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct RowScale {
  float s;        // the row's scale (NaN where the row is not finite)
  float a;        // its maximum
  float r;        // about 127 / a; 0 for a row of zeros, NaN where the fraction would overflow
  uint32_t keep;  // 0 where the row is not finite: its q are 0
  // bf16 rows: 127 up, a up and about 1 / (a up); up is a power of two that keeps all three in range
  float mul, top, inv;
};

__device__ __forceinline__ RowScale row_scale(unsigned amax_bits) {
  RowScale o;
  const bool finite = amax_bits < 0x7f800000u;
  o.a = __uint_as_float(amax_bits);
  o.s = finite ? o.a * (1.f / 127.f) : __uint_as_float(0x7fc00000u);
  o.r = amax_bits == 0 || !finite ? 0.f : o.a < 0x1p-100f ? __uint_as_float(0x7fc00000u) : 127.f / o.a;
  o.keep = finite ? 0xffffffffu : 0u;
  const float up = o.a < 0x1p-64f ? 0x1p64f : o.a > 0x1p64f ? 0x1p-64f : 1.f;
  o.mul = 127.f * up;
  o.top = o.a * up;
  o.inv = amax_bits == 0 ? 0.f : 1.f / o.top;
  return o;
}

// The nearest whole number to 127 x / a, a > 0, whatever t rounds to: n + 1/2 below 127 |x| / a is
// (2 n + 1) a below 254 |x|, and both products are held exactly in two fp32 (their rounding and,
// by a fused multiply-add, what it left), so that the sign of the difference is exact.  Rows below
// 2^-100 or above 2^100 are scaled by 2^64 or 2^-64 first.
__device__ __forceinline__ uint32_t quantize_exactly(float x, float a) {
#pragma clang fp contract(off)
  const float up = a < 0x1p-100f ? 0x1p64f : a > 0x1p100f ? 0x1p-64f : 1.f;
  const float m = fabsf(x) * up, top = a * up;
  const float f = floorf(m * (127.f / top));
  const float odd = __builtin_fmaf(2.f, f, 1.f);
  const float p = 254.f * m, q = odd * top;
  const float pl = __builtin_fmaf(254.f, m, -p), ql = __builtin_fmaf(odd, top, -q);
  const float over = (p - q) + (pl - ql);
  const int n = (int)f + (over > 0.f || (over == 0.f && ((int)f & 1)) ? 1 : 0);
  return (uint32_t)(x < 0.f ? -n : n) & 255u;
}

// Four values as the bytes of a word.  b = x r + 1.5 2^23, rounded once, holds the nearest whole
// number in its low byte; x r is off by at most 127 2^-23 = 1.6e-5, so where it lies within 5e-5 of
// a half (one value in 10,000; or is NaN) the ratio itself decides.  About five operations a value.
__device__ __forceinline__ uint32_t quantize4_f32(float x0, float x1, float x2, float x3, const RowScale& rs) {
  constexpr float C = 12582912.f, NEAR = 0.49995f;
  const float t0 = __builtin_fmaf(x0, rs.r, C), t1 = __builtin_fmaf(x1, rs.r, C);
  const float t2 = __builtin_fmaf(x2, rs.r, C), t3 = __builtin_fmaf(x3, rs.r, C);
  const float d0 = fabsf(__builtin_fmaf(x0, rs.r, C - t0)), d1 = fabsf(__builtin_fmaf(x1, rs.r, C - t1));
  const float d2 = fabsf(__builtin_fmaf(x2, rs.r, C - t2)), d3 = fabsf(__builtin_fmaf(x3, rs.r, C - t3));
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t1), __float_as_uint(t0), 0x0c0c0400);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(t3), __float_as_uint(t2), 0x04000c0c);
  uint32_t w = lo | hi;
  if (!(fmaxf(fmaxf(d0, d1), fmaxf(d2, d3)) <= NEAR))
    w = quantize_exactly(x0, rs.a) | quantize_exactly(x1, rs.a) << 8 | quantize_exactly(x2, rs.a) << 16 |
        quantize_exactly(x3, rs.a) << 24;
  return w & rs.keep;
}
// The same for bf16 values, whose ratios are often halves and else at least 1 / (2 255 256) from one:
// 127 x is exact, and its quotient by a, corrected by its exact remainder, is a half exactly where
// the ratio is one, and on the ratio's side of it elsewhere (a step of fp32 below 128 is 1 / 131,072).
__device__ __forceinline__ uint32_t quantize4_bf16(float x0, float x1, float x2, float x3, const RowScale& rs) {
#pragma clang fp contract(off)
  constexpr float C = 12582912.f;
  auto bits = [&](float x) {
    const float y = x * rs.mul, q = y * rs.inv;
    return __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, rs.top, y), rs.inv, q) + C);
  };
  const uint32_t lo = __builtin_amdgcn_perm(bits(x1), bits(x0), 0x0c0c0400);
  const uint32_t hi = __builtin_amdgcn_perm(bits(x3), bits(x2), 0x04000c0c);
  return (lo | hi) & rs.keep;
}

// From: the type that the values have
template <typename From = float>
__device__ __forceinline__ uint32_t quantize4(float x0, float x1, float x2, float x3, const RowScale& rs) {
  if constexpr (sizeof(From) == 2) return quantize4_bf16(x0, x1, x2, x3, rs);
  else return quantize4_f32(x0, x1, x2, x3, rs);
}
template <typename From = float>
__device__ __forceinline__ int quantize(float x, const RowScale& rs) {
  return (int)(int8_t)quantize4<From>(x, 0.f, 0.f, 0.f, rs);
}

// relu keeps a NaN (fmaxf would make it 0); sigmoid as csrc/dense.hip
__device__ __forceinline__ float activate(float v, int act) {
  if (act == 1) return v > 0.f ? v : (v != v ? v : 0.f);
  if (act == 2) return 1.f / (1.f + expf(-v));
  return v;
}

// A row is held in the registers of LPR lanes (4, 16 or 64), CH chunks of 16 bytes of x a
// lane, between its maximum and its rounding: x is read once, with 16-byte loads, and the
// rows of a wave's other lanes keep more loads on their way.  Bound by bytes.
// Loads and stores of a whole chunk need their element's alignment only (rows of odd
// lengths: k = 1023).
template <typename T> struct Chunk;
template <> struct Chunk<float> {
  static constexpr int V = 4;
  typedef float X __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Chunk<bf16> {
  static constexpr int V = 8;
  typedef bf16 X __attribute__((ext_vector_type(8), aligned(2)));
};

// columns [c, c + V) of a row; those from k on are zero
template <typename T>
__device__ __forceinline__ void load_chunk(const T* row, int c, int k, float (&v)[Chunk<T>::V]) {
  constexpr int V = Chunk<T>::V;
  if (c + V <= k) {
    const typename Chunk<T>::X x = *reinterpret_cast<const typename Chunk<T>::X*>(row + c);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)x[e];
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = c + e < k ? to_f32(row[c + e]) : 0.f;
  }
}

template <int LPR>
__device__ __forceinline__ unsigned row_max(unsigned a) {
#pragma unroll
  for (int h = LPR / 2; h > 0; h >>= 1) a = max(a, (unsigned)__shfl_xor((int)a, h));
  return a;
}

// R * 256 / LPR rows, from the block's first on, a workgroup of 256 threads.  q may be null: the
// scales alone.
template <typename T, int LPR, int CH, int R>
__device__ __forceinline__ void quantize_rows_block(int64_t block, const T* __restrict__ x, int64_t rows, int k,
                                                    int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                                                    float* __restrict__ scale) {
  constexpr int V = Chunk<T>::V;
  const int64_t m0 = block * (R * 256 / LPR) + threadIdx.x / LPR;  // and every 256 / LPR-th after it
  const int l = threadIdx.x % LPR;
  float v[R][CH][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < CH; ++i)
      load_chunk(x + min(m0 + r * (256 / LPR), rows - 1) * ldx, (i * LPR + l) * V, k, v[r][i]);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t m = m0 + r * (256 / LPR);
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) a = max(a, abs_bits(v[r][i][e]));
    const RowScale rs = row_scale(row_max<LPR>(a));
    if (m >= rows) return;  // (whole rows of lanes; those that follow are past the end too)
    if (l == 0) scale[m] = rs.s;
    if (q == nullptr) continue;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = (i * LPR + l) * V;
      if (c >= k) break;
      uint32_t w[V / 4];
#pragma unroll
      for (int e = 0; e < V; e += 4)
        w[e / 4] = quantize4<T>(v[r][i][e], v[r][i][e + 1], v[r][i][e + 2], v[r][i][e + 3], rs);
      int8_t* const to = q + m * ldq + c;
      if (c + V <= k) {
#pragma unroll
        for (int e = 0; e < V / 4; ++e) reinterpret_cast<uint32_t*>(to)[e] = w[e];
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (c + e < k) to[e] = (int8_t)(w[e / 4] >> (8 * (e % 4)));
      }
    }
  }
}

// How many lanes hold a row of k values, in how many chunks each, and how many rows they hold at a
// time: f(LPR, CH, R) is called with them as constants; false where no wave holds such a row.  The
// fewest lanes that hold a row in one chunk each, then more chunks a lane; 64 values a lane is the
// most that still leaves several waves a SIMD.  With rows for all CUs, short ones four at a time:
// 262,144 x 256 bf16 84 -> 53 us; longer ones are not faster two at a time (x 1024: 171, 189).
template <typename T, class F>
bool with_row_layout(int64_t rows, int k, const F& f) {
  const int chunks = (int)ceil_div(k, Chunk<T>::V);
  const bool many = rows * chunks >= (1 << 20);
  auto one = [&](auto lpr) {
    if (many) f(lpr, Const<1>{}, Const<4>{});
    else f(lpr, Const<1>{}, Const<1>{});
  };
  if (chunks <= 4) one(Const<4>{});
  else if (chunks <= 8) one(Const<8>{});
  else if (chunks <= 16) one(Const<16>{});
  else if (chunks <= 32) one(Const<32>{});
  else if (chunks <= 64) one(Const<64>{});
  else if (chunks <= 128) f(Const<64>{}, Const<2>{}, Const<1>{});
  else if (chunks <= 256) f(Const<64>{}, Const<4>{}, Const<1>{});
  else if (chunks <= 512) f(Const<64>{}, Const<8>{}, Const<1>{});
  else if (Chunk<T>::V == 4 && chunks <= 1024) f(Const<64>{}, Const<Chunk<T>::V == 4 ? 16 : 8>{}, Const<1>{});
  else return false;
  return true;
}

}  // namespace q8

int launch_quantize_rows(const void* x, int dtype, int64_t rows, int k, int64_t ldx, int8_t* q, int64_t ldq,
                         float* scale, hipStream_t stream);

}  // namespace inf
