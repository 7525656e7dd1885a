// A linear layer on rows and weights in 8-bit whole numbers (quant.hpp), for rendering:
//   acc_mn = sum_k qx_mk qw_nk                              exact, in 32 bits (k <= 2^17)
//   z_mn   = fl(fl(acc) fl(sx_m sw_n)) + bias_n + add_mn    each operation rounded once to fp32
//   y      = act(z), as fp32, rounded again to bf16, or in 8-bit rows again
// The roundings are written out one by one and never contracted: a row that goes into 8
// bits again has the same numbers whichever kernel made it.
//
// Four kernels.  Up to 16 rows: linear8_few_kernel, one launch, bound by its latency and by
// reading the weights once.  Up to 256 outputs: one launch that holds the weight and walks over
// the rows, linear8_rows_kernel (in LDS; many rows of up to 256 values) or linear8_long_kernel (in
// registers; up to 1024).  Otherwise x goes into 8 bits in a launch of its own (rows8.hip: a row's
// maximum is needed before its first product), then linear8_tile_kernel.
#include <algorithm>

#include "mtile.hpp"

namespace inf {
namespace {

using namespace q8;
using namespace mt;

struct Linear8Args {
  int64_t rows;
  int n, k;
  const int8_t* q;
  int64_t ldq;
  const float* qs;
  const int8_t* w;
  int64_t ldw;
  const float* ws;
  const float* bias;
  const float* add;
  int64_t ldadd;
  int act;
  void* out;
  int64_t ldo;
  float* os;  // scales of an int8 result
};

__device__ __forceinline__ float combine(int acc, float sx, float sw, float bias) {
#pragma clang fp contract(off)
  const float z = (float)acc * (sx * sw);
  return z + bias;
}
__device__ __forceinline__ float combine(int acc, float sx, float sw, float bias, float add, int act) {
  return activate(combine(acc, sx, sw, bias) + add, act);
}

// four neighbouring results of a row, as they are stored
template <typename T> struct Four;
template <> struct Four<float> { typedef float V __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Four<bf16> { typedef bf16 V __attribute__((ext_vector_type(4), aligned(2))); };

// ---- tiles ---------------------------------------------------------------------------
// BM rows of x by BN rows of the weight a workgroup, WM x WN waves, v_mfma_i32_16x16x64_i8.
// The weight is the instruction's first operand, so that a lane holds four neighbouring
// outputs of one row.  Per turn 128 values of k: both operands go straight from memory to LDS
// (two stages: the next one is on its way while this one is multiplied).  Behind k the
// weight's rows are zero, so what x's side reads there does not matter; rows past the end are
// the last row again and are not stored.
// T = int8_t: a row of the result goes into 8 bits here; BN holds all of its n values.
template <int BM, int BN, int WM, int WN>
struct L8 {
  static constexpr int THREADS = 64 * WM * WN;
  static constexpr int WROWS = BM / WM, WCOLS = BN / WN, TI = WROWS / 16, TJ = WCOLS / 16;
  static constexpr int STAGE = (BM + BN) * 128, LDS = 2 * STAGE;
  static constexpr int LOADS = STAGE / (THREADS * 16);
  static_assert(STAGE % (THREADS * 16) == 0 && LDS <= 160 * 1024 && TI >= 1 && TJ >= 1, "tile");
  static_assert(BM * WN * 4 + BM * BN <= LDS, "the result's image fits the stages");
};

template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void linear8_tile_kernel(Linear8Args a, int tiles_n, int nblocks) {
  using P = L8<BM, BN, WM, WN>;
  constexpr int TI = P::TI, TJ = P::TJ;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int bid = xcd_order((int)blockIdx.x, nblocks);
  const int64_t m0 = (int64_t)(bid / tiles_n) * BM;
  const int n0 = (bid % tiles_n) * BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave / WN, wc = wave % WN, r16 = lane & 15, g4 = lane >> 4;

  const char* src[P::LOADS];
#pragma unroll
  for (int i = 0; i < P::LOADS; ++i) {
    const int p = tid + P::THREADS * i, row = p >> 3;
    const int c = (p & 7) ^ swz(row);  // LDS is filled in order: the swizzle is the source's
    if (row < BN) {
      src[i] = reinterpret_cast<const char*>(a.w + min(n0 + row, a.n - 1) * a.ldw) + c * 16;
    } else {
      src[i] = reinterpret_cast<const char*>(a.q + min(m0 + row - BN, a.rows - 1) * a.ldq) + c * 16;
    }
  }
  auto issue = [&](int t) {
    char* st = smem + (t & 1) * P::STAGE;
#pragma unroll
    for (int i = 0; i < P::LOADS; ++i) {
      const char* from = src[i] + t * 128;
      __builtin_amdgcn_global_load_lds(from, (lds_void*)(st + (wave + (P::THREADS / 64) * i) * 1024), 16, 0, 0);
    }
  };
  i32x4 acc[TJ][TI];
#pragma unroll
  for (int j = 0; j < TJ; ++j)
#pragma unroll
    for (int i = 0; i < TI; ++i) acc[j][i] = i32x4{0, 0, 0, 0};

  const int turns = (int)(a.ldw / 128);
  issue(0);
#pragma unroll 1
  for (int t = 0; t < turns; ++t) {
    wait_all_barrier();
    if (t + 1 < turns) issue(t + 1);
    const char* st = smem + (t & 1) * P::STAGE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x4 wf[TJ], xf[TI];
#pragma unroll
      for (int j = 0; j < TJ; ++j)
        wf[j] = *reinterpret_cast<const i32x4*>(st + chunk_at(wc * P::WCOLS + 16 * j + r16, 4 * h + g4));
#pragma unroll
      for (int i = 0; i < TI; ++i)
        xf[i] = *reinterpret_cast<const i32x4*>(st + chunk_at(BN + wr * P::WROWS + 16 * i + r16, 4 * h + g4));
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int i = 0; i < TI; ++i)
          acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[i], acc[j][i], 0, 0, 0);
    }
  }

  // lane: row wr WROWS + 16 i + r16, columns wc WCOLS + 16 j + 4 g4 + (0..3)
  float z[TJ][TI][4];
  float sx[TI];
#pragma unroll
  for (int i = 0; i < TI; ++i) sx[i] = a.qs[min(m0 + wr * P::WROWS + 16 * i + r16, a.rows - 1)];
#pragma unroll
  for (int j = 0; j < TJ; ++j) {
    const int n = n0 + wc * P::WCOLS + 16 * j + 4 * g4;
    float sw[4], bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sw[e] = a.ws[min(n + e, a.n - 1)];
      bias[e] = a.bias != nullptr ? a.bias[min(n + e, a.n - 1)] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int64_t m = m0 + wr * P::WROWS + 16 * i + r16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float add = a.add != nullptr && m < a.rows && n + e < a.n ? a.add[m * a.ldadd + n + e] : 0.f;
        z[j][i][e] = combine(acc[j][i][e], sx[i], sw[e], bias[e], add, a.act);
      }
    }
  }
  if constexpr (sizeof(T) == 1) {
    unsigned* const top = reinterpret_cast<unsigned*>(smem);  // [BM][WN]
    char* const image = smem + BM * WN * 4;                    // [BM][BN]
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      unsigned b = 0;
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (wc * P::WCOLS + 16 * j + 4 * g4 + e < a.n) b = max(b, abs_bits(z[j][i][e]));
      b = max(b, (unsigned)__shfl_xor((int)b, 16));
      b = max(b, (unsigned)__shfl_xor((int)b, 32));
      if (g4 == 0) top[(wr * P::WROWS + 16 * i + r16) * WN + wc] = b;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int row = wr * P::WROWS + 16 * i + r16;
      unsigned b = 0;
#pragma unroll
      for (int v = 0; v < WN; ++v) b = max(b, top[row * WN + v]);
      const RowScale rs = row_scale(b);
      if (wc == 0 && g4 == 0 && m0 + row < a.rows) a.os[m0 + row] = rs.s;
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        const int col = wc * P::WCOLS + 16 * j + 4 * g4;
        *reinterpret_cast<uint32_t*>(image + row * BN + (((col >> 4) ^ (row & (BN / 16 - 1))) << 4) + (col & 15)) =
            quantize4(z[j][i][0], z[j][i][1], z[j][i][2], z[j][i][3], rs);
      }
    }
    __syncthreads();
    // whole 16-byte pieces: q rows are multiples of 16, so a piece that begins before n fits
    for (int p = tid; p < BM * (BN / 16); p += P::THREADS) {
      const int row = p / (BN / 16), c = p % (BN / 16);
      if (m0 + row < a.rows && c * 16 < a.n)
        *reinterpret_cast<u32x4*>((int8_t*)a.out + (m0 + row) * a.ldo + c * 16) =
            *reinterpret_cast<const u32x4*>(image + row * BN + ((c ^ (row & (BN / 16 - 1))) << 4));
    }
  } else {
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int n = n0 + wc * P::WCOLS + 16 * j + 4 * g4;
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const int64_t m = m0 + wr * P::WROWS + 16 * i + r16;
        if (m >= a.rows) continue;
        T* const to = reinterpret_cast<T*>(a.out) + m * a.ldo + n;
        if (n + 4 <= a.n) {
          typename Four<T>::V v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(z[j][i][e]);
          *reinterpret_cast<typename Four<T>::V*>(to) = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.n) to[e] = from_f32<T>(z[j][i][e]);
        }
      }
    }
  }
}

// ---- up to 16 rows -------------------------------------------------------------------
// A workgroup makes 16 columns of every row, its four waves a quarter of the turns each, and
// adds their sums in LDS.  It puts x into 8 bits itself (all workgroups the same numbers):
// one launch, and x is small next to the weight.  X: float, bf16, or int8_t rows.
constexpr int FEW = 16;
constexpr int FEW_LDS = 128 * 1024;  // x in 8 bits: 16 rows of up to 8 K

template <typename X, typename T>
__global__ __launch_bounds__(256) void linear8_few_kernel(Linear8Args a, const X* __restrict__ x, int64_t ldx,
                                                          int log_rows) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ unsigned top[FEW];
  __shared__ int part[4][16][FEW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g4 = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int ld = (int)a.ldw + 16;  // LDS rows: 16 bytes apart in the banks
  const int rows = (int)a.rows;
  const int turns = (int)(a.ldw / 64);
  const int8_t* const wrow = a.w + min(n0 + r16, a.n - 1) * a.ldw + 16 * g4;
  constexpr int AHEAD = 4;
  i32x4 wf[AHEAD];
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {  // on their way while x is put into 8 bits
    const int t = wave + 4 * u;
    if (t < turns) wf[u] = *reinterpret_cast<const i32x4*>(wrow + t * 64);
  }
  // 256 >> log_rows threads a row, 16 bytes of the result each
  const int per = 256 >> log_rows, m = tid / per, l = tid % per;
  if constexpr (sizeof(X) == 1) {
    if (m < rows)
      for (int c = l * 16; c < a.ldw; c += per * 16)
        *reinterpret_cast<i32x4*>(smem + m * ld + c) =
            c < a.k ? *reinterpret_cast<const i32x4*>(x + m * ldx + c) : i32x4{0, 0, 0, 0};
  } else {
    if (tid < FEW) top[tid] = 0;
    __syncthreads();
    if (m < rows) {
      unsigned b = 0;
      for (int c = l; c < a.k; c += per) b = max(b, abs_bits(to_f32(x[m * ldx + c])));
      atomicMax(&top[m], b);
    }
    __syncthreads();
    if (m < rows) {
      const RowScale rs = row_scale(top[m]);
      for (int c = l * 4; c < a.ldw; c += per * 4) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < a.k ? to_f32(x[m * ldx + c + e]) : 0.f;
        *reinterpret_cast<uint32_t*>(smem + m * ld + c) = quantize4<X>(v[0], v[1], v[2], v[3], rs);
      }
    }
  }
  __syncthreads();
  i32x4 acc = {0, 0, 0, 0};
  // rows past the end read row 0; their sums are not stored
  const char* const xrow = smem + (r16 < rows ? r16 : 0) * ld + 16 * g4;
  for (int t0 = wave; t0 < turns; t0 += 4 * AHEAD) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int t = t0 + 4 * u;
      if (t < turns) {
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], *reinterpret_cast<const i32x4*>(xrow + t * 64), acc, 0, 0, 0);
        if (t + 4 * AHEAD < turns) wf[u] = *reinterpret_cast<const i32x4*>(wrow + (t + 4 * AHEAD) * 64);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) part[wave][4 * g4 + e][r16] = acc[e];
  __syncthreads();
  const int r = tid / 16, n = n0 + tid % 16;
  if (r < rows && n < a.n) {
    const int sum = part[0][tid % 16][r] + part[1][tid % 16][r] + part[2][tid % 16][r] + part[3][tid % 16][r];
    const float sx = sizeof(X) == 1 ? a.qs[r] : row_scale(top[r]).s;
    const float y = combine(sum, sx, a.ws[n], a.bias != nullptr ? a.bias[n] : 0.f,
                            a.add != nullptr ? a.add[r * a.ldadd + n] : 0.f, a.act);
    reinterpret_cast<T*>(a.out)[r * a.ldo + n] = from_f32<T>(y);
  }
}

// ---- many rows, the weight in LDS -------------------------------------------------------
// A workgroup (one a CU) holds the whole weight in LDS and walks over the rows; a wave owns 16 of
// them at a time with all their outputs, so that nothing is exchanged between waves and no
// barrier is left in the loop.  x goes from memory into the registers that the instruction reads
// (v_mfma_i32_16x16x64_i8), the next rows' while these are worked on; fp32 and bf16 rows are put
// into 8 bits there, and so are the results, whose row maximum is two exchanges between lanes.
// Bound by the vector operations, a wave's phases of which and of matrix instructions overlap in part (a value
// in: 9 operations, none from 8 bits; a result: 6, 15 into 8 bits), and by bytes.  262,144 x 256 x 256, us: bf16
// into 8 bits 63, 8 bits into 8 bits 44 (their bytes: 39, 26), 8 bits into bf16 52 (39).
//   k runs over KS blocks of 64.  Within a block, byte p of lane group g's 16 is k = G (4 p / G +
//   g) + p % G with G = 16 bytes of x (4 fp32, 8 bf16, 16 int8 values): each load of 16 bytes then
//   lies next to the neighbouring lane groups'.  The weight is laid out the same way on its way to
//   LDS, in the order of the lanes that read it: a KiB for 16 outputs and 64 k.  Behind k its bytes are zero.
template <typename X> constexpr int granule() { return 16 / sizeof(X); }
constexpr int WALK_WAVES = 8;  // (16 have 128 registers each, and spill)

template <typename X, typename T, int KS, int TJ>
struct LR {
  static constexpr int NW = WALK_WAVES;
  static constexpr int THREADS = 64 * NW;
  static constexpr int OS = TJ * 16 + 16;                     // a result row in 8 bits
  static constexpr int WEIGHT = TJ * KS * 1024, SCALES = TJ * 16 * 8, OUT = sizeof(T) == 1 ? NW * 16 * OS : 0;
  static constexpr int LDS = WEIGHT + SCALES + OUT;
  static_assert(LDS <= 160 * 1024, "LDS");
};

template <typename X, typename T, int KS, int TJ>
__global__ __launch_bounds__(64 * WALK_WAVES) void linear8_rows_kernel(Linear8Args a, const X* __restrict__ x,
                                                                                 int64_t ldx) {
  using P = LR<X, T, KS, TJ>;
  constexpr int G = granule<X>(), L = 16 / G;  // values of a load, loads of a block
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* const sws = reinterpret_cast<float*>(smem + P::WEIGHT);  // scales, then biases
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g4 = lane >> 4;

  // the weight: 64 bytes of a row a thread and turn; dword d of them is k = 4 d on
  for (int i = tid; i < TJ * 16 * KS; i += P::THREADS) {
    const int n = i / KS, b = i % KS;
    i32x4 v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      v[c] = b * 64 < a.ldw ? *reinterpret_cast<const i32x4*>(a.w + min(n, a.n - 1) * a.ldw + b * 64 + c * 16)
                            : i32x4{0, 0, 0, 0};
    int* const to = reinterpret_cast<int*>(smem + (n / 16 * KS + b) * 1024 + n % 16 * 16);
#pragma unroll
    for (int d = 0; d < 16; ++d) {
      const int g = d * 4 / G % 4, load = d * 4 / G / 4, at = d * 4 % G;  // whose, in which load, where
      to[g * 64 + (load * G + at) / 4] = v[d / 4][d % 4];
    }
  }
  for (int i = tid; i < TJ * 16; i += P::THREADS) {
    sws[i] = i < a.n ? a.ws[i] : 0.f;  // columns behind the last are zero
    sws[TJ * 16 + i] = i < a.n && a.bias != nullptr ? a.bias[i] : 0.f;
  }
  __syncthreads();

  const int tiles = (int)((a.rows + 15) / 16), step = (int)gridDim.x * P::NW;
  typedef X XV __attribute__((ext_vector_type(G), aligned(sizeof(X))));
  XV raw[KS][L];
  const bool whole = a.k == KS * 64;
  auto fetch = [&](int tile) {
    const X* const row = x + min((int64_t)tile * 16 + r16, a.rows - 1) * ldx + g4 * G;
    if (whole) {
#pragma unroll
      for (int b = 0; b < KS; ++b)
#pragma unroll
        for (int i = 0; i < L; ++i) raw[b][i] = *reinterpret_cast<const XV*>(row + b * 64 + i * 4 * G);
    } else {
#pragma unroll
      for (int b = 0; b < KS; ++b)
#pragma unroll
        for (int i = 0; i < L; ++i) {
          const int k = b * 64 + i * 4 * G, left = a.k - g4 * G - k;  // of these, values in the row
          if constexpr (sizeof(X) == 1) {
            raw[b][i] = *reinterpret_cast<const XV*>(row + (left > 0 ? k : -g4 * G));  // zero weights behind k
          } else if (left >= G) {
            raw[b][i] = *reinterpret_cast<const XV*>(row + k);
          } else {
#pragma unroll
            for (int e = 0; e < G; ++e) raw[b][i][e] = e < left ? row[k + e] : (X)0.f;
          }
        }
    }
  };
  // ReLU in one operation, the maximum that keeps a NaN (inf 0 and inf - inf, of scales, biases and
  // overflows, have a negative sign here: a maximum of whole numbers would make zeros of them; three layers of
  // 262,144 x 256 took 141 us with it, 144 so).  Without ReLU the bound is below everything (and unknown to
  // the compiler, which else selects: an operation more).
  int least = a.act == 1 ? 0 : (int)0xff800000;  // the bits of 0 and of minus infinity
  asm volatile("" : "+s"(least));
  int tile = (int)blockIdx.x * P::NW + wave;
  if (tile < tiles) fetch(tile);
  for (; tile < tiles; tile += step) {
    const int64_t m = (int64_t)tile * 16 + r16;
    i32x4 xf[KS];
    float sx;
    if constexpr (sizeof(X) == 1) {
#pragma unroll
      for (int b = 0; b < KS; ++b) xf[b] = __builtin_bit_cast(i32x4, raw[b][0]);
      sx = a.qs[min(m, a.rows - 1)];
    } else {
      unsigned top = 0;
      if constexpr (sizeof(X) == 2) {  // two values at a time: bf16 is the upper half of its fp32
        u16x2 two = {0, 0};
#pragma unroll
        for (int b = 0; b < KS; ++b)
#pragma unroll
          for (int i = 0; i < L; ++i) {
            const u32x4 v = __builtin_bit_cast(u32x4, raw[b][i]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              two = __builtin_elementwise_max(two, __builtin_bit_cast(u16x2, v[e] & 0x7fff7fffu));
          }
        top = (unsigned)max(two[0], two[1]) << 16;
      } else {
#pragma unroll
        for (int b = 0; b < KS; ++b)
#pragma unroll
          for (int i = 0; i < L; ++i)
#pragma unroll
            for (int e = 0; e < G; ++e) top = max(top, abs_bits((float)raw[b][i][e]));
      }
      top = max(top, (unsigned)__shfl_xor((int)top, 16));
      top = max(top, (unsigned)__shfl_xor((int)top, 32));
      const RowScale rs = row_scale(top);
      sx = rs.s;
#pragma unroll
      for (int b = 0; b < KS; ++b)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int i = d * 4 / G, e = d * 4 % G;
          xf[b][d] = (int)quantize4<X>((float)raw[b][i][e], (float)raw[b][i][e + 1], (float)raw[b][i][e + 2],
                                    (float)raw[b][i][e + 3], rs);
        }
    }
    if (tile + step < tiles) fetch(tile + step);
    i32x4 acc[TJ];
#pragma unroll
    for (int j = 0; j < TJ; ++j) acc[j] = i32x4{0, 0, 0, 0};
    // Eight of the weight's fragments are read while eight are multiplied (one after the other: 68, 52
    // and 50 us for 262,144 x 256 x 256 from bf16 into 8 bits, from and into, into bf16; so 62, 50, 47).
    constexpr int GROUP = 8;
    i32x4 wf[2][GROUP];
    auto load_group = [&](int g) {
#pragma unroll
      for (int u = 0; u < GROUP; ++u) {
        const int j = g * GROUP % TJ + u, b = g * GROUP / TJ;
        wf[g & 1][u] = *reinterpret_cast<const i32x4*>(smem + (j * KS + b) * 1024 + lane * 16);
      }
    };
    load_group(0);
#pragma unroll
    for (int g = 0; g < KS * TJ / GROUP; ++g) {
      if (g + 1 < KS * TJ / GROUP) load_group(g + 1);
#pragma unroll
      for (int u = 0; u < GROUP; ++u) {
        const int j = g * GROUP % TJ + u, b = g * GROUP / TJ;
        acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[g & 1][u], xf[b], acc[j], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // lane: row m, columns 16 j + 4 g4 + (0..3); one j at a time (taken together they need more
    // registers than there are)
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      const int n = 16 * j + 4 * g4;
      const f32x4 sw = *reinterpret_cast<const f32x4*>(sws + n), bias = *reinterpret_cast<const f32x4*>(sws + TJ * 16 + n);
      float z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z[e] = combine(acc[j][e], sx, sw[e], bias[e]);
        z[e] = __builtin_elementwise_maximum(z[e], __int_as_float(least));
      }
      if constexpr (sizeof(T) == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          top = max(top, abs_bits(z[e]));
          acc[j][e] = __float_as_int(z[e]);
        }
      } else if (m < a.rows) {
        T* const to = reinterpret_cast<T*>(a.out) + m * a.ldo + n;
        if (n + 4 <= a.n) {
          typename Four<T>::V v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(z[e]);
          *reinterpret_cast<typename Four<T>::V*>(to) = v;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.n) to[e] = from_f32<T>(z[e]);
        }
      }
    }
    if constexpr (sizeof(T) == 1) {
      top = max(top, (unsigned)__shfl_xor((int)top, 16));
      top = max(top, (unsigned)__shfl_xor((int)top, 32));
      const RowScale rs = row_scale(top);
      if (g4 == 0 && m < a.rows) a.os[m] = rs.s;
      char* const mine = smem + P::WEIGHT + P::SCALES + wave * 16 * P::OS;
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        *reinterpret_cast<uint32_t*>(mine + r16 * P::OS + 16 * j + 4 * g4) =
            quantize4(__int_as_float(acc[j][0]), __int_as_float(acc[j][1]), __int_as_float(acc[j][2]),
                      __int_as_float(acc[j][3]), rs);
      }
      own_lds_order();
#pragma unroll
      for (int i = 0; i < TJ / 4; ++i) {  // 16 rows of TJ chunks of 16 bytes, 64 a turn
        const int r = (i * 64 + lane) / TJ, c = (i * 64 + lane) % TJ;
        if ((int64_t)tile * 16 + r < a.rows && c * 16 < a.n)
          *reinterpret_cast<u32x4*>((int8_t*)a.out + ((int64_t)tile * 16 + r) * a.ldo + c * 16) =
              *reinterpret_cast<const u32x4*>(mine + r * P::OS + c * 16);
      }
      own_lds_order();
    }
  }
}

template <typename X, typename T, int KS, int TJ>
int launch_rows(const Linear8Args& a, const X* x, int64_t ldx, hipStream_t stream) {
  using P = LR<X, T, KS, TJ>;
  const auto kernel = linear8_rows_kernel<X, T, KS, TJ>;
  static LdsLimit lds;
  const int allowed = lds.raise((const void*)kernel, P::LDS);
  if (allowed != INF_OK) return allowed;
  const int64_t groups = ceil_div(a.rows, 16 * P::NW);
  kernel<<<(unsigned)std::min<int64_t>(groups, 256), P::THREADS, P::LDS, stream>>>(a, x, ldx);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

// k up to 256 with up to 256 outputs, from 16,384 rows on: half of the CUs then have a workgroup, of 128 rows
// a turn.  256 x 256, us, here and in tiles: int8 into fp32 rows 9.4 and 6.0 for 8192 rows, 10.2 and 9.7 for 16,384,
// 12.0 and 13.6 for 32,768; bf16 into bf16 10.5 and 9.2, 11.5 and 14.0, 12.6 and 22.5 (into 8 bits this is
// ahead from fewer rows on: int8 8.1 and 12.5 for 8192).  Fewer outputs than 33 are bound by x's bytes whichever
// kernel reads them; a sigmoid or a sum to add to is a head's or a skip layer's, one a network.
bool rows_walk(int64_t rows, int n, int k, int act, bool with_add) {
  return rows >= 16384 && k <= 256 && n > 32 && n <= 256 && act != 2 && !with_add;
}

template <typename X, typename T>
int launch_rows_any(const Linear8Args& a, const void* x, int64_t ldx, hipStream_t stream) {
  if (a.k <= 128)
    return a.n <= 128 ? launch_rows<X, T, 2, 8>(a, (const X*)x, ldx, stream)
                      : launch_rows<X, T, 2, 16>(a, (const X*)x, ldx, stream);
  return a.n <= 128 ? launch_rows<X, T, 4, 8>(a, (const X*)x, ldx, stream)
                    : launch_rows<X, T, 4, 16>(a, (const X*)x, ldx, stream);
}

template <typename X>
int launch_rows_out(const Linear8Args& a, int out_dtype, const void* x, int64_t ldx, hipStream_t stream) {
  if (out_dtype == INF_DTYPE_I8) return launch_rows_any<X, int8_t>(a, x, ldx, stream);
  if (out_dtype == INF_DTYPE_BF16) return launch_rows_any<X, bf16>(a, x, ldx, stream);
  return launch_rows_any<X, float>(a, x, ldx, stream);
}

// ---- many long rows, up to 256 outputs -----------------------------------------------------
// A workgroup of 16 waves (one a CU) holds the whole weight in registers, 16 outputs a wave, as the
// instruction reads them, and walks over the rows, 32 at a time: each row of x, fp32 or bf16, is held in
// one wave's registers between its maximum and its rounding and goes to LDS in 8 bits, where every wave
// reads it; the next rows are on their way meanwhile.  Two stages, so one barrier a turn.
// 262,144 x 1024 x 256, us: fp32 260, its bytes at a copy's rate (in 8 bits through memory, then
// tiles: 414); bf16 186, where they would take 156 (264).  32 rows a turn where the registers hold them
// (16: 262,144 x 512 x 256, bf16 166 where these take 142), fp32 rows of more than 512 values 16 (32 spill:
// 394 where these take 260).
constexpr int LONG_WAVES = 16, LONG_K = 1024;

template <typename X, typename T, int CH, int ROWS>
struct LL {
  static constexpr int V = Chunk<X>::V, K = CH * 64 * V, BLOCKS = K / 128;  // the longest row
  static constexpr int THREADS = 64 * LONG_WAVES, R = ROWS / LONG_WAVES;
  static constexpr int STAGE = BLOCKS * ROWS * 128, SCALES = 2 * STAGE;
  static constexpr int TOPS = SCALES + 2 * ROWS * 4, IMAGE = TOPS + 2 * ROWS * 4;
  static constexpr int WS = IMAGE + (sizeof(T) == 1 ? ROWS * 256 : 0), LDS = WS + 16 * LONG_WAVES * 8;
  static_assert(LDS <= 160 * 1024, "LDS");
};

template <typename X, typename T, int CH, int ROWS>
__global__ __launch_bounds__(64 * LONG_WAVES) void linear8_long_kernel(Linear8Args a, const X* __restrict__ x,
                                                                        int64_t ldx) {
  using P = LL<X, T, CH, ROWS>;
  constexpr int V = P::V, R = P::R, TI = ROWS / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles = (int)((a.rows + ROWS - 1) / ROWS), blocks = (int)(a.ldw / 128);
  const bool busy = wave * 16 < a.n;

  i32x4 w[P::BLOCKS][2];
  float* const sws = reinterpret_cast<float*>(smem + P::WS);  // scales, then biases
  if (tid < 16 * LONG_WAVES) {
    sws[tid] = a.ws[min(tid, a.n - 1)];
    sws[16 * LONG_WAVES + tid] = a.bias != nullptr ? a.bias[min(tid, a.n - 1)] : 0.f;
  }
  {
    const char* const from = reinterpret_cast<const char*>(a.w + min(wave * 16 + lane % 16, a.n - 1) * a.ldw) + lane / 16 * 16;
#pragma unroll
    for (int b = 0; b < P::BLOCKS; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[b][h] = busy && b < blocks ? *reinterpret_cast<const i32x4*>(from + b * 128 + h * 64) : i32x4{0, 0, 0, 0};
  }

  // A chunk across the end of a row is loaded from its last V values and moved down when it is used
  // (no branch around a load: the loads stay on their way).
  typename Chunk<X>::X raw[R][CH];
  // Of rows that fill the registers, each turn works its addresses out again from the lane's number:
  // kept, they do not fit (284 us where these take 260).  Of shorter ones they do, and cost less: 262,144 x
  // 512 x 256 into bf16 169 and 142.
  auto this_lane = [&]() { return P::BLOCKS == LONG_K / 128 ? (int)pinned(tid & 63) : tid & 63; };
  auto fetch = [&](int tile) {
    const int lane = this_lane();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const X* const row = x + min((int64_t)tile * ROWS + wave * R + r, a.rows - 1) * ldx;
#pragma unroll
      for (int i = 0; i < CH; ++i)
        raw[r][i] = *reinterpret_cast<const typename Chunk<X>::X*>(
            reinterpret_cast<const char*>(row) + (unsigned)min((i * 64 + lane) * V, a.k - V) * sizeof(X));
    }
  };
  if (sizeof(T) == 1 && tid < 2 * ROWS) reinterpret_cast<unsigned*>(smem + P::TOPS)[tid] = 0;
  int tile = (int)blockIdx.x;
  if (tile < tiles) fetch(tile);
#pragma unroll 1
  for (int t = 0; tile < tiles; ++t) {
    const int lane = this_lane();
    char* const st = smem + (t & 1) * P::STAGE;
    float* const sxs = reinterpret_cast<float*>(smem + P::SCALES) + (t & 1) * ROWS;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      __builtin_amdgcn_sched_barrier(0);
      const int row = wave * R + r;
      float v[CH][V];
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = to_f32(raw[r][i][e]);
        if ((i + 1) * 64 * V > a.k) {
          const int past = (i * 64 + lane + 1) * V - a.k;  // values of the chunk behind the row's end
#pragma unroll
          for (int h = 1; h < V; h *= 2)
            if (past > 0 && (past & h))
#pragma unroll
              for (int e = 0; e < V; ++e) v[i][e] = e + h < V ? v[i][e + h] : 0.f;
          if (past >= V)
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) top = max(top, abs_bits(v[i][e]));
      }
      const RowScale rs = row_scale(row_max<64>(top));
      if (lane == 0) sxs[row] = rs.s;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = (i * 64 + lane) * V;
        uint32_t q[V / 4];
#pragma unroll
        for (int e = 0; e < V; e += 4) q[e / 4] = quantize4<X>(v[i][e], v[i][e + 1], v[i][e + 2], v[i][e + 3], rs);
        char* const to = st + c / 128 * ROWS * 128 + chunk_at(row, c % 128 / 16) + c % 16;
        if constexpr (V == 4) *reinterpret_cast<uint32_t*>(to) = q[0];
        else *reinterpret_cast<u32x2*>(to) = u32x2{q[0], q[V / 4 - 1]};
      }
    }
    const int64_t m0 = (int64_t)tile * ROWS;
    tile += (int)gridDim.x;
    __builtin_amdgcn_sched_barrier(0);
    if (tile < tiles) fetch(tile);
    wait_lds_barrier();

    const int again = this_lane(), r16 = again & 15, g4 = again >> 4, n = wave * 16 + 4 * g4;  // n: this lane's outputs
    i32x4 acc[TI];
#pragma unroll
    for (int i = 0; i < TI; ++i) acc[i] = i32x4{0, 0, 0, 0};
    if (busy) {
#pragma unroll
      for (int b = 0; b < P::BLOCKS; ++b) {
        __builtin_amdgcn_sched_barrier(0);
        if (b < blocks)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < TI; ++i) {
              const i32x4 xf =
                  *reinterpret_cast<const i32x4*>(st + b * ROWS * 128 + chunk_at(16 * i + r16, 4 * h + g4));
              acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[b][h], xf, acc[i], 0, 0, 0);
            }
      }
    }
    // lane: row 16 i + r16, outputs n + (0..3)
    __builtin_amdgcn_sched_barrier(0);
    const f32x4 sw = *reinterpret_cast<const f32x4*>(sws + n), bias = *reinterpret_cast<const f32x4*>(sws + 16 * LONG_WAVES + n);
    f32x4 z[TI];
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int64_t m = m0 + 16 * i + r16;
      const float sx = sxs[16 * i + r16];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[i][e] = combine(acc[i][e], sx, sw[e], bias[e]);
      if (a.add != nullptr)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[i][e] += a.add[min(m, a.rows - 1) * a.ldadd + min(n + e, a.n - 1)];
      if (a.act == 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[i][e] = activate(z[i][e], 1);
      if (a.act == 2)  // one copy of its code for the four
#pragma unroll 1
        for (int e = 0; e < 4; ++e) z[i] = f32x4{z[i][1], z[i][2], z[i][3], activate(z[i][0], 2)};
      if constexpr (sizeof(T) != 1) {
        if (m >= a.rows) continue;
        T* const to = reinterpret_cast<T*>(a.out) + m * a.ldo + n;
        if (n + 4 <= a.n) {
          typename Four<T>::V o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(z[i][e]);
          *reinterpret_cast<typename Four<T>::V*>(to) = o;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.n) to[e] = from_f32<T>(z[i][e]);
        }
      }
    }
    if constexpr (sizeof(T) == 1) {
      unsigned* const tops = reinterpret_cast<unsigned*>(smem + P::TOPS) + (t & 1) * ROWS;
      char* const image = smem + P::IMAGE;
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        unsigned b = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < a.n) b = max(b, abs_bits(z[i][e]));
        b = max(b, (unsigned)__shfl_xor((int)b, 16));
        b = max(b, (unsigned)__shfl_xor((int)b, 32));
        if (g4 == 0 && busy) atomicMax(&tops[16 * i + r16], b);  // a maximum: in any order the same
      }
      // the other turn's maxima: last read before this turn's first barrier, next used after its last
      if (tid < ROWS) reinterpret_cast<unsigned*>(smem + P::TOPS)[((t + 1) & 1) * ROWS + tid] = 0;
      wait_lds_barrier();
      if (tid < ROWS && m0 + tid < a.rows) a.os[m0 + tid] = row_scale(tops[tid]).s;
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const int row = 16 * i + r16;
        if (busy)
          *reinterpret_cast<uint32_t*>(image + row * 256 + ((wave ^ r16) << 4) + 4 * g4) =
              quantize4(z[i][0], z[i][1], z[i][2], z[i][3], row_scale(tops[row]));
      }
      wait_lds_barrier();
      // whole 16-byte pieces: q rows are multiples of 16, so a piece that begins before n fits
      if (tid < ROWS * 16) {
        const int row = tid / 16, c = tid % 16;
        if (m0 + row < a.rows && c * 16 < a.n)
          *reinterpret_cast<u32x4*>((int8_t*)a.out + (m0 + row) * a.ldo + c * 16) =
              *reinterpret_cast<const u32x4*>(image + row * 256 + ((c ^ (row & 15)) << 4));
      }
    }
  }
}

template <typename X, typename T, int CH, int ROWS>
int launch_long_as(const Linear8Args& a, const X* x, int64_t ldx, hipStream_t stream) {
  using P = LL<X, T, CH, ROWS>;
  const auto kernel = linear8_long_kernel<X, T, CH, ROWS>;
  static LdsLimit lds;
  const int allowed = lds.raise((const void*)kernel, P::LDS);
  if (allowed != INF_OK) return allowed;
  kernel<<<(unsigned)std::min<int64_t>(ceil_div(a.rows, ROWS), 256), P::THREADS, P::LDS, stream>>>(a, x, ldx);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

template <typename X>
int launch_long(const Linear8Args& a, int out_dtype, const void* x, int64_t ldx, hipStream_t stream) {
  constexpr int CH = LONG_K / 64 / Chunk<X>::V;
  const auto go = [&](auto t) {
    using T = decltype(t);
    return a.k <= LONG_K / 2 ? launch_long_as<X, T, CH / 2, 32>(a, (const X*)x, ldx, stream)
                             : launch_long_as<X, T, CH, sizeof(X) == 4 ? 16 : 32>(a, (const X*)x, ldx, stream);
  };
  if (out_dtype == INF_DTYPE_I8) return go(int8_t{});
  if (out_dtype == INF_DTYPE_BF16) return go(bf16{});
  return go(float{});
}

template <typename T, int BM, int BN, int WM, int WN>
int launch_tile(const Linear8Args& a, hipStream_t stream) {
  using P = L8<BM, BN, WM, WN>;
  const int tiles_n = (int)ceil_div(a.n, BN);
  const int64_t nblocks = ceil_div(a.rows, BM) * tiles_n;
  INF_CHECK_ARG(nblocks * P::THREADS < (int64_t)1 << 32, "linear_int: too many tiles");
  static LdsLimit lds;
  const int allowed = lds.raise((const void*)linear8_tile_kernel<T, BM, BN, WM, WN>, P::LDS);
  if (allowed != INF_OK) return allowed;
  linear8_tile_kernel<T, BM, BN, WM, WN>
      <<<(unsigned)nblocks, P::THREADS, P::LDS, stream>>>(a, tiles_n, (int)nblocks);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

// The widest tile that still gives every CU a workgroup (256 of them); a result in 8 bits
// needs whole rows (n <= 256).  4096 x 4096 x 2048, us: 128 x 128 43, 64 x 64 60, 256 x 256 (half the
// CUs) 59; 2048 x 4096 x 1024: 128 x 128 (half the CUs) 27, 64 x 64 21.
template <typename T>
int launch_tiles(const Linear8Args& a, hipStream_t stream) {
  const int64_t wide = ceil_div(a.rows, 256);
  if (a.n <= 32) return launch_tile<T, 256, 32, 4, 1>(a, stream);
  if (a.n <= 128 && wide >= 256) return launch_tile<T, 256, 128, 8, 2>(a, stream);
  if (a.n > 128 && wide * ceil_div(a.n, 256) >= 256) return launch_tile<T, 256, 256, 4, 4>(a, stream);
  if constexpr (sizeof(T) != 1)
    if (a.n > 64 && ceil_div(a.rows, 128) * ceil_div(a.n, 128) >= 256) return launch_tile<T, 128, 128, 4, 2>(a, stream);
  if (sizeof(T) == 1 && a.n > 64) return launch_tile<T, 64, 256, 1, 4>(a, stream);
  return launch_tile<T, 64, 64, 2, 2>(a, stream);
}

int launch_linear8(const Linear8Args& a, int out_dtype, hipStream_t stream) {
  if (out_dtype == INF_DTYPE_I8) return launch_tiles<int8_t>(a, stream);
  if (out_dtype == INF_DTYPE_BF16) return launch_tiles<bf16>(a, stream);
  return launch_tiles<float>(a, stream);
}

template <typename X, typename T>
int launch_few(const Linear8Args& a, const X* x, int64_t ldx, hipStream_t stream) {
  static LdsLimit lds;
  const int allowed = lds.raise((const void*)linear8_few_kernel<X, T>, FEW_LDS);
  if (allowed != INF_OK) return allowed;
  int log_rows = 0;
  while ((1 << log_rows) < a.rows) ++log_rows;
  linear8_few_kernel<X, T><<<(unsigned)ceil_div(a.n, 16), 256, (size_t)(a.rows * (a.ldw + 16)), stream>>>(a, x, ldx,
                                                                                                       log_rows);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

template <typename X>
int launch_few_out(const Linear8Args& a, int out_dtype, const void* x, int64_t ldx, hipStream_t stream) {
  if (out_dtype == INF_DTYPE_BF16) return launch_few<X, bf16>(a, (const X*)x, ldx, stream);
  return launch_few<X, float>(a, (const X*)x, ldx, stream);
}

bool is_few(int64_t rows, int k) { return rows <= FEW && rows * (round_up(k, W_ALIGN) + 16) <= FEW_LDS; }
// Rows of any number that are longer than linear8_rows_kernel's.  4096 x 1024, us: 64 outputs 9 (in two
// launches 5 + 8), 256 outputs 13 (5 + 8); 128 rows 8 (4 + 7) and 12 (4 + 8).
bool takes_long(int64_t rows, int n, int k, int x_dtype) {
  return x_dtype != INF_DTYPE_I8 && !is_few(rows, k) && k > 256 && k <= LONG_K && n <= 16 * LONG_WAVES;
}
// whether a result in 8 bits is made by the product's own kernel
bool rows_whole(int64_t rows, int n, int k) { return n <= 256 && !is_few(rows, k); }

// Which kernel makes the products of a call: the workspace's size and the launch go by the same rule.
// (Calls in several turns have thousands of rows in each, so that the rule names the same kernel for them.)
enum class Form { FEW, WALK, LONG, TILES };
Form form_of(int64_t rows, int n, int k, int x_dtype, int act, bool with_add) {
  if (is_few(rows, k)) return Form::FEW;
  if (rows_walk(rows, n, k, act, with_add)) return Form::WALK;
  return takes_long(rows, n, k, x_dtype) ? Form::LONG : Form::TILES;
}

struct Workspace {
  int64_t q, qs, y, bytes;  // offsets: x in 8 bits, its scales, the fp32 rows that go into 8 bits
};

Workspace workspace_of(Form form, int64_t rows, int n, int k, int x_dtype, int out_dtype) {
  Workspace w{0, 0, 0, 0};
  if (x_dtype != INF_DTYPE_I8 && form == Form::TILES) {
    w.q = w.bytes;
    w.bytes += round_up(rows * round_up(k, Q_ALIGN) + Q_SLACK, 256);
    w.qs = w.bytes;
    w.bytes += round_up(rows * 4, 256);
  }
  if (out_dtype == INF_DTYPE_I8 && !rows_whole(rows, n, k)) {
    w.y = w.bytes;
    w.bytes += round_up(rows * n * 4, 256);
  }
  return w;
}

// Rows of one turn (in_turns): their product, and their way into and out of 8 bits.
int linear_rows(const Linear8Args& call, const void* x, int x_dtype, int out_dtype, char* wsp, hipStream_t st) {
  Linear8Args a = call;
  const int64_t rows = a.rows, ld_x = a.ldq;
  const int n = a.n, k = a.k;
  const bool x8 = x_dtype == INF_DTYPE_I8;
  const Form form = form_of(rows, n, k, x_dtype, a.act, a.add != nullptr);
  const Workspace o = workspace_of(form, rows, n, k, x_dtype, out_dtype);
  const bool put_after = out_dtype == INF_DTYPE_I8 && !rows_whole(rows, n, k);
  if (put_after) {
    a.out = wsp + o.y;
    a.ldo = n;
  }
  const int product_dtype = put_after ? INF_DTYPE_F32 : out_dtype;
  int rc;
  if (form == Form::FEW) {
    rc = x8 ? launch_few_out<int8_t>(a, product_dtype, x, ld_x, st)
            : x_dtype == INF_DTYPE_BF16 ? launch_few_out<bf16>(a, product_dtype, x, ld_x, st)
                                        : launch_few_out<float>(a, product_dtype, x, ld_x, st);
  } else if (form == Form::WALK) {
    rc = x8 ? launch_rows_out<int8_t>(a, product_dtype, x, ld_x, st)
            : x_dtype == INF_DTYPE_BF16 ? launch_rows_out<bf16>(a, product_dtype, x, ld_x, st)
                                        : launch_rows_out<float>(a, product_dtype, x, ld_x, st);
  } else if (form == Form::LONG) {
    rc = x_dtype == INF_DTYPE_BF16 ? launch_long<bf16>(a, product_dtype, x, ld_x, st)
                                   : launch_long<float>(a, product_dtype, x, ld_x, st);
  } else {
    if (!x8) {
      a.q = (int8_t*)(wsp + o.q);
      a.ldq = round_up(k, q8::Q_ALIGN);
      a.qs = (float*)(wsp + o.qs);
      rc = launch_quantize_rows(x, x_dtype, rows, k, ld_x, (int8_t*)a.q, a.ldq, (float*)a.qs, st);
      if (rc != INF_OK) return rc;
    }
    rc = launch_linear8(a, product_dtype, st);
  }
  if (rc != INF_OK || !put_after) return rc;
  return launch_quantize_rows(a.out, INF_DTYPE_F32, rows, n, n, (int8_t*)call.out, call.ldo, call.os, st);
}

}  // namespace
}  // namespace inf

using namespace inf;

extern "C" {

int64_t inf_linear_int_workspace_bytes(int64_t rows, int n, int k, int x_dtype, int out_dtype) {
  if (rows < 0 || n < 1 || k < 1) return -1;
  const Form form = form_of(rows, n, k, x_dtype, 2, true);  // (the only one that needs none because of them is WALK)
  return workspace_of(form, rows, n, k, x_dtype, out_dtype).bytes;
}

int64_t inf_linear_int_call_workspace_bytes(int64_t rows, int n, int k, int x_dtype, int out_dtype, int act, int with_add) {
  if (rows < 0 || n < 1 || k < 1) return -1;
  return workspace_of(form_of(rows, n, k, x_dtype, act, with_add != 0), rows, n, k, x_dtype, out_dtype).bytes;
}

int inf_linear_int(int64_t rows, int n, int k, const void* x, int x_dtype, int64_t ld_x, const float* x_scale,
                   const int8_t* w, const float* w_scale, const float* bias, const float* add, int64_t ld_add, int act,
                   void* out, int out_dtype, int64_t ld_out, float* out_scale, void* workspace, inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && n >= 1 && k >= 1 && ld_x >= 0 && ld_out >= n, "linear_int: bad shape");
  INF_CHECK_ARG(rows < (int64_t)1 << 31, "linear_int: too many rows");
  INF_CHECK_ARG(k <= 1 << 17, "linear_int: k is at most 2^17 (the sums are held in 32 bits)");
  INF_CHECK_ARG(act >= 0 && act <= 2, "linear_int: act must be 0 (none), 1 (ReLU) or 2 (sigmoid)");
  INF_CHECK_ARG(x_dtype == INF_DTYPE_F32 || x_dtype == INF_DTYPE_BF16 || x_dtype == INF_DTYPE_I8,
                "linear_int: x must be fp32, bf16 or int8 rows");
  INF_CHECK_ARG(out_dtype == INF_DTYPE_F32 || out_dtype == INF_DTYPE_BF16 || out_dtype == INF_DTYPE_I8,
                "linear_int: out must be fp32, bf16 or int8 rows");
  if (rows == 0) return INF_OK;
  INF_CHECK_ARG(x != nullptr && w != nullptr && w_scale != nullptr && out != nullptr, "linear_int: null argument");
  INF_CHECK_ARG((uintptr_t)w % 16 == 0, "linear_int: the weight must be packed");
  INF_CHECK_ARG(add == nullptr || ld_add >= n, "linear_int: bad ld_add");
  const bool x8 = x_dtype == INF_DTYPE_I8, y8 = out_dtype == INF_DTYPE_I8;
  INF_CHECK_ARG(!x8 || (x_scale != nullptr && ld_x >= k && ld_x % q8::Q_ALIGN == 0 && (uintptr_t)x % 16 == 0),
                "linear_int: int8 rows need their scales and rows that start on 16 bytes");
  INF_CHECK_ARG(!y8 || (out_scale != nullptr && ld_out % q8::Q_ALIGN == 0 && (uintptr_t)out % 16 == 0),
                "linear_int: int8 output needs scales and rows that start on 16 bytes");
  const Workspace o = workspace_of(form_of(rows, n, k, x_dtype, act, add != nullptr), rows, n, k, x_dtype, out_dtype);
  INF_CHECK_ARG(o.bytes == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0),
                "linear_int: null or unaligned workspace");
  const int64_t x_size = x8 ? 1 : x_dtype == INF_DTYPE_BF16 ? 2 : 4, out_size = y8 ? 1 : out_dtype == INF_DTYPE_BF16 ? 2 : 4;
  return q8::in_turns(rows, n, [&](int64_t r, int64_t count) {
    const char* const from = (const char*)x + r * ld_x * x_size;
    const Linear8Args a{count, n, k, (const int8_t*)from, ld_x, x8 ? x_scale + r : nullptr, w, round_up(k, q8::W_ALIGN),
                        w_scale, bias, add != nullptr ? add + r * ld_add : nullptr, ld_add, act,
                        (char*)out + r * ld_out * out_size, ld_out, y8 ? out_scale + r : nullptr};
    return linear_rows(a, from, x_dtype, out_dtype, (char*)workspace, (hipStream_t)stream);
  });
}

}  // extern "C"
