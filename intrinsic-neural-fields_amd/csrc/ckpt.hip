// A linear layer whose inputs are kept in 8 bits until its backward (quant.hpp), for training:
//   forward   y = act(x W^T + bias + add)       from x as it is, in fp32
//             kept: q, s of x; one bit y > 0 (ReLU); y itself is the layer's output (sigmoid)
//   backward  dz = dy [y > 0] | dy y (1 - y) | dy
//             dx = dz W     dW = dz^T (s q)     db = sum_m dz
//
// Products of fp32 on the 16-bit matrix instructions.
//   x W^T and dz W: each row of either side is scaled by a power of two so that its largest
//   value lies in [2^14, 2^15), and a value is two fp16 pieces, hi = fp16(v), lo = fp16(v - hi), which
//   leave at most 2^-23 of it, or 2^-39 of the row's largest where that is more (a subnormal lo).
//   hi hi + hi lo + lo hi, summed in fp32; lo lo, at most 2^-22 of the product, is left out: a product
//   is within 2^-21, where fp32 has 2^-24, of values that are not 2^-16 of their row's largest.
//   (lo lo would be a fourth matrix instruction beside three.)  A bf16 x is one piece, exact down to
//   2^-31 of the row's largest: two products.  The powers of two leave the result exactly.
//   dW: q is exact in bf16 and dz s is three bf16 pieces, all 24 bits of it: three products, no
//   scale (a column of dz has no scale that a sum over its rows could be divided by): from dz s below 2^-110
//   on its low pieces are subnormal, and a term is off by less than 2^-133 |q|, 2^-126 at most.
// A row of x whose 8-bit scale is 0 (its largest value is below 2^-143) counts as a row of zeros.
// A value that is not finite makes NaN of the rows (and columns) that it enters.
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "mtile.hpp"

namespace inf {
namespace {

using namespace q8;
using namespace mt;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum { DZ_NONE = 0, DZ_RELU = 1, DZ_SIGMOID = 2 };  // act

// the power of two that takes a row of largest value a below 2^15
__device__ __forceinline__ int shift_of(float a) { return 15 - __builtin_amdgcn_frexp_expf(a); }
__device__ __forceinline__ float by_power(float v, int e) { return __builtin_amdgcn_ldexpf(v, e); }

// x = hi + lo, each rounded to nearest
__device__ __forceinline__ _Float16 piece_hi(float x) { return (_Float16)x; }
__device__ __forceinline__ _Float16 piece_lo(float x, _Float16 hi) { return (_Float16)(x - (float)hi); }

// ---- the weight's rows as fp16 pieces ---------------------------------------------------
// Row r of the product's side: V(r, k) = W[r sr + k sk], k < K, as the images that the instruction
// reads: for 16 rows and 32 k a KiB hi and a KiB lo, lane l's 16 bytes at 16 l (row l % 16, k = 8
// (l / 16) on).  Zero behind K up to a multiple of 64; rows behind the last hold anything.
__host__ __device__ __forceinline__ int blocks_of_32(int K) { return (K + 63) / 64 * 2; }

__device__ __forceinline__ void put_pieces(char* image, int r, const float* w, int64_t sk, int c, int K, int e) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c * 8 + i < K ? w[(c * 8 + i) * sk] : 0.f;
  f16x8 hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = by_power(v[i], e);
    hi[i] = piece_hi(x);
    lo[i] = piece_lo(x, hi[i]);
  }
  char* const to = image + ((int64_t)(r / 16) * blocks_of_32(K) + c / 4) * 2048 + (c % 4 * 16 + r % 16) * 16;
  *reinterpret_cast<f16x8*>(to) = hi;
  *reinterpret_cast<f16x8*>(to + 1024) = lo;
}

struct Weight {
  const float* W;
  int64_t sr, sk;
  int rows, K;
  char* out;
  int* shift;
};

// Workgroups of 256 threads; scratch: 16 words of LDS.
// sk is the short stride: a workgroup a row, its threads along k
__device__ __forceinline__ void split_row(int block, const Weight& a, unsigned* scratch) {
  const int r = block, tid = threadIdx.x;
  const float* const w = a.W + r * a.sr;
  unsigned t = 0;
#pragma unroll 4
  for (int k = tid; k < a.K; k += 256) t = max(t, abs_bits(w[k * a.sk]));
  t = row_max<64>(t);
  if (tid % 64 == 0) scratch[tid / 64] = t;
  __syncthreads();
  const int e = shift_of(__uint_as_float(max(max(scratch[0], scratch[1]), max(scratch[2], scratch[3]))));
  if (tid == 0) a.shift[r] = e;
  for (int c = tid; c < blocks_of_32(a.K) * 4; c += 256) put_pieces(a.out, r, w, a.sk, c, a.K, e);
}

// sr is the short stride: a workgroup 16 rows, 16 threads along them and 16 along k
__device__ __forceinline__ void split_columns(int block, const Weight& a, unsigned* scratch) {
  const int l = threadIdx.x % 16, g = threadIdx.x / 16, r = block * 16 + l;
  const float* const w = a.W + min(r, a.rows - 1) * a.sr;
  if (threadIdx.x < 16) scratch[threadIdx.x] = 0;
  __syncthreads();
  unsigned t = 0;
#pragma unroll 8
  for (int k = g; k < a.K; k += 16) t = max(t, abs_bits(w[k * a.sk]));
  t = max(t, (unsigned)__shfl_xor((int)t, 16));
  t = max(t, (unsigned)__shfl_xor((int)t, 32));
  if (threadIdx.x % 64 < 16) atomicMax(&scratch[l], t);  // a maximum: in any order the same
  __syncthreads();
  if (r >= a.rows) return;
  const int e = shift_of(__uint_as_float(scratch[l]));
  if (g == 0) a.shift[r] = e;
  for (int c = g; c < blocks_of_32(a.K) * 4; c += 16) put_pieces(a.out, r, w, a.sk, c, a.K, e);
}

bool along_k(const Weight& w) { return std::abs(w.sk) <= std::abs(w.sr); }
int split_blocks(const Weight& w) { return along_k(w) ? w.rows : (int)ceil_div(w.rows, 16); }

// One launch before the forward product: the weight's pieces, and the rows of x in 8 bits.
template <typename T, int LPR, int CH, int R, bool ALONG_K>
__global__ __launch_bounds__(256) void before_forward_kernel(Weight w, int nw, const T* __restrict__ x, int64_t rows,
                                                             int k, int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                                                             float* __restrict__ scale) {
  __shared__ unsigned scratch[16];
  if ((int)blockIdx.x < nw) {
    if constexpr (ALONG_K) split_row(blockIdx.x, w, scratch);
    else split_columns(blockIdx.x, w, scratch);
  } else {
    quantize_rows_block<T, LPR, CH, R>((int64_t)blockIdx.x - nw, x, rows, k, ldx, q, ldq, scale);
  }
}

template <bool ALONG_K>
__global__ __launch_bounds__(256) void split_kernel(Weight w) {
  __shared__ unsigned scratch[16];
  if constexpr (ALONG_K) split_row(blockIdx.x, w, scratch);
  else split_columns(blockIdx.x, w, scratch);
}

// ---- dz -------------------------------------------------------------------------------
struct Dz {
  const float* dy;
  int64_t lddy;
  const float* y;
  int64_t ldy;
  const uint32_t* mask;
  int words;  // of the mask, a row
};

template <int ACT>
__device__ __forceinline__ float dz_at(const Dz& d, int64_t m, int c) {
  const float g = d.dy[m * d.lddy + c];
  if (ACT == DZ_RELU) return (d.mask[m * d.words + c / 32] >> (c % 32)) & 1 ? g : 0.f;
  if (ACT == DZ_SIGMOID) {
    const float y = d.y[m * d.ldy + c];
    return g * (y * (1.f - y));
  }
  return g;
}

// One launch before the backward products: the pieces of the weight's columns, and each row's
// shift of dz, LPR lanes a row, four values a turn.
template <int ACT, int LPR, bool ALONG_K>
__global__ __launch_bounds__(256) void before_dx_kernel(Weight w, int nw, Dz d, int64_t rows, int n,
                                                        int* __restrict__ shift) {
  __shared__ unsigned scratch[16];
  if ((int)blockIdx.x < nw) {
    if constexpr (ALONG_K) split_row(blockIdx.x, w, scratch);
    else split_columns(blockIdx.x, w, scratch);
    return;
  }
  const int64_t m = ((int64_t)blockIdx.x - nw) * (256 / LPR) + threadIdx.x / LPR;
  if (m >= rows) return;
  unsigned a = 0;
#pragma unroll 2
  for (int c = threadIdx.x % LPR * 4; c < n; c += LPR * 4) {
    if (c + 4 <= n) {
      const f32x4u g = *reinterpret_cast<const f32x4u*>(d.dy + m * d.lddy + c);
      f32x4u y = {};
      uint32_t bits = 0;
      if (ACT == DZ_SIGMOID) y = *reinterpret_cast<const f32x4u*>(d.y + m * d.ldy + c);
      if (ACT == DZ_RELU) bits = d.mask[m * d.words + c / 32] >> (c % 32);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = g[e];
        if (ACT == DZ_SIGMOID) v *= y[e] * (1.f - y[e]);
        if (ACT == DZ_RELU) v = (bits >> e) & 1 ? v : 0.f;
        a = max(a, abs_bits(v));
      }
    } else {
      for (int e = c; e < n; ++e) a = max(a, abs_bits(dz_at<ACT>(d, m, e)));
    }
  }
  a = row_max<LPR>(a);
  if (threadIdx.x % LPR == 0) shift[m] = shift_of(__uint_as_float(a));
}

// ---- x W^T and dz W -----------------------------------------------------------------------
// out(m, c) = sum_k side(m, k) V(c, k): BM rows by BN columns a workgroup, WM x WN waves,
// v_mfma_f32_16x16x32_f16 with V as its first operand (a lane holds four neighbouring
// columns of one row).  Per turn 32 k.  LDS: two stages, V's images as they are, filled straight from
// memory one turn ahead, and 128-byte rows of the side (64 hi, 64 lo).  The rows of x or dz are
// read in whole lines into registers a turn ahead and split on their way to LDS, each value once.
struct SideArgs {
  int64_t rows;
  int cols, K;          // output columns; length of the sums
  const void* x;        // forward: x
  int64_t ldx;
  const float* scale;   // forward: the rows' 8-bit scales (their largest value / 127)
  const int* shift;     // dx: the rows' shifts
  Dz dz;
  const char* V;        // pieces of the weight's rows
  const int* vshift;
  const float* bias;    // forward
  const float* add;
  int64_t ldadd;
  int act;
  void* out;
  int64_t ldo;
  uint32_t* mask;
};

// add, activation of a forward result's four columns
__device__ __forceinline__ void finish_forward(const SideArgs& a, int64_t m, int n, f32x4& z) {
  if (a.add != nullptr && m < a.rows) {
    const float* const from = a.add + m * a.ldadd + n;
    if (n + 4 <= a.cols) {
      const f32x4u v = *reinterpret_cast<const f32x4u*>(from);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] += v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.cols) z[e] += from[e];
    }
  }
  if (a.act == DZ_RELU) {
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = activate(z[e], DZ_RELU);
  } else if (a.act == DZ_SIGMOID) {
    // one copy of its code for the four: with 16 of these a thread, 64 took the 65,536 x 256 x 256
    // product from 49 to 58 us, ReLU or not
#pragma unroll 1
    for (int e = 0; e < 4; ++e) z = f32x4{z[1], z[2], z[3], activate(z[0], DZ_SIGMOID)};
  }
}

// 16 bits of a row's mask: this lane's four, joined with those of the other lane groups
__device__ __forceinline__ uint32_t mask_bits(const f32x4& z, int n, int cols, int g4) {
  uint32_t b = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) b |= (uint32_t)(z[e] > 0.f && n + e < cols) << (4 * g4 + e);
  b |= (uint32_t)__shfl_xor((int)b, 16);
  return b | (uint32_t)__shfl_xor((int)b, 32);
}

// Rows that all start on 16 bytes (`direct`) are stored from the registers.  Others (k = 1023) go
// through the wave's own piece of LDS, so that a store is one run of a row: 16-byte stores across
// lines took 224 us where these took 164 (65,536 x 1023 x 256, dx, in 256 x 256 tiles).
template <typename T>
__device__ __forceinline__ void store_four(const SideArgs& a, int64_t m, int n, const f32x4& z) {
  if (m >= a.rows) return;
  T* const to = reinterpret_cast<T*>(a.out) + m * a.ldo + n;
  if (n + 4 <= a.cols) {
    typedef T V4 __attribute__((ext_vector_type(4)));
    V4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = from_f32<T>(z[e]);
    *reinterpret_cast<V4*>(to) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.cols) to[e] = from_f32<T>(z[e]);
  }
}
template <typename T, int ROWS, int COLS>
__device__ __forceinline__ void store_runs(const SideArgs& a, const char* mine, int stride, int64_t m0, int n0, int lane) {
  own_lds_order();
  const int c = lane % COLS, n = n0 + c;
#pragma unroll
  for (int r = 0; r < ROWS; r += 64 / COLS) {
    const int row = r + lane / COLS;
    const float v = *reinterpret_cast<const float*>(mine + row * stride + c * 4);
    if (m0 + row < a.rows && n < a.cols) reinterpret_cast<T*>(a.out)[(m0 + row) * a.ldo + n] = from_f32<T>(v);
  }
  own_lds_order();
}

template <int BM, int BN, int WM, int WN>
struct ST {
  static constexpr int THREADS = 64 * WM * WN;
  static constexpr int WROWS = BM / WM, WCOLS = BN / WN, TI = WROWS / 16, TJ = WCOLS / 16;
  static constexpr int V_STAGE = BN * 128, STAGE = V_STAGE + BM * 128, LDS = 2 * STAGE;
  static constexpr int LOADS = V_STAGE / (THREADS * 16);
  static_assert(V_STAGE % (THREADS * 16) == 0 && LDS <= 160 * 1024, "tile");
  static_assert(WCOLS % 32 == 0, "a wave holds whole words of the mask");
};

// MODE 0: forward, the side is X rows; 1: dx, the side is dz (ACT)
template <int MODE, int ACT, typename X, typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void split_tile_kernel(SideArgs a, int tiles_n, int nblocks) {
  using P = ST<BM, BN, WM, WN>;
  constexpr int TI = P::TI, TJ = P::TJ;
  constexpr bool LO = sizeof(X) == 4;         // a bf16 value is one piece
  constexpr int V = 16 / sizeof(X);           // values of a 16-byte load
  constexpr int LANES = 32 / V;               // lanes that load a row's 32 values
  constexpr int PASS = BM * LANES / P::THREADS;
  constexpr bool MASK = MODE == 1 && ACT == DZ_RELU, WITH_Y = MODE == 1 && ACT == DZ_SIGMOID;
  constexpr int ROW_LOADS = PASS * (MASK || WITH_Y ? 2 : 1);  // at least so many loads a turn
  static_assert(PASS * P::THREADS == BM * LANES, "tile");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int bid = xcd_order((int)blockIdx.x, nblocks);
  const int64_t m0 = (int64_t)(bid / tiles_n) * BM;
  const int n0 = (bid % tiles_n) * BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave / WN, wc = wave % WN, r16 = lane & 15, g4 = lane >> 4;
  const int turns = (a.K + 31) / 32;

  // Offsets of 32 bits from uniform bases: with 128 registers a lane each address counts.  Rows of V
  // behind the last are in the workspace, whatever they hold: their columns are not stored.
  const int blocks = blocks_of_32(a.K);
  auto issue = [&](int t, int stage) {
    char* st = smem + (stage & 1) * P::STAGE;
#pragma unroll
    for (int i = 0; i < P::LOADS; ++i) {
      const int kib = wave + WM * WN * i;  // 16 rows of V, hi or lo
      const char* const V = a.V + ((int64_t)(n0 / 16 + kib / 2) * blocks + t) * 2048 + kib % 2 * 1024;
      const char* from = V + pinned(lane * 16u);
      __builtin_amdgcn_global_load_lds(from, (lds_void*)(st + kib * 1024), 16, 0, 0);
    }
  };
  // this thread's rows (PASS of them) and its values of each turn: k = V (tid % LANES) + (0..V)
  const int kc = (tid % LANES) * V;
  auto row_of = [&](int p) { return tid / LANES + p * (P::THREADS / LANES); };
  const X* const side = MODE == 0 ? (const X*)a.x + m0 * a.ldx : (const X*)a.dz.dy + m0 * a.dz.lddy;
  const float* const ys = WITH_Y ? a.dz.y + m0 * a.dz.ldy : nullptr;
  const uint32_t* const words = MASK ? a.dz.mask + m0 * a.dz.words : nullptr;
  int shift[PASS], off[PASS], yoff[WITH_Y ? PASS : 1], woff[MASK ? PASS : 1];
#pragma unroll
  for (int p = 0; p < PASS; ++p) {
    const int r = (int)min((int64_t)row_of(p), a.rows - 1 - m0);
    shift[p] = MODE == 0 ? shift_of(a.scale[m0 + r] * 127.f) : a.shift[m0 + r];
    off[p] = r * (int)(MODE == 0 ? a.ldx : a.dz.lddy);
    if constexpr (WITH_Y) yoff[p] = r * (int)a.dz.ldy;
    if constexpr (MASK) woff[p] = r * a.dz.words;
  }
  struct Raw {
    X v[PASS][V];
    float y[WITH_Y ? PASS : 1][4];
    uint32_t w[MASK ? PASS : 1];
  };
  typedef X XV __attribute__((ext_vector_type(V), aligned(sizeof(X))));
  // The last 32 k, which may be fewer, are the first turn: the loop has whole ones alone.
  auto block_of = [&](int t) { return t == 0 ? turns - 1 : min(t, turns - 1) - 1; };
  // Nothing here uses what it loads: the waits belong to put(), a turn later.
  auto fetch = [&](Raw& r, int block) {
    const int k = block * 32 + kc;
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      const XV x = *reinterpret_cast<const XV*>((const char*)side + pinned((unsigned)(off[p] + k) * sizeof(X)));
#pragma unroll
      for (int e = 0; e < V; ++e) r.v[p][e] = x[e];
      if constexpr (WITH_Y) {
        const f32x4u y = *reinterpret_cast<const f32x4u*>((const char*)ys + pinned((unsigned)(yoff[p] + k) * 4u));
#pragma unroll
        for (int e = 0; e < 4; ++e) r.y[p][e] = y[e];
      }
      if constexpr (MASK)
        r.w[p] = *reinterpret_cast<const uint32_t*>((const char*)words + pinned((unsigned)(woff[p] + block) * 4u));
    }
  };
  auto fetch_last = [&](Raw& r) {
    const int k = (turns - 1) * 32 + kc;
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int ke = min(k + e, a.K - 1);
        r.v[p][e] = k + e < a.K ? side[off[p] + ke] : (X)0.f;
        if constexpr (WITH_Y) r.y[p][e] = ys[yoff[p] + ke];
      }
      if constexpr (MASK) r.w[p] = words[woff[p] + turns - 1];
    }
  };
  auto put = [&](const Raw& r, int t) {
    char* st = smem + (t & 1) * P::STAGE + P::V_STAGE;
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      typedef _Float16 Piece __attribute__((ext_vector_type(V)));
      Piece hi, lo;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float v = to_f32(r.v[p][e]);
        if constexpr (WITH_Y) v *= r.y[p][e] * (1.f - r.y[p][e]);
        if constexpr (MASK) v = (r.w[p] >> (kc + e)) & 1 ? v : 0.f;
        const float x = by_power(v, shift[p]);
        hi[e] = piece_hi(x);
        if (LO) lo[e] = piece_lo(x, hi[e]);
      }
      const int row = row_of(p);
      *reinterpret_cast<Piece*>(st + chunk_at(row, kc / 8) + (kc % 8) * 2) = hi;
      if (LO) *reinterpret_cast<Piece*>(st + chunk_at(row, 4 + kc / 8) + (kc % 8) * 2) = lo;
    }
  };

  f32x4 acc[TJ][TI];
#pragma unroll
  for (int j = 0; j < TJ; ++j)
#pragma unroll
    for (int i = 0; i < TI; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Two passes over the products, so that one of V's pieces at a time is held: hi of V by both
  // pieces of the rows, then lo of V by hi of the rows.
  auto turn_products = [&](int t) {
    const char* const vs = smem + (t & 1) * P::STAGE;
    const char* const xs = vs + P::V_STAGE;
    f16x8 w[TJ];
#pragma unroll
    for (int j = 0; j < TJ; ++j) w[j] = *reinterpret_cast<const f16x8*>(vs + (wc * TJ + j) * 2048 + lane * 16);
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int r = wr * P::WROWS + 16 * i + r16;
      if (LO) {
        const f16x8 xl = *reinterpret_cast<const f16x8*>(xs + chunk_at(r, 4 + g4));
#pragma unroll
        for (int j = 0; j < TJ; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], xl, acc[j][i], 0, 0, 0);
      }
      const f16x8 xh = *reinterpret_cast<const f16x8*>(xs + chunk_at(r, g4));
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], xh, acc[j][i], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < TJ; ++j)
      w[j] = *reinterpret_cast<const f16x8*>(vs + (wc * TJ + j) * 2048 + 1024 + lane * 16);
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const f16x8 xh = *reinterpret_cast<const f16x8*>(xs + chunk_at(wr * P::WROWS + 16 * i + r16, g4));
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[j], xh, acc[j][i], 0, 0, 0);
    }
  };
  Raw raw;
  issue(block_of(0), 0);
  if (a.K % 32 == 0) fetch(raw, turns - 1);
  else fetch_last(raw);
  put(raw, 0);
  if (turns > 1) fetch(raw, block_of(1));
  wait_barrier<0>();
#pragma unroll 1
  for (int t = 0; t + 1 < turns; ++t) {
    issue(block_of(t + 1), t + 1);
    // the parts stay apart: interleaved they need more registers than there are
    __builtin_amdgcn_sched_barrier(0);
    turn_products(t);
    __builtin_amdgcn_sched_barrier(0);
    put(raw, t + 1);
    __builtin_amdgcn_sched_barrier(0);
    fetch(raw, block_of(t + 2));  // past the last: the last again, so that the waits can be counted
    wait_barrier<ROW_LOADS>();    // V's loads are older than the rows'
  }
  turn_products(turns - 1);
  wait_barrier<0>();

  // lane: row wr WROWS + 16 i + r16, columns wc WCOLS + 16 j + 4 g4 + (0..3)
  int sm[TI];
  // NaN for a bf16 row that is not finite, else 0: such a value has no low piece whose inf - inf would make NaN
  // of all that it meets, and an infinity of its own sign, or after a ReLU a zero, would come out
  float bad[LO ? 1 : TI];
#pragma unroll
  for (int i = 0; i < TI; ++i) {
    const int64_t m = min(m0 + wr * P::WROWS + 16 * i + r16, a.rows - 1);
    sm[i] = MODE == 0 ? shift_of(a.scale[m] * 127.f) : a.shift[m];
    if constexpr (!LO) bad[i] = a.scale[m] * 0.f;
  }
  int sn[TJ][4];
  float bias[TJ][4];
#pragma unroll
  for (int j = 0; j < TJ; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = min(n0 + wc * P::WCOLS + 16 * j + 4 * g4 + e, a.cols - 1);
      sn[j][e] = a.vshift[n];
      bias[j][e] = MODE == 0 && a.bias != nullptr ? a.bias[n] : 0.f;
    }
  const bool direct = ((uintptr_t)a.out | (uintptr_t)(a.ldo * sizeof(T))) % 16 == 0;
  constexpr int RS = P::WCOLS * 4 + 16;
  static_assert(WM * WN * 16 * RS <= P::LDS, "the waves' pieces fit the stages");
  char* const mine = smem + wave * 16 * RS;
#pragma unroll
  for (int i = 0; i < TI; ++i) {
    const int64_t m = m0 + wr * P::WROWS + 16 * i + r16;
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int n = n0 + wc * P::WCOLS + 16 * j + 4 * g4;
      f32x4 z;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z[e] = by_power(acc[j][i][e], -(sm[i] + sn[j][e])) + bias[j][e];
        if constexpr (!LO) z[e] += bad[i];
      }
      if (MODE == 0) finish_forward(a, m, n, z);
      if (direct) store_four<T>(a, m, n, z);
      else *reinterpret_cast<f32x4*>(mine + r16 * RS + (16 * j + 4 * g4) * 4) = z;
      if (MODE == 0 && a.mask != nullptr) {
        const uint32_t b = mask_bits(z, n, a.cols, g4);
        if (j % 2 == 0) bits = b;
        else if (g4 == 0 && m < a.rows && n - 16 < a.cols)
          a.mask[m * ((a.cols + 31) / 32) + (n - 16) / 32] = bits | b << 16;
      }
    }
    if (!direct)
      store_runs<T, 16, P::WCOLS>(a, mine, RS, m0 + wr * P::WROWS + 16 * i, n0 + wc * P::WCOLS, lane);
  }
}

// ---- dx of short sums, many rows and columns -------------------------------------------------
// Sums of up to 256.  A workgroup takes 64 whole rows of dz: their largest values and their pieces
// come from registers that hold them once, and the pieces stay in LDS.  Then each of its 4 waves
// makes 64 columns of all 64 rows at a time, with V's images straight from L2 into its registers a
// step ahead: no barrier, nothing split twice, no launch before it that reads dy as well.  Two
// workgroups a CU: one's rows come in beside the other's products (one of 128 rows and 8 waves,
// which reads V half as often, 142 us where these take 138: 65,536 x 1024 x 256).
constexpr int PB = 64, PW = 4, PJ = 4, PC = 16 * PJ, P_BLOCKS = 8;
constexpr int P_ROW = PC * 4 + 16;  // a row of a wave's piece for results: 8 rows
constexpr int panel_lds(int blocks) { return blocks * PB * 128 + PB * 4 + PW * 8 * P_ROW; }
static_assert(panel_lds(P_BLOCKS) <= 160 * 1024, "LDS");

template <int ACT, typename T>
__global__ __launch_bounds__(64 * PW, 2) void panel_kernel(SideArgs a) {
  constexpr int LANES = 8, ROWS = 64 * PW / LANES, PASS = PB / ROWS;
  constexpr bool MASK = ACT == DZ_RELU, WITH_Y = ACT == DZ_SIGMOID;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.x * PB;
  const int blocks = blocks_of_32(a.K);
  int* const shifts = reinterpret_cast<int*>(smem + blocks * PB * 128);
  char* const mine = smem + blocks * PB * 128 + PB * 4 + wave * 8 * P_ROW;

  // the rows: LANES lanes each, four values of each block of 32
  const int kc = tid % LANES * 4;
#pragma unroll
  for (int p = 0; p < PASS; ++p) {
    const int r = tid / LANES + p * ROWS;
    const int64_t m = min(m0 + r, a.rows - 1);
    const float* const row = a.dz.dy + m * a.dz.lddy;
    f32x4 v[P_BLOCKS], y[WITH_Y ? P_BLOCKS : 1];
    uint32_t w[MASK ? P_BLOCKS : 1];
    auto load = [&](f32x4& to, const float* from, int k) {
      if (k + 4 <= a.K) {
        to = *reinterpret_cast<const f32x4u*>(from + k);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = k + e < a.K ? from[k + e] : 0.f;
      }
    };
#pragma unroll
    for (int b = 0; b < P_BLOCKS; ++b)
      if (b < blocks) {
        load(v[b], row, b * 32 + kc);
        if constexpr (WITH_Y) load(y[b], a.dz.y + m * a.dz.ldy, b * 32 + kc);
        if constexpr (MASK) w[b] = a.dz.mask[m * a.dz.words + min(b, a.dz.words - 1)];
      }
    unsigned top = 0;
#pragma unroll
    for (int b = 0; b < P_BLOCKS; ++b)
      if (b < blocks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (WITH_Y) v[b][e] *= y[b][e] * (1.f - y[b][e]);
          if constexpr (MASK) v[b][e] = (w[b] >> (kc + e)) & 1 ? v[b][e] : 0.f;
          top = max(top, abs_bits(v[b][e]));
        }
    top = row_max<LANES>(top);
    const int e2 = shift_of(__uint_as_float(top));
    if (tid % LANES == 0) shifts[r] = e2;
#pragma unroll
    for (int b = 0; b < P_BLOCKS; ++b)
      if (b < blocks) {
        typedef _Float16 Piece __attribute__((ext_vector_type(4)));
        Piece hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = by_power(v[b][e], e2);
          hi[e] = piece_hi(x);
          lo[e] = piece_lo(x, hi[e]);
        }
        char* const st = smem + b * PB * 128;
        *reinterpret_cast<Piece*>(st + chunk_at(r, kc / 8) + (kc % 8) * 2) = hi;
        *reinterpret_cast<Piece*>(st + chunk_at(r, 4 + kc / 8) + (kc % 8) * 2) = lo;
      }
  }
  __syncthreads();

  const int tiles = (a.cols + PC - 1) / PC;
  struct Images {
    f16x8 hi[PJ], lo[PJ];
  } va, vb;
  auto load_v = [&](Images& f, int tile, int b) {
    const char* const from = a.V + ((int64_t)tile * PJ * blocks + b) * 2048;
#pragma unroll
    for (int j = 0; j < PJ; ++j) {
      f.hi[j] = *reinterpret_cast<const f16x8*>(from + j * blocks * 2048 + pinned(lane * 16u));
      f.lo[j] = *reinterpret_cast<const f16x8*>(from + j * blocks * 2048 + 1024 + pinned(lane * 16u));
    }
  };
  const bool direct = ((uintptr_t)a.out | (uintptr_t)(a.ldo * sizeof(T))) % 16 == 0;
  int tile = wave;
  if (tile < tiles) load_v(va, tile, 0);
  for (; tile < tiles; tile += PW) {
    f32x4 acc[PJ][PB / 16];
#pragma unroll
    for (int j = 0; j < PJ; ++j)
#pragma unroll
      for (int i = 0; i < PB / 16; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto products = [&](const Images& f, int b) {
      const char* const st = smem + b * PB * 128;
#pragma unroll
      for (int i = 0; i < PB / 16; ++i) {
        const f16x8 xh = *reinterpret_cast<const f16x8*>(st + chunk_at(16 * i + r16, g4));
        const f16x8 xl = *reinterpret_cast<const f16x8*>(st + chunk_at(16 * i + r16, 4 + g4));
#pragma unroll
        for (int j = 0; j < PJ; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.lo[j], xh, acc[j][i], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < PJ; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.hi[j], xl, acc[j][i], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < PJ; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.hi[j], xh, acc[j][i], 0, 0, 0);
      }
    };
#pragma unroll 1
    for (int b = 0; b < blocks; b += 2) {
      load_v(vb, tile, b + 1);
      __builtin_amdgcn_sched_barrier(0);
      products(va, b);
      __builtin_amdgcn_sched_barrier(0);
      const bool last = b + 2 == blocks;
      load_v(va, last ? min(tile + PW, tiles - 1) : tile, last ? 0 : b + 2);
      __builtin_amdgcn_sched_barrier(0);
      products(vb, b + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    // lane: row 16 i + r16, columns 16 j + 4 g4 + (0..3) of the tile's
    const int n0 = tile * PC;
    int sn[PJ][4];
#pragma unroll
    for (int j = 0; j < PJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sn[j][e] = a.vshift[min(n0 + 16 * j + 4 * g4 + e, a.cols - 1)];
#pragma unroll
    for (int i = 0; i < PB / 16; ++i) {
      const int sm = shifts[16 * i + r16];
      f32x4 z[PJ];
#pragma unroll
      for (int j = 0; j < PJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[j][e] = by_power(acc[j][i][e], -(sm + sn[j][e]));
      if (direct) {
#pragma unroll
        for (int j = 0; j < PJ; ++j) store_four<T>(a, m0 + 16 * i + r16, n0 + 16 * j + 4 * g4, z[j]);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (r16 / 8 == h)
#pragma unroll
            for (int j = 0; j < PJ; ++j)
              *reinterpret_cast<f32x4*>(mine + r16 % 8 * P_ROW + (16 * j + 4 * g4) * 4) = z[j];
          store_runs<T, 8, PC>(a, mine, P_ROW, m0 + 16 * i + 8 * h, n0, lane);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

template <int ACT, typename T>
int launch_panel(const SideArgs& a, hipStream_t stream) {
  const auto kernel = panel_kernel<ACT, T>;
  static LdsLimit lds;
  const int allowed = lds.raise((const void*)kernel, panel_lds(P_BLOCKS));
  if (allowed != INF_OK) return allowed;
  kernel<<<(unsigned)ceil_div(a.rows, PB), 64 * PW, panel_lds(blocks_of_32(a.K)), stream>>>(a);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

// Rows for two workgroups a CU, columns for each wave, and sums that the fill is worth.  With the
// launch before it, here and in tiles, us: 65,536 x 1024 x 256 133 and 169 (x 128 95 and 112, x 32 66
// and 62), 65,536 x 256 x 256 56 and 56; 32,768 x 1024 x 256 68 and 77, 16,384 45 and 45.
bool takes_panel(int64_t rows, int K, int cols) {
  return rows >= 32768 && K > 64 && K <= 32 * P_BLOCKS && cols >= PW * PC;
}

// ---- dW and db ------------------------------------------------------------------------
// dW(n, k) = sum_m dz(m, n) s_m q(m, k): 128 n by 256 k a workgroup, 4 x 4 waves, 32 rows m a
// turn, v_mfma_f32_16x16x32_bf16 with q as its first operand (a lane holds four neighbouring
// k of one n).  Both sides are turned on the way to LDS: a thread loads one column (four of q) of
// 4 (2) rows, neighbouring threads neighbouring columns.  Bound by these conversions next to
// the products: 16 waves, so that one's run beside another's.  The rows are divided over `splits`
// workgroups a tile, whose sums add_slabs_kernel adds in order: no atomics.
constexpr int DW_N = 128, DW_K = 256, DW_THREADS = 1024;
constexpr int DW_STAGE = DW_K * 64 + 3 * DW_N * 64;  // q rows, then the pieces of dz: hi, mid, lo
constexpr int DW_LDS = 2 * DW_STAGE;

// Chunk c (16 bytes) of a 64-byte LDS row.  A 16-byte read serves 16 lanes at a time, rows 0-3 and
// 12-15 of one c with rows 4-11 of the next: the last term but one sends them to 16 places.  The
// turn of four rows and the last term do the same for writes to every fourth row.
__device__ __forceinline__ int at64(int r, int c) {
  return (r >> 2) * 256 + (((r + (r >> 2)) & 3) << 6) + (((c ^ -(r >> 2) ^ (r >> 4)) & 3) << 4);
}
__device__ __forceinline__ uint32_t top_halves(float a, float b) {  // bf16 of a (low) and b, both exact
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
}

struct DwArgs {
  int64_t rows;
  int n, k;
  Dz dz;
  const int8_t* q;
  int64_t ldq;
  const float* s;
  int tiles_k, tiles, splits;
  int64_t rows_a_split;  // a multiple of 32
  float* out;            // [splits][n][ldw]
  int64_t ldw;
  float* db;             // [splits][n], or null
};

template <int ACT>
__global__ __launch_bounds__(DW_THREADS) void dw_tile_kernel(DwArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // the tiles of one split next to each other on one XCD: they read the same rows
  const int bid = xcd_order((int)blockIdx.x, a.tiles * a.splits);
  const int split = bid / a.tiles, tile = bid % a.tiles;
  const int n0 = tile / a.tiles_k * DW_N, k0 = tile % a.tiles_k * DW_K;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave / 4, wk = wave % 4, r16 = lane & 15, g4 = lane >> 4;  // 32 n by 64 k a wave
  const int64_t mb = split * a.rows_a_split, me = min(mb + a.rows_a_split, a.rows);
  const int turns = (int)((me - mb + 31) / 32);

  const int zc = tid & 127, zg = tid >> 7;  // dz: column, group of 4 rows
  const int n = n0 + zc, nc = min(n, a.n - 1);
  const bool in_n = n < a.n, with_db = a.db != nullptr && k0 == 0;
  const int qc = tid & 63, qg = tid >> 6;   // q: 4 columns, group of 2 rows
  const int kq = (int)min((int64_t)(k0 + 4 * qc), a.ldq - 4);
  float z[4], y[ACT == DZ_SIGMOID ? 4 : 1], s[4];
  uint32_t w[ACT == DZ_RELU ? 4 : 1];
  float dbsum = 0.f;
  int q[2];
  // The rows of a split's last turn, which may be fewer, are the first: the loop has whole turns
  // alone, whose addresses are a uniform base each and one offset of 32 bits.
  const auto block_of = [&](int t) { return t == 0 ? turns - 1 : t - 1; };
  const unsigned zoff = (unsigned)(zg * 4) * (unsigned)a.dz.lddy + nc, yoff = (unsigned)(zg * 4) * (unsigned)a.dz.ldy + nc;
  const unsigned woff = (unsigned)(zg * 4 * a.dz.words + nc / 32), qoff = (unsigned)(qg * 2) * (unsigned)a.ldq + kq;
  auto fetch = [&](int block) {
    const int64_t m = mb + block * 32;
    const float* const dy = a.dz.dy + m * a.dz.lddy;
    const f32x4u s0 = *reinterpret_cast<const f32x4u*>(a.s + m + zg * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      z[e] = (dy + e * a.dz.lddy)[pinned(zoff)];
      s[e] = s0[e];
      if constexpr (ACT == DZ_RELU) w[e] = (a.dz.mask + (m + e) * a.dz.words)[pinned(woff)];
      if constexpr (ACT == DZ_SIGMOID) y[e] = (a.dz.y + (m + e) * a.dz.ldy)[pinned(yoff)];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) q[e] = *reinterpret_cast<const int*>(a.q + (m + e) * a.ldq + pinned(qoff));
  };
  auto fetch_last = [&]() {  // rows past the end: the last row, times zero
    const int64_t mz = mb + (turns - 1) * 32 + zg * 4, mq = mb + (turns - 1) * 32 + qg * 2;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t m = min(mz + e, me - 1);
      z[e] = mz + e < me ? a.dz.dy[m * a.dz.lddy + nc] : 0.f;
      s[e] = mz + e < me ? a.s[m] : 0.f;
      if constexpr (ACT == DZ_RELU) w[e] = a.dz.mask[m * a.dz.words + nc / 32];
      if constexpr (ACT == DZ_SIGMOID) y[e] = mz + e < me ? a.dz.y[m * a.dz.ldy + nc] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) q[e] = *reinterpret_cast<const int*>(a.q + min(mq + e, me - 1) * a.ldq + kq);
  };
  auto put = [&](int t) {
    char* st = smem + (t & 1) * DW_STAGE;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (ACT == DZ_RELU)  // the mask's bit as all bits
        z[e] = __uint_as_float(__float_as_uint(z[e]) & (unsigned)__builtin_amdgcn_sbfe((int)w[e], nc & 31, 1));
      if constexpr (ACT == DZ_SIGMOID) z[e] *= y[e] * (1.f - y[e]);
    }
    if (with_db)
#pragma unroll
      for (int e = 0; e < 4; ++e) dbsum += z[e];
    u32x2 piece[3];
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      float v[2] = {z[e] * s[e], z[e + 1] * s[e + 1]};
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        piece[p][e / 2] = top_halves(v[0], v[1]);
        if (p < 2)
#pragma unroll
          for (int u = 0; u < 2; ++u) v[u] -= __uint_as_float(__float_as_uint(v[u]) & 0xffff0000u);
      }
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)
      *reinterpret_cast<u32x2*>(st + DW_K * 64 + p * DW_N * 64 + at64(zc, zg / 2) + (zg & 1) * 8) = piece[p];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<uint32_t*>(st + at64(4 * qc + c, qg / 4) + (qg & 3) * 4) =
          top_halves((float)(int8_t)(q[0] >> (8 * c)), (float)(int8_t)(q[1] >> (8 * c)));
  };
  f32x4 acc[4][2];  // [k tile][n tile]
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto turn_products = [&](int t) {
    const char* st = smem + (t & 1) * DW_STAGE;
    bf16x8 qf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) qf[j] = *reinterpret_cast<const bf16x8*>(st + at64(wk * 64 + 16 * j + r16, g4));
#pragma unroll
    for (int p = 2; p >= 0; --p) {
      bf16x8 zf[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        zf[i] = *reinterpret_cast<const bf16x8*>(st + DW_K * 64 + p * DW_N * 64 + at64(wn * 32 + 16 * i + r16, g4));
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[j], zf[i], acc[j][i], 0, 0, 0);
    }
  };
  if (turns > 0) {
    fetch_last();
    put(0);
    if (turns > 1) fetch(block_of(1));
    wait_all_barrier();
#pragma unroll 1
    for (int t = 0; t + 1 < turns; ++t) {
      turn_products(t);
      put(t + 1);
      if (t + 2 < turns) fetch(block_of(t + 2));
      wait_lds_barrier();
    }
    turn_products(turns - 1);
    wait_all_barrier();
  }
  float* const out = a.out + (int64_t)split * a.n * a.ldw;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = n0 + wn * 32 + 16 * i + r16;
    if (c >= a.n) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + wk * 64 + 16 * j + 4 * g4;
      float* const to = out + c * a.ldw + k;
      if (k + 4 <= a.k) {
        f32x4u o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = acc[j][i][e];
        *reinterpret_cast<f32x4u*>(to) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < a.k) to[e] = acc[j][i][e];
      }
    }
  }
  if (a.db != nullptr && k0 == 0) {
    float* const part = reinterpret_cast<float*>(smem);
    part[zg * DW_N + zc] = dbsum;
    __syncthreads();
    if (tid < DW_N && in_n)
    {
      float v = 0.f;
#pragma unroll
      for (int g = 0; g < 8; ++g) v += part[g * DW_N + zc];
      a.db[(int64_t)split * a.n + n] = v;
    }
  }
}

// dW and db from the splits' sums: 32 outputs a workgroup, eight threads each an eighth of the
// splits in order, then the eight in order.
__global__ __launch_bounds__(256) void add_slabs_kernel(const float* __restrict__ slabs, int64_t count, int k,
                                                        int splits, float* __restrict__ dW, int64_t lddw,
                                                        const float* __restrict__ dbs, int n, float* __restrict__ db) {
  __shared__ float part[8][32];
  const int l = threadIdx.x % 32, g = threadIdx.x / 32;
  const int64_t i = (int64_t)blockIdx.x * 32 + l;
  const bool is_w = i < count, is_b = !is_w && i - count < n && db != nullptr;
  const int s0 = splits * g / 8, s1 = splits * (g + 1) / 8;
  float v = 0.f;
  if (is_w)
#pragma unroll 8
    for (int s = s0; s < s1; ++s) v += slabs[s * count + i];
  if (is_b)
    for (int s = s0; s < s1; ++s) v += dbs[(int64_t)s * n + (i - count)];
  part[g][l] = v;
  __syncthreads();
  if (g != 0 || !(is_w || is_b)) return;
#pragma unroll
  for (int h = 1; h < 8; ++h) v += part[h][l];
  if (is_w) dW[i / k * lddw + i % k] = v;
  else db[i - count] = v;
}

// db alone (no weight gradient asked for)
template <int ACT>
__global__ __launch_bounds__(256) void db_kernel(Dz d, int64_t rows, int n, float* __restrict__ db) {
  __shared__ float part[256];
  float v = 0.f;
  for (int64_t m = threadIdx.x; m < rows; m += 256) v += dz_at<ACT>(d, m, blockIdx.x);
  part[threadIdx.x] = v;
  __syncthreads();
  for (int h = 128; h > 0; h >>= 1) {
    if (threadIdx.x < h) part[threadIdx.x] += part[threadIdx.x + h];
    __syncthreads();
  }
  if (threadIdx.x == 0) db[blockIdx.x] = part[0];
}

// ---- a ReLU's bits for the layer whose products are plain fp32 ------------------------------
// A wave 64 neighbouring values of a row; bound by bytes.
__global__ __launch_bounds__(256) void relu_mask_kernel(int64_t rows, int n, const float* __restrict__ y, int64_t ldy,
                                                        uint32_t* __restrict__ mask) {
  const int lane = threadIdx.x % 64, parts = (n + 63) / 64, words = (n + 31) / 32;
  for (int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; i < rows * parts; i += (int64_t)gridDim.x * 4) {
    const int64_t m = i / parts;
    const int part = (int)(i % parts), c = part * 64 + lane;
    const uint64_t bits = __ballot(c < n && y[m * ldy + min(c, n - 1)] > 0.f);
    const int word = part * 2 + lane / 32;
    if (lane % 32 == 0 && word < words) mask[m * words + word] = (uint32_t)(bits >> lane);
  }
}
__global__ __launch_bounds__(256) void relu_mask_bwd_kernel(int64_t rows, int n, Dz d, float* __restrict__ dz,
                                                            int64_t lddz) {
  const int lane = threadIdx.x % 64, parts = (n + 63) / 64;
  for (int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; i < rows * parts; i += (int64_t)gridDim.x * 4) {
    const int64_t m = i / parts;
    const int c = (int)(i % parts) * 64 + lane;
    if (c < n) dz[m * lddz + c] = dz_at<DZ_RELU>(d, m, c);
  }
}
unsigned mask_blocks(int64_t rows, int n) {
  return (unsigned)std::min<int64_t>(ceil_div(rows * ceil_div(n, 64), 4), 1 << 16);
}

// ---- launches -------------------------------------------------------------------------
template <int MODE, int ACT, typename X, typename T, int BM, int BN, int WM, int WN>
int launch_tile(const SideArgs& a, hipStream_t stream) {
  using P = ST<BM, BN, WM, WN>;
  const int tiles_n = (int)ceil_div(a.cols, BN);
  const int64_t nblocks = ceil_div(a.rows, BM) * tiles_n;
  INF_CHECK_ARG(nblocks * P::THREADS < (int64_t)1 << 32, "linear_ckpt: too many tiles");
  const auto kernel = split_tile_kernel<MODE, ACT, X, T, BM, BN, WM, WN>;
  static LdsLimit lds;
  const int allowed = lds.raise((const void*)kernel, P::LDS);
  if (allowed != INF_OK) return allowed;
  kernel<<<(unsigned)nblocks, P::THREADS, P::LDS, stream>>>(a, tiles_n, (int)nblocks);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

// The widest tile that still gives each CU a workgroup.  65,536 x 1024 x 256: forward 108 us with 256 x
// 256 (one of 16 waves a CU), 128 with 128 x 128 (two of 8); dx, whose results are many, 163 with 128 x
// 128, where one's stores run beside the other's products, 172 with 256 x 128.  16,384 x 1024 x 256
// forward: 34 with 128 x 128, 42 with 64 x 64; 8192 rows, half as many tiles as CUs, 31 and 26.
template <int MODE, int ACT, typename X, typename T>
int launch_tiles(const SideArgs& a, hipStream_t stream) {
  const int64_t wide = ceil_div(a.rows, 256);
  if (a.cols <= 32) return launch_tile<MODE, ACT, X, T, 64, 32, 4, 1>(a, stream);
  if constexpr (MODE == 0)
    if (a.cols > 128 && wide * ceil_div(a.cols, 256) >= 256)
      return launch_tile<MODE, ACT, X, T, 256, 256, 4, 4>(a, stream);
  if (ceil_div(a.rows, 128) * ceil_div(a.cols, 128) >= 256) return launch_tile<MODE, ACT, X, T, 128, 128, 4, 2>(a, stream);
  return launch_tile<MODE, ACT, X, T, 64, 64, 2, 2>(a, stream);
}

int launch_split(const Weight& w, hipStream_t stream) {
  const auto kernel = along_k(w) ? split_kernel<true> : split_kernel<false>;
  kernel<<<(unsigned)split_blocks(w), 256, 0, stream>>>(w);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

template <typename T>
int launch_before_forward(const Weight& w, const T* x, int64_t rows, int k, int64_t ldx, int8_t* q, int64_t ldq,
                          float* scale, hipStream_t stream) {
  const int nw = split_blocks(w);
  const bool held = with_row_layout<T>(rows, k, [&](auto lpr, auto ch, auto r) {
    constexpr int LPR = decltype(lpr)::value, CH = decltype(ch)::value, R = decltype(r)::value;
    const auto kernel = along_k(w) ? before_forward_kernel<T, LPR, CH, R, true>
                                   : before_forward_kernel<T, LPR, CH, R, false>;
    kernel<<<(unsigned)(nw + ceil_div(rows, R * 256 / LPR)), 256, 0, stream>>>(w, nw, x, rows, k, ldx, q, ldq, scale);
  });
  if (!held) {
    const int rc = launch_quantize_rows(x, sizeof(T) == 4 ? INF_DTYPE_F32 : INF_DTYPE_BF16, rows, k, ldx, q, ldq, scale,
                                        stream);
    return rc != INF_OK ? rc : launch_split(w, stream);
  }
  INF_LAUNCH_CHECK();
  return INF_OK;
}

template <int ACT, int LPR>
void launch_before_dx_as(const Weight& w, const Dz& d, int64_t rows, int n, int* shift, hipStream_t stream) {
  const int nw = split_blocks(w);
  const auto kernel = along_k(w) ? before_dx_kernel<ACT, LPR, true> : before_dx_kernel<ACT, LPR, false>;
  kernel<<<(unsigned)(nw + ceil_div(rows, 256 / LPR)), 256, 0, stream>>>(w, nw, d, rows, n, shift);
}

template <int ACT>
int launch_before_dx(const Weight& w, const Dz& d, int64_t rows, int n, int* shift, hipStream_t stream) {
  if (n <= 16) launch_before_dx_as<ACT, 4>(w, d, rows, n, shift, stream);
  else if (n <= 64) launch_before_dx_as<ACT, 16>(w, d, rows, n, shift, stream);
  else launch_before_dx_as<ACT, 64>(w, d, rows, n, shift, stream);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

template <int ACT>
int launch_dw(const DwArgs& a, hipStream_t stream) {
  static LdsLimit lds;
  const int allowed = lds.raise((const void*)dw_tile_kernel<ACT>, DW_LDS);
  if (allowed != INF_OK) return allowed;
  dw_tile_kernel<ACT><<<(unsigned)(a.tiles * a.splits), DW_THREADS, DW_LDS, stream>>>(a);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

struct DwShape {
  int tiles_k, tiles, splits;
  int64_t rows_a_split;
};

// As many splits as give each CU a workgroup, of two turns at least: with add_slabs_kernel 14 us for
// 512 x 256 x 256 and 12 for 4096 x 64 x 64 (of eight turns: 21 and 19).
DwShape dw_shape(int64_t rows, int n, int k) {
  DwShape d;
  d.tiles_k = (int)ceil_div(k, DW_K);
  d.tiles = d.tiles_k * (int)ceil_div(n, DW_N);
  const int64_t turns = std::max<int64_t>(ceil_div(rows, 32), 1);
  const int64_t splits = std::min<int64_t>(std::max<int64_t>(256 / d.tiles, 1), ceil_div(turns, 2));
  d.rows_a_split = ceil_div(turns, splits) * 32;
  d.splits = (int)std::max<int64_t>(ceil_div(rows, d.rows_a_split), 1);
  return d;
}

// what the products' 32-bit offsets reach: a weight's pieces, and 256 rows
bool fits(int n, int k, int64_t ld) {
  return round_up(n, 256) * round_up(k, 64) < (int64_t)1 << 29 && round_up(k, 256) * round_up(n, 64) < (int64_t)1 << 29 &&
         ld < (int64_t)1 << 21;
}

// offsets in the workspace
struct ForwardSpace {
  int64_t scale, V, vshift, bytes;
};
ForwardSpace forward_space(int64_t rows, int n, int k) {
  ForwardSpace w;
  w.scale = 0;
  w.V = w.scale + round_up(rows * 4, 256);
  w.vshift = w.V + round_up(n, 256) * round_up(k, 64) * 4;
  w.bytes = w.vshift + round_up((int64_t)n * 4, 256);
  return w;
}
struct BackwardSpace {
  int64_t shift, V, vshift, slabs, db, bytes;
};
BackwardSpace backward_space(int64_t rows, int n, int k) {
  const DwShape d = dw_shape(rows, n, k);
  BackwardSpace w;
  w.shift = 0;
  w.V = w.shift + round_up(rows * 4, 256);
  w.vshift = w.V + round_up(k, 256) * round_up(n, 64) * 4;
  w.slabs = w.vshift + round_up((int64_t)k * 4, 256);
  w.db = w.slabs + round_up((int64_t)d.splits * n * k * 4, 256);
  w.bytes = w.db + round_up((int64_t)d.splits * n * 4, 256);
  return w;
}

template <int ACT>
int backward_dx(int64_t rows, int n, int k, const Dz& dz, const float* W, int64_t swn, int64_t swk, void* dx, int dx_dtype,
                int64_t lddx, char* ws, const BackwardSpace& o, hipStream_t st) {
  const Weight w{W, swk, swn, k, n, ws + o.V, (int*)(ws + o.vshift)};
  const bool panel = takes_panel(rows, n, k);
  const int rc = panel ? launch_split(w, st) : launch_before_dx<ACT>(w, dz, rows, n, (int*)(ws + o.shift), st);
  if (rc != INF_OK) return rc;
  SideArgs a{};
  a.rows = rows;
  a.cols = k;
  a.K = n;
  a.shift = (int*)(ws + o.shift);
  a.dz = dz;
  a.V = ws + o.V;
  a.vshift = (int*)(ws + o.vshift);
  a.out = dx;
  a.ldo = lddx;
  if (panel) return dx_dtype == INF_DTYPE_F32 ? launch_panel<ACT, float>(a, st) : launch_panel<ACT, bf16>(a, st);
  return dx_dtype == INF_DTYPE_F32 ? launch_tiles<1, ACT, float, float>(a, st) : launch_tiles<1, ACT, float, bf16>(a, st);
}

template <int ACT>
int backward(int64_t rows, int n, int k, const Dz& dz, const int8_t* q, int64_t ldq, const float* scale, const float* W,
             int64_t swn, int64_t swk, void* dx, int dx_dtype, int64_t lddx, float* dW, int64_t lddw, float* db,
             char* ws, hipStream_t st) {
  const BackwardSpace o = backward_space(rows, n, k);
  int rc = INF_OK;
  if (dx != nullptr)
    rc = in_turns(rows, k, [&](int64_t r, int64_t count) {
      Dz part = dz;
      part.dy += r * dz.lddy;
      if (ACT == DZ_SIGMOID) part.y += r * dz.ldy;
      if (ACT == DZ_RELU) part.mask += r * dz.words;
      char* const out = (char*)dx + r * lddx * (dx_dtype == INF_DTYPE_F32 ? 4 : 2);
      return backward_dx<ACT>(count, n, k, part, W, swn, swk, out, dx_dtype, lddx, ws, o, st);
    });
  if (rc != INF_OK) return rc;
  if (dW != nullptr) {
    const DwShape d = dw_shape(rows, n, k);
    DwArgs a{rows, n, k, dz, q, ldq, scale, d.tiles_k, d.tiles, d.splits, d.rows_a_split, (float*)(ws + o.slabs), k,
             db != nullptr ? (float*)(ws + o.db) : nullptr};
    if (d.splits == 1) {  // nothing to add
      a.out = dW;
      a.ldw = lddw;
      a.db = db;
    }
    rc = launch_dw<ACT>(a, st);
    if (rc != INF_OK) return rc;
    if (d.splits > 1) {
      const int64_t count = (int64_t)n * k;
      add_slabs_kernel<<<(unsigned)ceil_div(count + n, 32), 256, 0, st>>>(a.out, count, k, d.splits, dW, lddw, a.db, n,
                                                                           db);
      INF_LAUNCH_CHECK();
    }
  } else if (db != nullptr) {
    db_kernel<ACT><<<n, 256, 0, st>>>(dz, rows, n, db);
    INF_LAUNCH_CHECK();
  }
  return INF_OK;
}

}  // namespace
}  // namespace inf

using namespace inf;

extern "C" {

int64_t inf_linear_ckpt_workspace_bytes(int64_t rows, int n, int k, int x_dtype, int backward) {
  if (rows < 0 || n < 1 || k < 1) return -1;
  (void)x_dtype;
  return backward ? backward_space(rows, n, k).bytes : forward_space(rows, n, k).bytes;
}

int inf_linear_ckpt_forward(int64_t rows, int n, int k, const void* x, int x_dtype, int64_t ld_x, const float* W,
                            int64_t stride_wn, int64_t stride_wk, const float* bias, const float* add, int64_t ld_add,
                            int act, float* y, int64_t ld_y, uint32_t* mask, int8_t* q, int64_t ld_q, float* scale,
                            void* workspace, inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && n >= 1 && k >= 1 && ld_x >= 0 && ld_y >= n, "linear_ckpt: bad shape");
  INF_CHECK_ARG(rows < (int64_t)1 << 31 && fits(n, k, ld_x), "linear_ckpt: too large");
  INF_CHECK_ARG(act >= 0 && act <= 2, "linear_ckpt: act must be 0 (none), 1 (ReLU) or 2 (sigmoid)");
  INF_CHECK_ARG(x_dtype == INF_DTYPE_F32 || x_dtype == INF_DTYPE_BF16, "linear_ckpt: x must be fp32 or bf16");
  if (rows == 0) return INF_OK;
  INF_CHECK_ARG(x != nullptr && W != nullptr && y != nullptr && workspace != nullptr, "linear_ckpt: null argument");
  INF_CHECK_ARG(add == nullptr || ld_add >= n, "linear_ckpt: bad ld_add");
  INF_CHECK_ARG(q == nullptr || (scale != nullptr && ld_q >= k && ld_q % q8::Q_ALIGN == 0 && (uintptr_t)q % 16 == 0),
                "linear_ckpt: q rows must start on 16 bytes and have scales");
  const hipStream_t st = (hipStream_t)stream;
  char* const ws = (char*)workspace;
  const ForwardSpace o = forward_space(rows, n, k);
  const Weight w{W, stride_wn, stride_wk, n, k, ws + o.V, (int*)(ws + o.vshift)};
  const bool f32 = x_dtype == INF_DTYPE_F32;
  return q8::in_turns(rows, n, [&](int64_t r, int64_t count) {
    SideArgs a{};
    a.rows = count;
    a.cols = n;
    a.K = k;
    a.x = (const char*)x + r * ld_x * (f32 ? 4 : 2);
    a.ldx = ld_x;
    a.V = ws + o.V;
    a.vshift = (int*)(ws + o.vshift);
    a.bias = bias;
    a.add = add != nullptr ? add + r * ld_add : nullptr;
    a.ldadd = ld_add;
    a.act = act;
    a.out = y + r * ld_y;
    a.ldo = ld_y;
    a.mask = mask != nullptr ? mask + r * ((n + 31) / 32) : nullptr;
    float* const s = scale != nullptr ? scale + r : (float*)(ws + o.scale);
    a.scale = s;
    int8_t* const to = q != nullptr ? q + r * ld_q : nullptr;
    const int rc = to == nullptr && scale != nullptr ? launch_split(w, st)
                   : f32 ? launch_before_forward(w, (const float*)a.x, count, k, ld_x, to, ld_q, s, st)
                         : launch_before_forward(w, (const bf16*)a.x, count, k, ld_x, to, ld_q, s, st);
    if (rc != INF_OK) return rc;
    return f32 ? launch_tiles<0, 0, float, float>(a, st) : launch_tiles<0, 0, bf16, float>(a, st);
  });
}

int inf_linear_ckpt_backward(int64_t rows, int n, int k, const float* dy, int64_t ld_dy, int act, const float* y,
                             int64_t ld_y, const uint32_t* mask, const int8_t* q, int64_t ld_q, const float* scale,
                             const float* W, int64_t stride_wn, int64_t stride_wk, void* dx, int dx_dtype,
                             int64_t ld_dx, float* dW, int64_t ld_dw, float* db, void* workspace,
                             inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && n >= 1 && k >= 1 && ld_dy >= 0, "linear_ckpt backward: bad shape");
  INF_CHECK_ARG(rows < (int64_t)1 << 31 && fits(n, k, ld_dy) && fits(n, k, ld_y), "linear_ckpt backward: too large");
  INF_CHECK_ARG(act >= 0 && act <= 2, "linear_ckpt backward: act must be 0 (none), 1 (ReLU) or 2 (sigmoid)");
  INF_CHECK_ARG(dx == nullptr || (W != nullptr && ld_dx >= k && (dx_dtype == INF_DTYPE_F32 || dx_dtype == INF_DTYPE_BF16)),
                "linear_ckpt backward: dx needs the weight and is fp32 or bf16");
  INF_CHECK_ARG(dW == nullptr || ld_dw >= k, "linear_ckpt backward: bad ld_dw");
  INF_CHECK_ARG(rows == 0 || (dy != nullptr && workspace != nullptr), "linear_ckpt backward: null argument");
  INF_CHECK_ARG(rows == 0 || act != 1 || mask != nullptr, "linear_ckpt backward: a ReLU needs its mask");
  INF_CHECK_ARG(rows == 0 || act != 2 || (y != nullptr && ld_y >= n), "linear_ckpt backward: a sigmoid needs its output");
  INF_CHECK_ARG(rows == 0 || dW == nullptr || (q != nullptr && scale != nullptr && ld_q >= k &&
                                               ld_q % q8::Q_ALIGN == 0 && (uintptr_t)q % 16 == 0),
                "linear_ckpt backward: dW needs the 8-bit rows");
  const hipStream_t st = (hipStream_t)stream;
  const Dz dz{dy, ld_dy, y, ld_y, mask, (n + 31) / 32};
  char* const ws = (char*)workspace;
#define INF_BACKWARD(ACT) \
  backward<ACT>(rows, n, k, dz, q, ld_q, scale, W, stride_wn, stride_wk, dx, dx_dtype, ld_dx, dW, ld_dw, db, ws, st)
  return act == 1 ? INF_BACKWARD(DZ_RELU) : act == 2 ? INF_BACKWARD(DZ_SIGMOID) : INF_BACKWARD(DZ_NONE);
#undef INF_BACKWARD
}

int inf_relu_mask(int64_t rows, int n, const float* y, int64_t ld_y, uint32_t* mask, inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && n >= 1 && ld_y >= n && rows < (int64_t)1 << 31, "relu_mask: bad shape");
  if (rows == 0) return INF_OK;
  INF_CHECK_ARG(y != nullptr && mask != nullptr, "relu_mask: null argument");
  relu_mask_kernel<<<mask_blocks(rows, n), 256, 0, (hipStream_t)stream>>>(rows, n, y, ld_y, mask);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

int inf_relu_mask_bwd(int64_t rows, int n, const float* dy, int64_t ld_dy, const uint32_t* mask, float* dz, int64_t ld_dz,
                      inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && n >= 1 && ld_dy >= 0 && ld_dz >= n && rows < (int64_t)1 << 31, "relu_mask_bwd: bad shape");
  if (rows == 0) return INF_OK;
  INF_CHECK_ARG(dy != nullptr && mask != nullptr && dz != nullptr, "relu_mask_bwd: null argument");
  const Dz d{dy, ld_dy, nullptr, 0, mask, (n + 31) / 32};
  relu_mask_bwd_kernel<<<mask_blocks(rows, n), 256, 0, (hipStream_t)stream>>>(rows, n, d, dz, ld_dz);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

}  // extern "C"
