// A linear layer whose inputs are kept in 8 bits until its backward (quant.hpp), for training:
//   forward   y = act(x W^T + bias + add)       from x as it is, in fp32
//             kept: q, s of x; one bit y > 0 (ReLU); y itself is the layer's output (sigmoid)
//   backward  dz = dy [y > 0] | dy y (1 - y) | dy
//             dx = dz W     dW = dz^T (s q)     db = sum_m dz
#include <algorithm>

#include "quant.hpp"

namespace inf {
namespace {

using namespace q8;

constexpr int CT = 64, CK = 16;  // output tile, k tile

// C(m, n) = act(sum_k A(m, k) B(n, k) + bias[n] + beta C(m, n)); A and B by functor, stored by functor
template <class FA, class FB, class ST>
__device__ __forceinline__ void tile_product(int64_t m0, int64_t n0, int64_t M, int64_t N, int64_t K, const FA& fa,
                                             const FB& fb, const ST& store) {
  __shared__ float As[CK][CT + 1], Bs[CK][CT + 1];
  const int t = threadIdx.x, tm = (t / 16) * 4, tn = (t % 16) * 4;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += CK) {
    for (int i = t; i < CK * CT; i += 256) {
      const int kk = i / CT, r = i % CT;
      As[kk][r] = m0 + r < M && k0 + kk < K ? fa(m0 + r, k0 + kk) : 0.f;
      Bs[kk][r] = n0 + r < N && k0 + kk < K ? fb(n0 + r, k0 + kk) : 0.f;
    }
    __syncthreads();
    for (int kk = 0; kk < CK; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[kk][tm + i], Bs[kk][tn + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j)
      if (m0 + tm + i < M && n0 + tn + j < N) store(m0 + tm + i, n0 + tn + j, acc[i][j]);
}

template <typename T>
__global__ __launch_bounds__(256) void forward_kernel(int64_t rows, int n, int k, const T* __restrict__ x, int64_t ldx,
                                                      const float* __restrict__ W, int64_t swn, int64_t swk,
                                                      const float* __restrict__ bias, const float* __restrict__ add,
                                                      int64_t ldadd, int act, float* __restrict__ y, int64_t ldy) {
  for (int64_t m0 = (int64_t)blockIdx.y * CT; m0 < rows; m0 += (int64_t)gridDim.y * CT)
    tile_product(m0, (int64_t)blockIdx.x * CT, rows, n, k, [&](int64_t m, int64_t c) { return to_f32(x[m * ldx + c]); },
                 [&](int64_t r, int64_t c) { return W[r * swn + c * swk]; },
                 [&](int64_t m, int64_t c, float v) {
                   if (bias != nullptr) v += bias[c];
                   if (add != nullptr) v += add[m * ldadd + c];
                   y[m * ldy + c] = activate(v, act);
                 });
}

// bit j of word w of a row: y[32 w + j] > 0
__global__ __launch_bounds__(256) void mask_kernel(int64_t rows, int n, const float* __restrict__ y, int64_t ldy,
                                                   uint32_t* __restrict__ mask) {
  const int words = (n + 31) / 32;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * words; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / words;
    const int w = (int)(i % words);
    uint32_t b = 0;
    for (int j = 0; j < 32 && 32 * w + j < n; ++j) b |= (uint32_t)(y[m * ldy + 32 * w + j] > 0.f) << j;
    mask[i] = b;
  }
}

__global__ __launch_bounds__(256) void dz_kernel(int64_t rows, int n, const float* __restrict__ dy, int64_t lddy,
                                                 int act, const float* __restrict__ y, int64_t ldy,
                                                 const uint32_t* __restrict__ mask, float* __restrict__ dz) {
  const int words = (n + 31) / 32;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * n; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / n;
    const int c = (int)(i % n);
    float g = dy[m * lddy + c];
    if (act == 1) g = (mask[m * words + c / 32] >> (c % 32)) & 1 ? g : 0.f;
    if (act == 2) g = g * (y[m * ldy + c] * (1.f - y[m * ldy + c]));
    dz[i] = g;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void dx_kernel(int64_t rows, int n, int k, const float* __restrict__ dz,
                                                 const float* __restrict__ W, int64_t swn, int64_t swk,
                                                 T* __restrict__ dx, int64_t lddx) {
  for (int64_t m0 = (int64_t)blockIdx.y * CT; m0 < rows; m0 += (int64_t)gridDim.y * CT)
    tile_product(m0, (int64_t)blockIdx.x * CT, rows, k, n, [&](int64_t m, int64_t c) { return dz[m * n + c]; },
                 [&](int64_t r, int64_t c) { return W[c * swn + r * swk]; },
                 [&](int64_t m, int64_t c, float v) { dx[m * lddx + c] = from_f32<T>(v); });
}

__global__ __launch_bounds__(256) void dw_kernel(int64_t rows, int n, int k, const float* __restrict__ dz,
                                                 const int8_t* __restrict__ q, int64_t ldq,
                                                 const float* __restrict__ s, float* __restrict__ dW, int64_t lddw) {
  tile_product((int64_t)blockIdx.y * CT, (int64_t)blockIdx.x * CT, n, k, rows,
               [&](int64_t r, int64_t m) { return dz[m * n + r]; },
               [&](int64_t c, int64_t m) { return (float)q[m * ldq + c] * s[m]; },
               [&](int64_t r, int64_t c, float v) { dW[r * lddw + c] = v; });
}

__global__ __launch_bounds__(256) void db_kernel(int64_t rows, int n, const float* __restrict__ dz,
                                                 float* __restrict__ db) {
  __shared__ float part[256];
  float v = 0.f;
  for (int64_t m = threadIdx.x; m < rows; m += 256) v += dz[m * n + blockIdx.x];
  part[threadIdx.x] = v;
  __syncthreads();
  for (int h = 128; h > 0; h >>= 1) {
    if (threadIdx.x < h) part[threadIdx.x] += part[threadIdx.x + h];
    __syncthreads();
  }
  if (threadIdx.x == 0) db[blockIdx.x] = part[0];
}

unsigned blocks_of(int64_t n) { return (unsigned)std::min<int64_t>(std::max<int64_t>(ceil_div(n, 256), 1), 1 << 16); }
dim3 tiles(int64_t m, int64_t n) {
  return dim3((unsigned)ceil_div(n, CT), (unsigned)std::min<int64_t>(std::max<int64_t>(ceil_div(m, CT), 1), 65535));
}

}  // namespace
}  // namespace inf

using namespace inf;

extern "C" {

int64_t inf_linear_ckpt_workspace_bytes(int64_t rows, int n, int k, int x_dtype, int backward) {
  if (rows < 0 || n < 1 || k < 1) return -1;
  (void)x_dtype;
  return backward ? round_up(std::max<int64_t>(rows * n * 4, 256), 256) : 256;
}

int inf_linear_ckpt_forward(int64_t rows, int n, int k, const void* x, int x_dtype, int64_t ld_x, const float* W,
                            int64_t stride_wn, int64_t stride_wk, const float* bias, const float* add, int64_t ld_add,
                            int act, float* y, int64_t ld_y, uint32_t* mask, int8_t* q, int64_t ld_q, float* scale,
                            void* workspace, inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && n >= 1 && k >= 1 && ld_x >= 0 && ld_y >= n, "linear_ckpt: bad shape");
  INF_CHECK_ARG(act >= 0 && act <= 2, "linear_ckpt: act must be 0 (none), 1 (ReLU) or 2 (sigmoid)");
  INF_CHECK_ARG(x_dtype == INF_DTYPE_F32 || x_dtype == INF_DTYPE_BF16, "linear_ckpt: x must be fp32 or bf16");
  if (rows == 0) return INF_OK;
  INF_CHECK_ARG(x != nullptr && W != nullptr && y != nullptr && workspace != nullptr, "linear_ckpt: null argument");
  INF_CHECK_ARG(add == nullptr || ld_add >= n, "linear_ckpt: bad ld_add");
  INF_CHECK_ARG(q == nullptr || (scale != nullptr && ld_q >= k && ld_q % q8::Q_ALIGN == 0 && (uintptr_t)q % 16 == 0),
                "linear_ckpt: q rows must start on 16 bytes and have scales");
  const hipStream_t st = (hipStream_t)stream;
  if (q != nullptr) {
    const int rc = launch_quantize_rows(x, x_dtype, rows, k, ld_x, q, ld_q, scale, st);
    if (rc != INF_OK) return rc;
  }
  if (x_dtype == INF_DTYPE_F32)
    forward_kernel<<<tiles(rows, n), 256, 0, st>>>(rows, n, k, (const float*)x, ld_x, W, stride_wn, stride_wk, bias,
                                                    add, ld_add, act, y, ld_y);
  else
    forward_kernel<<<tiles(rows, n), 256, 0, st>>>(rows, n, k, (const bf16*)x, ld_x, W, stride_wn, stride_wk, bias, add,
                                                    ld_add, act, y, ld_y);
  INF_LAUNCH_CHECK();
  if (mask != nullptr) {
    mask_kernel<<<blocks_of(rows * ((n + 31) / 32)), 256, 0, st>>>(rows, n, y, ld_y, mask);
    INF_LAUNCH_CHECK();
  }
  return INF_OK;
}

int inf_linear_ckpt_backward(int64_t rows, int n, int k, const float* dy, int64_t ld_dy, int act, const float* y,
                             int64_t ld_y, const uint32_t* mask, const int8_t* q, int64_t ld_q, const float* scale,
                             const float* W, int64_t stride_wn, int64_t stride_wk, void* dx, int dx_dtype,
                             int64_t ld_dx, float* dW, int64_t ld_dw, float* db, void* workspace,
                             inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && n >= 1 && k >= 1 && ld_dy >= 0, "linear_ckpt backward: bad shape");
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
  float* dz = (float*)workspace;
  if (rows > 0) {
    dz_kernel<<<blocks_of(rows * n), 256, 0, st>>>(rows, n, dy, ld_dy, act, y, ld_y, mask, dz);
    INF_LAUNCH_CHECK();
  }
  if (dx != nullptr && rows > 0) {
    if (dx_dtype == INF_DTYPE_F32)
      dx_kernel<<<tiles(rows, k), 256, 0, st>>>(rows, n, k, dz, W, stride_wn, stride_wk, (float*)dx, ld_dx);
    else
      dx_kernel<<<tiles(rows, k), 256, 0, st>>>(rows, n, k, dz, W, stride_wn, stride_wk, (bf16*)dx, ld_dx);
    INF_LAUNCH_CHECK();
  }
  if (dW != nullptr) {
    dw_kernel<<<tiles(n, k), 256, 0, st>>>(rows, n, k, dz, q, ld_q, scale, dW, ld_dw);
    INF_LAUNCH_CHECK();
  }
  if (db != nullptr) {
    db_kernel<<<n, 256, 0, st>>>(rows, n, dz, db);
    INF_LAUNCH_CHECK();
  }
  return INF_OK;
}

}  // extern "C"
