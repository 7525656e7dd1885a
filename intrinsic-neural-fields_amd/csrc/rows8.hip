// Rows in 8 bits (quant.hpp): the quantiser, its inverse, and the packing of 8-bit weights.
//   inf_quantize_rows: x [rows][k] fp32 / bf16 -> q int8, scale fp32
//   inf_restore_rows:  q s, rounded once to fp32 / bf16
//   inf_pack_weight:   int8 weights of any strides -> rows of whole 128 bytes, zero behind k
#include <algorithm>

#include "quant.hpp"

namespace inf {
namespace {

using namespace q8;

template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int k, int64_t ldx,
                                                            int8_t* __restrict__ q, int64_t ldq,
                                                            float* __restrict__ scale) {
  __shared__ unsigned part[256];
  for (int64_t m = blockIdx.x; m < rows; m += gridDim.x) {
    unsigned a = 0;
    for (int j = threadIdx.x; j < k; j += 256) a = max(a, abs_bits(to_f32(x[m * ldx + j])));
    part[threadIdx.x] = a;
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) {
      if (threadIdx.x < h) part[threadIdx.x] = max(part[threadIdx.x], part[threadIdx.x + h]);
      __syncthreads();
    }
    const RowScale rs = row_scale(part[0]);
    __syncthreads();
    for (int j = threadIdx.x; j < k; j += 256) q[m * ldq + j] = (int8_t)quantize(to_f32(x[m * ldx + j]), rs);
    if (threadIdx.x == 0) scale[m] = rs.s;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void restore_rows_kernel(const int8_t* __restrict__ q, int64_t ldq,
                                                           const float* __restrict__ scale, int64_t rows, int k,
                                                           T* __restrict__ out, int64_t ldo) {
  for (int64_t m = blockIdx.x; m < rows; m += gridDim.x) {
    const float s = scale[m];
    for (int j = threadIdx.x; j < k; j += 256) out[m * ldo + j] = from_f32<T>((float)q[m * ldq + j] * s);
  }
}

__global__ __launch_bounds__(256) void pack_weight_kernel(const int8_t* __restrict__ q, int64_t sn, int64_t sk, int n,
                                                          int k, int8_t* __restrict__ packed, int64_t ldw) {
  const int64_t total = (int64_t)n * ldw;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / ldw, c = i % ldw;
    packed[i] = c < k ? q[r * sn + c * sk] : 0;
  }
}

unsigned blocks_of(int64_t n) { return (unsigned)std::min<int64_t>(std::max<int64_t>(n, 1), 1 << 16); }

}  // namespace

int launch_quantize_rows(const void* x, int dtype, int64_t rows, int k, int64_t ldx, int8_t* q, int64_t ldq,
                         float* scale, hipStream_t stream) {
  if (dtype == INF_DTYPE_F32)
    quantize_rows_kernel<<<blocks_of(rows), 256, 0, stream>>>((const float*)x, rows, k, ldx, q, ldq, scale);
  else
    quantize_rows_kernel<<<blocks_of(rows), 256, 0, stream>>>((const bf16*)x, rows, k, ldx, q, ldq, scale);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

}  // namespace inf

using namespace inf;

extern "C" {

int inf_quantize_rows(const void* x, int x_dtype, int64_t rows, int k, int64_t ld_x, int8_t* q, int64_t ld_q,
                      float* scale, inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && k >= 1 && ld_x >= 0, "quantize_rows: bad shape");
  INF_CHECK_ARG(x_dtype == INF_DTYPE_F32 || x_dtype == INF_DTYPE_BF16, "quantize_rows: x must be fp32 or bf16");
  INF_CHECK_ARG(ld_q >= k && ld_q % q8::Q_ALIGN == 0, "quantize_rows: q rows must start on 16 bytes");
  if (rows == 0) return INF_OK;
  INF_CHECK_ARG(x != nullptr && q != nullptr && scale != nullptr && (uintptr_t)q % 16 == 0,
                "quantize_rows: null or unaligned argument");
  return launch_quantize_rows(x, x_dtype, rows, k, ld_x, q, ld_q, scale, (hipStream_t)stream);
}

int inf_restore_rows(const int8_t* q, int64_t ld_q, const float* scale, int64_t rows, int k, void* out, int out_dtype,
                     int64_t ld_out, inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && k >= 1 && ld_out >= k, "restore_rows: bad shape");
  INF_CHECK_ARG(out_dtype == INF_DTYPE_F32 || out_dtype == INF_DTYPE_BF16, "restore_rows: out must be fp32 or bf16");
  INF_CHECK_ARG(ld_q >= k && ld_q % q8::Q_ALIGN == 0, "restore_rows: q rows must start on 16 bytes");
  if (rows == 0) return INF_OK;
  INF_CHECK_ARG(q != nullptr && scale != nullptr && out != nullptr && (uintptr_t)q % 16 == 0,
                "restore_rows: null or unaligned argument");
  if (out_dtype == INF_DTYPE_F32)
    restore_rows_kernel<<<blocks_of(rows), 256, 0, (hipStream_t)stream>>>(q, ld_q, scale, rows, k, (float*)out, ld_out);
  else
    restore_rows_kernel<<<blocks_of(rows), 256, 0, (hipStream_t)stream>>>(q, ld_q, scale, rows, k, (bf16*)out, ld_out);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

int64_t inf_packed_weight_bytes(int n, int k) {
  if (n < 0 || k < 1) return -1;
  return n * round_up(k, q8::W_ALIGN);
}

int inf_pack_weight(const int8_t* q, int64_t stride_n, int64_t stride_k, int n, int k, int8_t* packed,
                    inf_stream_t stream) {
  INF_CHECK_ARG(n >= 0 && k >= 1, "pack_weight: bad shape");
  if (n == 0) return INF_OK;
  INF_CHECK_ARG(q != nullptr && packed != nullptr && (uintptr_t)packed % 16 == 0, "pack_weight: null or unaligned argument");
  const int64_t ldw = round_up(k, q8::W_ALIGN);
  pack_weight_kernel<<<blocks_of(ceil_div(n * ldw, 256)), 256, 0, (hipStream_t)stream>>>(q, stride_n, stride_k, n, k,
                                                                                        packed, ldw);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

}  // extern "C"
