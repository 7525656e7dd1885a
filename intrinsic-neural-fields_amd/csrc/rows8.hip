// Rows in 8 bits (quant.hpp): the quantiser, its inverse, and the packing of 8-bit weights.
//   inf_quantize_rows: x [rows][k] fp32 / bf16 -> q int8, scale fp32
//   inf_restore_rows:  q s, rounded to fp32, for bf16 then to that
//   inf_pack_weight:   int8 weights of any strides -> rows of whole 128 bytes, zero behind k
#include <algorithm>

#include "quant.hpp"

namespace inf {
namespace {

using namespace q8;

template <typename T, int LPR, int CH, int R>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int k, int64_t ldx,
                                                            int8_t* __restrict__ q, int64_t ldq,
                                                            float* __restrict__ scale) {
  quantize_rows_block<T, LPR, CH, R>(blockIdx.x, x, rows, k, ldx, q, ldq, scale);
}

// Rows too long for a wave's registers: a workgroup a row, which is read twice.
template <typename T>
__global__ __launch_bounds__(256) void quantize_long_rows_kernel(const T* __restrict__ x, int64_t rows, int k,
                                                                 int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                                                                 float* __restrict__ scale) {
  constexpr int V = Chunk<T>::V;
  __shared__ unsigned part[4];
  for (int64_t m = blockIdx.x; m < rows; m += gridDim.x) {
    unsigned a = 0;
    float v[V];
    for (int c = threadIdx.x * V; c < k; c += 256 * V) {
      load_chunk(x + m * ldx, c, k, v);
#pragma unroll
      for (int e = 0; e < V; ++e) a = max(a, abs_bits(v[e]));
    }
    a = row_max<64>(a);
    __syncthreads();  // the last row's maximum has been read
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = a;
    __syncthreads();
    const RowScale rs = row_scale(max(max(part[0], part[1]), max(part[2], part[3])));
    if (threadIdx.x == 0) scale[m] = rs.s;
    if (q == nullptr) continue;
    for (int c = threadIdx.x * V; c < k; c += 256 * V) {
      load_chunk(x + m * ldx, c, k, v);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c + e < k) q[m * ldq + c + e] = (int8_t)quantize<T>(v[e], rs);
    }
  }
}

// LPR lanes a row, each lane 4 values a turn (one 4-byte load, one 16- or 8-byte store).
template <typename T, int LPR>
__global__ __launch_bounds__(256) void restore_rows_kernel(const int8_t* __restrict__ q, int64_t ldq,
                                                           const float* __restrict__ scale, int64_t rows, int k,
                                                           T* __restrict__ out, int64_t ldo) {
  typedef T O __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const int64_t m = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (m >= rows) return;
  const float s = scale[m];
  const int8_t* const from = q + m * ldq;
  T* const to = out + m * ldo;
#pragma unroll 4
  for (int c = (threadIdx.x % LPR) * 4; c < k; c += LPR * 4) {
    // q rows start on 16 bytes and their length is a multiple: a whole load stays in the row
    const int w = *reinterpret_cast<const int*>(from + c);
    O o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = from_f32<T>((float)(int8_t)(w >> (8 * e)) * s);
    if (c + 4 <= k) {
      *reinterpret_cast<O*>(to + c) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < k) to[c + e] = o[e];
    }
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

template <typename T>
static void quantize_rows_any(const T* x, int64_t rows, int k, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                              hipStream_t st) {
  const bool held = with_row_layout<T>(rows, k, [&](auto lpr, auto ch, auto r) {
    constexpr int LPR = decltype(lpr)::value, CH = decltype(ch)::value, R = decltype(r)::value;
    quantize_rows_kernel<T, LPR, CH, R><<<(unsigned)ceil_div(rows, R * 256 / LPR), 256, 0, st>>>(x, rows, k, ldx, q, ldq, scale);
  });
  if (!held) quantize_long_rows_kernel<<<blocks_of(rows), 256, 0, st>>>(x, rows, k, ldx, q, ldq, scale);
}

template <typename T>
static void restore_rows_any(const int8_t* q, int64_t ldq, const float* scale, int64_t rows, int k, T* out,
                             int64_t ldo, hipStream_t st) {
  if (k <= 16) restore_rows_kernel<T, 4><<<(unsigned)ceil_div(rows, 64), 256, 0, st>>>(q, ldq, scale, rows, k, out, ldo);
  else if (k <= 64) restore_rows_kernel<T, 16><<<(unsigned)ceil_div(rows, 16), 256, 0, st>>>(q, ldq, scale, rows, k, out, ldo);
  else if (k <= 4096) restore_rows_kernel<T, 64><<<(unsigned)ceil_div(rows, 4), 256, 0, st>>>(q, ldq, scale, rows, k, out, ldo);
  else restore_rows_kernel<T, 256><<<(unsigned)rows, 256, 0, st>>>(q, ldq, scale, rows, k, out, ldo);
}

int launch_quantize_rows(const void* x, int dtype, int64_t rows, int k, int64_t ldx, int8_t* q, int64_t ldq,
                         float* scale, hipStream_t stream) {
  return in_turns(rows, 1, [&](int64_t r, int64_t count) {
    int8_t* const to = q != nullptr ? q + r * ldq : nullptr;
    if (dtype == INF_DTYPE_F32) quantize_rows_any((const float*)x + r * ldx, count, k, ldx, to, ldq, scale + r, stream);
    else quantize_rows_any((const bf16*)x + r * ldx, count, k, ldx, to, ldq, scale + r, stream);
    INF_LAUNCH_CHECK();
    return INF_OK;
  });
}

}  // namespace inf

using namespace inf;

extern "C" {

int inf_quantize_rows(const void* x, int x_dtype, int64_t rows, int k, int64_t ld_x, int8_t* q, int64_t ld_q,
                      float* scale, inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && k >= 1 && ld_x >= 0, "quantize_rows: bad shape");
  INF_CHECK_ARG(x_dtype == INF_DTYPE_F32 || x_dtype == INF_DTYPE_BF16, "quantize_rows: x must be fp32 or bf16");
  INF_CHECK_ARG(ld_q >= k && ld_q % q8::Q_ALIGN == 0, "quantize_rows: q rows must start on 16 bytes");
  INF_CHECK_ARG(rows < (int64_t)1 << 31, "quantize_rows: too many rows");
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
  INF_CHECK_ARG(rows < (int64_t)1 << 31, "restore_rows: too many rows");
  if (rows == 0) return INF_OK;
  INF_CHECK_ARG(q != nullptr && scale != nullptr && out != nullptr && (uintptr_t)q % 16 == 0,
                "restore_rows: null or unaligned argument");
  const hipStream_t st = (hipStream_t)stream;
  return q8::in_turns(rows, 1, [&](int64_t r, int64_t count) {
    const int8_t* const from = q + r * ld_q;
    if (out_dtype == INF_DTYPE_F32) restore_rows_any(from, ld_q, scale + r, count, k, (float*)out + r * ld_out, ld_out, st);
    else restore_rows_any(from, ld_q, scale + r, count, k, (bf16*)out + r * ld_out, ld_out, st);
    INF_LAUNCH_CHECK();
    return INF_OK;
  });
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
