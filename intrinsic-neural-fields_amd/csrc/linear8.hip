// A linear layer on rows and weights in 8-bit whole numbers (quant.hpp), for rendering:
//   acc_mn = sum_k qx_mk qw_nk                              exact, in 32 bits (k <= 2^17)
//   z_mn   = fl(fl(acc) fl(sx_m sw_n)) + bias_n + add_mn    each operation rounded once to fp32
//   y      = act(z), as fp32, bf16, or in 8-bit rows again
// The roundings are written out one by one and never contracted: a row that goes into 8
// bits again has the same numbers whichever kernel made it.
#include <algorithm>

#include "quant.hpp"

namespace inf {
namespace {

using namespace q8;

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
};

__device__ __forceinline__ float combine(int acc, float sx, float sw, float bias, float add, int act) {
#pragma clang fp contract(off)
  float z = (float)acc * (sx * sw);
  z = z + bias;
  z = z + add;
  return activate(z, act);
}

template <typename T>
__global__ __launch_bounds__(256) void linear8_kernel(Linear8Args a) {
  __shared__ int As[64][17], Bs[64][17];  // 64 rows of 64 values each
  const int t = threadIdx.x;
  const int tm = (t / 16) * 4, tn = (t % 16) * 4;
  const int n0 = blockIdx.x * 64;
  for (int64_t m0 = (int64_t)blockIdx.y * 64; m0 < a.rows; m0 += (int64_t)gridDim.y * 64) {
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.k; k0 += 64) {
      for (int i = t; i < 64 * 16; i += 256) {
        const int r = i / 16, c = i % 16;
        int av = 0, bv = 0;
        for (int e = 0; e < 4; ++e) {
          const int kk = k0 + 4 * c + e;
          if (kk < a.k && m0 + r < a.rows) av |= (int)(uint8_t)a.q[(m0 + r) * a.ldq + kk] << (8 * e);
          if (kk < a.k && n0 + r < a.n) bv |= (int)(uint8_t)a.w[(int64_t)(n0 + r) * a.ldw + kk] << (8 * e);
        }
        As[r][c] = av;
        Bs[r][c] = bv;
      }
      __syncthreads();
      for (int c = 0; c < 16; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[i][j] = __builtin_amdgcn_sdot4(As[tm + i][c], Bs[tn + j][c], acc[i][j], false);
      __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const int64_t m = m0 + tm + i;
        const int n = n0 + tn + j;
        if (m >= a.rows || n >= a.n) continue;
        const float y = combine(acc[i][j], a.qs[m], a.ws[n], a.bias != nullptr ? a.bias[n] : 0.f,
                                a.add != nullptr ? a.add[m * a.ldadd + n] : 0.f, a.act);
        reinterpret_cast<T*>(a.out)[m * a.ldo + n] = from_f32<T>(y);
      }
  }
}

int launch_linear8(const Linear8Args& a, int out_dtype, hipStream_t stream) {
  const dim3 grid((unsigned)ceil_div(a.n, 64), (unsigned)std::min<int64_t>(ceil_div(a.rows, 64), 65535));
  if (out_dtype == INF_DTYPE_BF16) linear8_kernel<bf16><<<grid, 256, 0, stream>>>(a);
  else linear8_kernel<float><<<grid, 256, 0, stream>>>(a);
  INF_LAUNCH_CHECK();
  return INF_OK;
}

struct Workspace {
  int64_t q, qs, y, bytes;  // offsets: x in 8 bits, its scales, the fp32 rows that go into 8 bits
};

Workspace workspace_of(int64_t rows, int n, int k, int x_dtype, int out_dtype) {
  Workspace w{0, 0, 0, 0};
  if (x_dtype != INF_DTYPE_I8) {
    w.q = w.bytes;
    w.bytes += round_up(rows * round_up(k, Q_ALIGN) + Q_SLACK, 256);
    w.qs = w.bytes;
    w.bytes += round_up(rows * 4, 256);
  }
  if (out_dtype == INF_DTYPE_I8) {
    w.y = w.bytes;
    w.bytes += round_up(rows * n * 4, 256);
  }
  return w;
}

}  // namespace
}  // namespace inf

using namespace inf;

extern "C" {

int64_t inf_linear_int_workspace_bytes(int64_t rows, int n, int k, int x_dtype, int out_dtype) {
  if (rows < 0 || n < 1 || k < 1) return -1;
  return workspace_of(rows, n, k, x_dtype, out_dtype).bytes;
}

int inf_linear_int(int64_t rows, int n, int k, const void* x, int x_dtype, int64_t ld_x, const float* x_scale,
                   const int8_t* w, const float* w_scale, const float* bias, const float* add, int64_t ld_add, int act,
                   void* out, int out_dtype, int64_t ld_out, float* out_scale, void* workspace, inf_stream_t stream) {
  INF_CHECK_ARG(rows >= 0 && n >= 1 && k >= 1 && ld_x >= 0 && ld_out >= n, "linear_int: bad shape");
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
  const Workspace o = workspace_of(rows, n, k, x_dtype, out_dtype);
  INF_CHECK_ARG(o.bytes == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0),
                "linear_int: null or unaligned workspace");
  char* const wsp = (char*)workspace;
  Linear8Args a{rows, n, k, (const int8_t*)x, ld_x, x_scale, w, round_up(k, q8::W_ALIGN), w_scale, bias, add, ld_add,
                act, out, ld_out};
  if (!x8) {
    a.q = (int8_t*)(wsp + o.q);
    a.ldq = round_up(k, q8::Q_ALIGN);
    a.qs = (float*)(wsp + o.qs);
    const int rc = launch_quantize_rows(x, x_dtype, rows, k, ld_x, (int8_t*)a.q, a.ldq, (float*)a.qs, (hipStream_t)stream);
    if (rc != INF_OK) return rc;
  }
  if (!y8) return launch_linear8(a, out_dtype, (hipStream_t)stream);
  a.out = wsp + o.y;
  a.ldo = n;
  const int rc = launch_linear8(a, INF_DTYPE_F32, (hipStream_t)stream);
  if (rc != INF_OK) return rc;
  return launch_quantize_rows(a.out, INF_DTYPE_F32, rows, n, n, (int8_t*)out, ld_out, out_scale, (hipStream_t)stream);
}

}  // extern "C"
