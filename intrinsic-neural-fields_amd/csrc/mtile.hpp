// The parts that the matrix tiles of linear8.hip and ckpt.hip share: LDS stages of 128-byte
// rows, filled straight from memory, and their fragments.
#pragma once

#include <atomic>

#include "quant.hpp"

namespace inf {
namespace mt {

typedef __attribute__((address_space(3))) void lds_void;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// An offset that the compiler adds to its uniform base in the load itself: left to it, it adds
// them before the loop, into two registers each, and spills.
__device__ __forceinline__ unsigned pinned(unsigned o) {
  asm volatile("" : "+v"(o));
  return o;
}

// Chunk c (16 bytes) of a stage row lies at c ^ ((row >> 1) & 7): the 16 rows that a
// fragment read touches at one c fall into all 64 banks evenly.
__device__ __forceinline__ int swz(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int chunk_at(int row, int c) { return row * 128 + ((c ^ swz(row)) << 4); }

// The workgroup's barrier once this wave's LDS writes, and its loads (to registers and to LDS)
// but the last N that it issued, have arrived.  The wait is the builtin, not inline assembly:
// the compiler then knows which registers are there, and does not wait for later loads to use
// them (s_waitcnt vmcnt(N) expcnt(7) lgkmcnt(0)).
template <int N>
__device__ __forceinline__ void wait_barrier() {
  static_assert(N < 16, "vmcnt's low field");
  asm volatile("" ::: "memory");  // (a fence would wait for every load)
  __builtin_amdgcn_s_waitcnt(0x0070 | N);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_all_barrier() { wait_barrier<0>(); }

// The same where nothing but LDS writes is waited for: the loads are registers'.
__device__ __forceinline__ void wait_lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // vmcnt(63) expcnt(7) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Between writes and reads of a piece of LDS that one wave alone uses: its LDS accesses are served
// in order, the compiler has to leave them so.
__device__ __forceinline__ void own_lds_order() { asm volatile("" ::: "memory"); }

// Workgroups that one XCD receives (every eighth) take consecutive tiles, so that tiles which
// share rows find them in that XCD's L2.
__device__ __forceinline__ int xcd_order(int orig, int nblocks) {
  const int q = nblocks / 8, r = nblocks % 8, xcd = orig % 8;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + orig / 8;
}

// Leave for a kernel to take more LDS than a launch may by default: asked for once a device, by
// whichever call comes first.
struct LdsLimit {
  std::atomic<uint64_t> devices{0};
  int raise(const void* kernel, int bytes) {
    int device = 0;
    INF_HIP_TRY(hipGetDevice(&device));
    const uint64_t bit = (uint64_t)1 << (device & 63);
    if (!(devices.load(std::memory_order_relaxed) & bit)) {
      INF_HIP_TRY(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
      devices.fetch_or(bit, std::memory_order_relaxed);
    }
    return INF_OK;
  }
};

}  // namespace mt
}  // namespace inf
