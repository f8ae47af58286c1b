// Device helpers shared by the operators around a decoder's matmuls.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include "decoder_ops.h"

namespace htp {

constexpr int kKvI8   = 0;  // HTP_B200_KV_I8
constexpr int kKvE4m3 = 1;  // HTP_B200_KV_E4M3

// First error wins.  The word is host memory that the device addresses: written only when something is wrong.
__device__ __forceinline__ void record_error(int *err, int code) {
  if (*reinterpret_cast<volatile int *>(err) == 0) {
    *reinterpret_cast<volatile int *>(err) = code;
  }
}

// 16 bytes of a cache: read once, so not kept in L1 (and not through the read-only path - the kernel before
// this one on the stream may have written them).
__device__ __forceinline__ uint4 ld_stream16(const void *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream8(const void *p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows and context of sequence b.  False: lengths out of their ranges.
__device__ __forceinline__ bool sequence_of(const KvView &kv, int b, int max_q, int max_ctx, int &q0, int &q_len,
                                            int &ctx) {
  q0           = kv.q_start[b];
  const int q1 = kv.q_start[b + 1];
  ctx          = kv.ctx_len[b];
  q_len        = q1 - q0;
  return q0 >= 0 && q1 >= q0 && q1 <= kv.n_rows && q_len <= max_q && ctx >= 0 && ctx <= max_ctx &&
         ctx <= (long long) kv.table_stride << kv.page_shift;
}

// How many of first(1) .. first(n) are <= at: the index of the interval [first(i), first(i + 1)) that holds
// `at`, found by the whole CTA in one pass of loads.
template <typename F>
__device__ __forceinline__ int interval_of(int n, long long at, F first) {
  int found = 0;
  for (int i = 0; i < n; i += blockDim.x) {
    const int j = i + threadIdx.x;
    found += __syncthreads_count(j < n && first(j + 1) <= at);
  }
  return found;
}

}  // namespace htp
