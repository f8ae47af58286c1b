// What the two attention kernels over the paged 8-bit cache share: exact conversion of codes, the two-term
// split of fp32 values, and the constants of the lagging maximum (see attn_decode.cu).
#pragma once

#include <cuda_fp16.h>

#include "decoder_common.cuh"
#include "unpack.cuh"

namespace htp {

constexpr float kLift  = 8.f;     // weights are kept times 2^8: fp16 terms of small weights stay normal numbers
constexpr float kSlack = 6.f;     // M may lag the maximum by this much: weights stay below 2^(8 + 6) < 65504
constexpr float kFloor = -1e30f;  // M before the first score
// From this M on, folding M into the product's addend (one rounding of numbers as large as M, another one for each
// block of tokens) would shift the blocks against each other by parts of a power of two: the difference to M
// is then taken from the rounded score instead, exactly.
constexpr float kHuge = 65536.f;

// Four codes (lowest byte first) as two fp16 pairs.
template <int KVT>
__device__ __forceinline__ void codes_to_h2(uint32_t w, uint32_t (&h)[2]) {
  if constexpr (KVT == kKvI8) {
    q8_0_unpack_word(w, h);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(h[0]), "=r"(h[1])
        : "r"(w));
  }
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  return h2_as_u32(__floats2half2_rn(a, b));
}

// hi + lo fp16 terms of two fp32 values
__device__ __forceinline__ void split_h2(float a, float b, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2  f = __half22float2(h);
  hi              = h2_as_u32(h);
  lo              = pack_h2(a - f.x, b - f.y);
}

// The power of two that brings a row's largest magnitude into [2^13, 2^14) - nothing overflows fp16, the
// second term keeps its bits -, as what to multiply by and what that has to be undone with.
__device__ __forceinline__ void query_unit(float amax, float &unit, float &by) {
  int e = ((__float_as_int(amax) >> 23) & 0xff) - 127 - 13;
  e     = amax == 0.f ? 0 : (e < -100 ? -100 : e);
  unit  = __int_as_float((127 + e) << 23);
  by    = __int_as_float((127 - e) << 23);
}

// What a block's scales become: factor of its scores, addend to its exponents, divisor of its weights in the
// denominator.  (The logarithm of the mantissa alone: off by 2^-22 whatever the exponent.)
__device__ __forceinline__ void block_scales(float ks, float vs, float scale_log2, float &by, float &up, float &inv) {
  const float v = vs > 0.f ? vs : 1.f;
  const int   e = (__float_as_int(v) >> 23) - 127;
  float       m;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(m) : "f"(__int_as_float((__float_as_int(v) & 0x007fffff) | 0x3f800000)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(v));
  by = (ks > 0.f ? ks : 1.f) * scale_log2;
  up = (float) e + m;
}

// Two fp32 operations of one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

}  // namespace htp
