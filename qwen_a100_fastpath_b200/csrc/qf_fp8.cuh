// qf_fp8.cuh -- device helpers of the block-scaled fp8 path: the activation quantizer's arithmetic and the e4m3 forms
// used by its kernels.
#pragma once
#include <cuda_bf16.h>

#include <cstdint>

#include "qf_ptx.cuh"

namespace qf {

constexpr int kFp8Block = 128;                   // one scale for this many elements along k (and channels of a weight)
constexpr float kE4m3Max = 448.0f;               // largest finite e4m3 value
constexpr float kFp8ScaleFloor = 8.673617379884035e-19f;  // 2^-60: the scale of an all-zero group
constexpr float kFp8AmaxFloor = kE4m3Max * kFp8ScaleFloor;

// max that keeps a NaN of either side (a group with a NaN gets a NaN scale and NaN values).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 1 / (1 + e^-x) of two values: e^-x = 2^t * 2^c with t = -x * log2(e) rounded and c what the rounding left, 2^t by the
// special-function unit (2 ulp) and 2^c = 1 + c * ln(2), then the unit's reciprocal with one Newton step: good to
// 8 * 2^-24, at some ten instructions a value (packed fp32 pairs) where expf and an IEEE quotient take some thirty.  Beyond |x| = 88.5,
// where the result is 1 or under 2^-127, x counts as that bound, which makes the latter zero; a NaN stays one.
__device__ __forceinline__ float2 sigmoid2(float a, float b) {
  const uint64_t kL = pack_f32x2(-1.44269502f, -1.44269502f);              // log2(e) = 1.44269502 + 1.92596303e-8
  const uint64_t kLLow = pack_f32x2(-1.92596303e-8f, -1.92596303e-8f);
  const uint64_t kLn2 = pack_f32x2(0.693147182f, 0.693147182f);
  const uint64_t kOne = pack_f32x2(1.f, 1.f);
  const uint64_t x = pack_f32x2(min_nan(max_nan(a, -88.5f), 88.5f), min_nan(max_nan(b, -88.5f), 88.5f));
  const uint64_t t = mul_f32x2(x, kL);
  const float2 tf = unpack_f32x2(t);
  uint64_t c = pack_f32x2(-tf.x, -tf.y);
  fma_f32x2(c, x, kL);     // exact
  fma_f32x2(c, x, kLLow);
  uint64_t f = kOne;
  fma_f32x2(f, c, kLn2);
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(tf.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(tf.y));
  uint64_t d = kOne;
  fma_f32x2(d, pack_f32x2(e.x, e.y), f);
  const float2 df = unpack_f32x2(d);
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(df.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(df.y));
  uint64_t rest = kOne, q = pack_f32x2(r.x, r.y);
  fma_f32x2(rest, pack_f32x2(-df.x, -df.y), q);  // 1 - d * r, exact
  fma_f32x2(q, q, rest);
  return unpack_f32x2(q);
}

// Two fp32 -> two e4m3 bytes (lo in bits 0-7), round to nearest even, saturated to +-448, NaN kept.
__device__ __forceinline__ uint32_t f32x2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t f32x4_to_e4m3x4(float a, float b, float c, float d) {
  return f32x2_to_e4m3x2(a, b) | (f32x2_to_e4m3x2(c, d) << 16);
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// D[16x8] += A[16x32] (row) * B[32x8] (col), e4m3 inputs, fp32 accumulators.  Thread (g, t) = (lane / 4, lane % 4)
// holds A rows g (a0, a2) and g + 8 (a1, a3), four k each (4t.. in a0 / a1 / b0, 16 + 4t.. in a2 / a3 / b1), B column
// g, and D rows g (d0, d1) and g + 8 (d2, d3), columns 2t and 2t + 1.
__device__ __forceinline__ void mma_e4m3_m16n8k32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                  uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace qf
