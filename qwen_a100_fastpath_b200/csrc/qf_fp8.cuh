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

// 1 / (1 + e^-x) of two values.  e^-x = 2^n * 2^f with n = -x * log2(e) rounded to a whole number and f the rest (log2(e)
// in two parts); 2^f = 1 + f * g(f), g the polynomial of degree 5 through its values at the six Chebyshev nodes of
// [-1/2, 1/2] (2^f is then 0.16 * 2^-24 off with the coefficients rounded).  The sum is formed as 2^-64 + 2^(n-64) * 2^f,
// in one rounding, so that neither it nor its reciprocal leaves the normal range before the last product; the reciprocal
// is the special-function unit's with one Newton step.
// Over all bf16 x, which is what the gates are: within 2 * 2^-24 of the value where that is a normal number (2.3 * 2^-24 for
// 1 / (1 + expf(-x))), within half a step where it is subnormal (zero from x = -104 on, expf's form from -88.7).  Above
// 40 the result is 1; a NaN stays one.  Some 11 instructions a value (packed fp32 pairs), where expf and an IEEE quotient
// take some thirty (4096 x 17408 with the gate: 76.7 us through the call, 99.6).
__device__ __forceinline__ float2 sigmoid2(float a, float b) {
  auto both = [](float v) { return pack_f32x2(v, v); };
  const uint64_t x = pack_f32x2(min_nan(max_nan(a, -105.f), 40.f), min_nan(max_nan(b, -105.f), 40.f));
  // 1.5 * 2^23 rounds a sum to whole numbers; 63 = 127 - 64 makes its low bits the exponent of 2^(n-64), n -58 to 151
  constexpr float kMagic = 12582912.f + 63.f;
  uint64_t t = both(kMagic);
  fma_f32x2(t, x, both(-1.44269502f));      // log2(e) = 1.44269502 + 1.92596303e-8
  uint64_t f = both(kMagic);
  fma_f32x2(f, t, both(-1.f));              // -n, exact
  fma_f32x2(f, x, both(-1.44269502f));
  fma_f32x2(f, x, both(-1.92596303e-8f));
  constexpr float kG[6] = {0.6931471824645996f,   0.24022650718688965f,  0.055503569543361664f,
                           0.009618083015084267f, 0.0013390863314270973f, 0.00015453163359779865f};
  uint64_t g = both(kG[5]);
#pragma unroll
  for (int i = 4; i >= 0; --i) {
    uint64_t next = both(kG[i]);
    fma_f32x2(next, g, f);
    g = next;
  }
  uint64_t p = both(1.f);
  fma_f32x2(p, g, f);
  const float2 tf = unpack_f32x2(t);
  uint64_t d = both(0x1p-64f);
  fma_f32x2(d, p,
            pack_f32x2(__uint_as_float(__float_as_uint(tf.x) << 23), __uint_as_float(__float_as_uint(tf.y) << 23)));
  const float2 df = unpack_f32x2(d);
  float2 r;  // negative, which saves negating d
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(-df.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(-df.y));
  uint64_t rest = both(1.f), q = pack_f32x2(r.x, r.y);
  fma_f32x2(rest, d, q);
  fma_f32x2(q, q, rest);
  return unpack_f32x2(mul_f32x2(q, both(-0x1p-64f)));
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
