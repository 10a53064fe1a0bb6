// qf_kv4.cuh -- the 4-bit cache format shared by the kernels that write, read and attend it.
//
// A group is 64 consecutive dimensions of one head of one token.  With lo and hi its least and greatest value,
//   s = bf16((hi - lo) * (1 / 15)),   c = bf16(lo - 16 s),   n = clamp(rint((x - c) / s), 16, 31) - 16  (0 where s = 0)
// (fp32 operations, 1 / 15 as an fp32 number, round to nearest even) and the nibble n stands for bf16((n + 16) s + c).  The 16 in front is what makes
// it cheap to take apart: a nibble put into the four upper mantissa bits of the bf16 number 16 is the bf16 number n + 16, so
// that two values cost a shift, one logical operation and one packed multiply-add.  (s, c) and not (s, lo): c carries
// that 16, at the price of c's own rounding, 2^-8 |lo - 16 s|, at most s / 16 + 2^-8 |lo| beside the s / 2 of the nibble.
// A group with a NaN, an infinity or a magnitude of 2^126 or more becomes NaN as a whole (below that no step, offset or
// value of a group can overflow).
#pragma once
#include <cuda_bf16.h>

#include <cstdint>

#include "../../include/qf_b200.h"
#include "qf_ptx.cuh"

namespace qf {

constexpr int kKv4Group = QF_KV4_GROUP;

// Device copy of qf_kv4_cache; strides in bytes.
struct Kv4View {
  uint8_t* codes[2];
  uint8_t* scale[2];
  int64_t head, shead;
  uint32_t page, slot, spage, sslot;
  int num_pages, page_size, heads;
  uint32_t div_mul, div_shift;  // by the page size
  __device__ __forceinline__ int64_t codes_at(uint32_t pg, uint32_t off) const {
    return static_cast<int64_t>(static_cast<uint64_t>(pg) * page + static_cast<uint64_t>(off) * slot);
  }
  __device__ __forceinline__ int64_t scale_at(uint32_t pg, uint32_t off) const {
    return static_cast<int64_t>(static_cast<uint64_t>(pg) * spage + static_cast<uint64_t>(off) * sslot);
  }
  // Where a slot is: false if it is none of the cache's.
  __device__ __forceinline__ bool place(int64_t s, uint32_t& pg, uint32_t& off) const {
    if (static_cast<uint64_t>(s) < 0x80000000u) {
      pg = (__umulhi(static_cast<uint32_t>(s), div_mul) + static_cast<uint32_t>(s)) >> div_shift;
      off = static_cast<uint32_t>(s) - pg * static_cast<uint32_t>(page_size);
      return pg < static_cast<uint32_t>(num_pages);
    }
    pg = off = 0;
    if (s < 0 || s >= static_cast<int64_t>(num_pages) * page_size) return false;
    pg = static_cast<uint32_t>(s / page_size);
    off = static_cast<uint32_t>(s - static_cast<int64_t>(pg) * page_size);
    return true;
  }
};

// Checks of a caller's cache that need no device; fills the view.  QF_OK or the code recorded by fail().
int kv4_view(const qf_kv4_cache* cache, Kv4View* view);

// n / d = (umulhi(n, mul) + n) >> shift for n below 2^31 (Granlund and Montgomery, PLDI 1994).
inline void kv4_divisor(int d, uint32_t* mul, uint32_t* shift) {
  *shift = 0;
  while ((1ull << *shift) < static_cast<uint64_t>(d)) ++*shift;
  *mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << *shift) - static_cast<uint64_t>(d))) / static_cast<uint64_t>(d) + 1);
}

// Step and offset of a group from its least and greatest value (any NaN among them makes both NaN).
__device__ __forceinline__ void kv4_scale(float lo, float hi, float& s, float& c) {
  s = __bfloat162float(__float2bfloat16_rn((hi - lo) * (1.f / 15.f)));
  c = __bfloat162float(__float2bfloat16_rn(fmaf(-16.f, s, lo)));
  constexpr float kMax = 8.507059173023462e37f;  // 2^126
  if (!(fabsf(lo) < kMax && fabsf(hi) < kMax)) s = c = __int_as_float(0x7fffffff);
}

// The nibbles of a group's values.  The quotient (x - c) / s is the correctly rounded fp32 one of the definition, by
// Markstein's theorem (IBM J. Res. Dev. 34, 1990): with y the correctly rounded 1 / s and q = d y, the sum q + (d - q s) y in
// two fused operations rounds to d / s.  On packed pairs that is 1.5 instructions a value (a call of the division some ten).
// It needs a step whose remainders are normal numbers; smaller ones (and zero and NaN, which give 0) take the division.
struct Kv4Coder {
  float s, c, inv;
  bool plain;
  __device__ __forceinline__ Kv4Coder(float step, float offset) {
    s = step, c = offset;
    plain = step > 1e-25f;
    inv = plain ? __frcp_rn(step) : 0.f;
  }
  // Bits of 1.5 * 2^23 + the whole number next to the quotient (the sum rounds to whole numbers, ties to even), from 16 to 31.
  static constexpr float kWhole = 12582912.f;
  static constexpr int kBits = 0x4b400000;
  __device__ __forceinline__ static uint32_t clamp(float m) {
    return static_cast<uint32_t>(min(max(__float_as_int(m), kBits + 16), kBits + 31));
  }
  __device__ __forceinline__ uint32_t slow(float x) const {
    return clamp(s > 0.f ? rintf(__fdiv_rn(x - c, s)) + kWhole : kWhole);
  }
  __device__ __forceinline__ void pair(float x0, float x1, uint32_t& n0, uint32_t& n1) const {
    const uint64_t one = pack_f32x2(1.f, 1.f), y = pack_f32x2(inv, inv);
    uint64_t d = pack_f32x2(-c, -c), m = pack_f32x2(kWhole, kWhole);
    fma_f32x2(d, pack_f32x2(x0, x1), one);
    uint64_t q = mul_f32x2(d, y), r = d;
    fma_f32x2(r, q, pack_f32x2(-s, -s));
    fma_f32x2(q, r, y);
    fma_f32x2(m, q, one);
    const float2 mm = unpack_f32x2(m);
    n0 = clamp(mm.x), n1 = clamp(mm.y);
  }
};

// The word of eight values' nibbles.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], float s, float c) {
  const Kv4Coder code(s, c);
  uint32_t n[8];
  if (__builtin_expect(code.plain, 1)) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) code.pair(x[j], x[j + 1], n[j], n[j + 1]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) n[j] = code.slow(x[j]);
  }
  uint32_t r = n[7];
#pragma unroll
  for (int j = 6; j >= 0; --j) r = 16u * r + n[j];
  // (each term has kBits + 16 more than its nibble; sums of 32-bit numbers lose nothing that a difference wants back)
  return r - 0x11111111u * static_cast<uint32_t>(Kv4Coder::kBits + 16);
}

// The greatest value, and the greatest of the negated ones, of eight bf16 values in four words and of the seven neighbouring
// threads' (the lanes of `mask`, which differ in the lowest three bits): the low and the high half of one word, NaN if any is.
__device__ __forceinline__ uint32_t kv4_extremes(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t mask) {
  auto max2 = [](uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  };
  auto min2 = [](uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  };
  const uint32_t hi = max2(max2(w0, w1), max2(w2, w3)), lo = min2(min2(w0, w1), min2(w2, w3)) ^ 0x80008000u;
  uint32_t r = max2(__byte_perm(hi, lo, 0x5410), __byte_perm(hi, lo, 0x7632));
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) r = max2(r, __shfl_xor_sync(mask, r, d));
  return r;
}

// The two values of the nibbles at bits 4 k and 16 + 4 k of w, as the low and the high half of a bf16 pair.
template <int K> __device__ __forceinline__ uint32_t kv4_pair(uint32_t w, uint32_t ss, uint32_t cc) {
  uint32_t m = K == 0 ? w << 3 : w >> (4 * K - 3), r;
  // (m & 0x00780078) | 0x41804180: n + 16 in both halves
  asm("lop3.b32 %0, %1, 0x00780078, 0x41804180, 0xEA;" : "=r"(r) : "r"(m));
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(r), "r"(ss), "r"(cc));
  return r;
}

// Both halves of a (step, offset) word on their own: (s, s) and (c, c).
__device__ __forceinline__ uint32_t dup_lo(uint32_t v) { return __byte_perm(v, v, 0x1010); }
__device__ __forceinline__ uint32_t dup_hi(uint32_t v) { return __byte_perm(v, v, 0x3232); }

}  // namespace qf
