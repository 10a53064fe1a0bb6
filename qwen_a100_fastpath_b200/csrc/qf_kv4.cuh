// qf_kv4.cuh -- the 4-bit cache format shared by the kernels that write, read and attend it.
//
// A group is 64 consecutive dimensions of one head of one token.  With lo and hi its least and greatest value,
//   s = bf16((hi - lo) / 15),   c = bf16(lo - 16 s),   n = clamp(rint((x - c) / s), 16, 31) - 16  (0 where s = 0)
// (fp32 operations, round to nearest even) and the nibble n stands for bf16((n + 16) s + c).  The 16 in front is what makes
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
  const float s32 = __fdiv_rn(hi - lo, 15.f);
  s = __bfloat162float(__float2bfloat16_rn(s32));
  c = __bfloat162float(__float2bfloat16_rn(fmaf(-16.f, s, lo)));
  constexpr float kMax = 8.507059173023462e37f;  // 2^126
  if (!(fabsf(lo) < kMax && fabsf(hi) < kMax)) s = c = __int_as_float(0x7fffffff);
}

// The nibbles of two of a group's values, without a division: n is the whole number next to (x - c) / s by the reciprocal,
// at most one off and that only next to a border between two nibbles, and the exact remainder d - n s, d = x - c, tells on
// which side of the border d lies.  On the border itself, and where the rounding of the quotient to fp32 would put it there
// (within 2^-20 of it, half a step for quotients from 16 to 32), the even one is taken.  (Quotients are below 128: the step is
// at least 2^-13 of the largest magnitude, and c's rounding moves them by less than a hundred.)  A step of zero or NaN gives 0.
struct Kv4Coder {
  uint64_t c2, s2, inv2;  // -c, -s and 1 / s, twice each
  float s, tol;
  bool plain;
  __device__ __forceinline__ Kv4Coder(float step, float offset) {
    s = step, tol = step * 1.9073486328125e-06f;  // 2^-19
    plain = step > 1e-30f;  // reciprocal, remainders and tolerance are normal numbers
    const float inv = plain ? __frcp_rn(step) : 0.f;
    c2 = pack_f32x2(-offset, -offset), s2 = pack_f32x2(-step, -step), inv2 = pack_f32x2(inv, inv);
  }
  __device__ __forceinline__ float settle(float n, float m, float r) const {
    const float a = fmaf(2.f, fabsf(r), -s);  // > 0: nearer to the next whole number
    if (a >= -tol && (a > tol || (__float_as_int(m) & 1))) n += r < 0.f ? -1.f : 1.f;
    return n;
  }
  __device__ __forceinline__ uint32_t bits(float n) const {
    return static_cast<uint32_t>(__float_as_int(fminf(fmaxf(n, 16.f), 31.f) + kWhole)) & 15u;  // 16 -> 0, 31 -> 15
  }
  __device__ __forceinline__ uint32_t slow(float x, float offset) const {
    return s > 0.f ? bits(rintf(__fdiv_rn(x - offset, s))) : 0u;
  }
  // lo's nibble in bits 0 to 3, hi's in bits 4 to 7
  __device__ __forceinline__ uint32_t operator()(float lo, float hi) const {
    if (!plain) {
      const float offset = -unpack_f32x2(c2).x;
      return slow(lo, offset) | slow(hi, offset) << 4;
    }
    const uint64_t one = pack_f32x2(1.f, 1.f);
    uint64_t d = c2, m = pack_f32x2(kWhole, kWhole), n = pack_f32x2(-kWhole, -kWhole);
    fma_f32x2(d, pack_f32x2(lo, hi), one);
    fma_f32x2(m, d, inv2);
    fma_f32x2(n, m, one);
    uint64_t r = d;
    fma_f32x2(r, n, s2);
    const float2 nn = unpack_f32x2(n), mm = unpack_f32x2(m), rr = unpack_f32x2(r);
    return bits(settle(nn.x, mm.x, rr.x)) + 16u * bits(settle(nn.y, mm.y, rr.y));
  }
  static constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: adding it rounds to whole numbers, ties to even
};

// The word of eight values' nibbles.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], float s, float c) {
  const Kv4Coder code(s, c);
  uint32_t r = code(x[6], x[7]);
#pragma unroll
  for (int j = 4; j >= 0; j -= 2) r = 256u * r + code(x[j], x[j + 1]);
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
