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

namespace qf {

constexpr int kKv4Group = QF_KV4_GROUP;

// Device copy of qf_kv4_cache with typed pointers; strides of codes in bytes, of scales in bf16 elements.
struct Kv4View {
  uint8_t* codes[2];
  __nv_bfloat16* scale[2];
  int64_t page, head, slot;
  int64_t spage, shead, sslot;
  int num_pages, page_size, heads;
};

// Checks of a caller's cache that need no device; fills the view.  QF_OK or the code recorded by fail().
int kv4_view(const qf_kv4_cache* cache, Kv4View* view);

// Step and offset of a group from its least and greatest value (any NaN among them makes both NaN).
__device__ __forceinline__ void kv4_scale(float lo, float hi, float& s, float& c) {
  const float s32 = __fdiv_rn(hi - lo, 15.f);
  s = __bfloat162float(__float2bfloat16_rn(s32));
  c = __bfloat162float(__float2bfloat16_rn(fmaf(-16.f, s, lo)));
  constexpr float kMax = 8.507059173023462e37f;  // 2^126
  if (!(fabsf(lo) < kMax && fabsf(hi) < kMax)) s = c = __int_as_float(0x7fffffff);
}

// The nibble of a value.  NaN groups keep nibble 0.
__device__ __forceinline__ uint32_t kv4_code(float x, float s, float c) {
  const float q = rintf(__fdiv_rn(x - c, s));
  return s > 0.f ? static_cast<uint32_t>(fminf(fmaxf(q, 16.f), 31.f)) - 16u : 0u;
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
