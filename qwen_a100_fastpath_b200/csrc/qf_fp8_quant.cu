// qf_fp8_quant.cu -- run-time quantizer of the activations of a block-scaled fp8 layer: e4m3 values and one fp32 scale
// for each 128 elements of a token row, alone or behind the MLP's SiLU gate.
//
// Mathematics, per group of 128 consecutive k (the last group of a row may be shorter):
//   v = x[m, k], or silu(x[m, k]) * x[m, K + k] in fp32;  a = max(max |v|, 448 * 2^-60);
//   scale = a / 448;  q = e4m3(v * (448 / a)), round to nearest even (both quotients IEEE fp32).
// A NaN in a group makes its scale and values NaN; an infinity makes its scale infinite and the product NaN.
//
// Bound by memory: 2 (4 with the gate) bytes read and 1 written per element, so one pass with everything in registers.
// Eight threads share a group (16 elements, 32 contiguous bytes each), its maximum is three shuffles, nothing
// crosses a warp, and the groups of all rows form one flat index, so one row fills as many SMs as it has work for.
// Eight CTAs per SM, six with the gate: its arithmetic needs the registers, 40 with what a thread has loaded kept packed
// until it is used.  4096 x 17408 takes 34 us (6.2 TB/s), with the gate 69 us in a graph, 77 through the call (4.7 TB/s;
// five CTAs 82; neither DRAM, 56 %, nor issue, 75 %, is at its limit); one row of 5120 1.3 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/qf_b200.h"
#include "qf_fp8.cuh"
#include "qf_host.h"
#include "qf_ptx.cuh"

namespace qf {
namespace {

constexpr int kQtPer = 16;                        // elements per thread
constexpr int kQtLanes = kFp8Block / kQtPer;      // threads per group

struct QtParams {
  const __nv_bfloat16* x;
  int64_t ldx;
  uint8_t* q;
  int64_t ldq;
  float* scale;
  int64_t lds;
  int K;
  uint32_t kb;       // groups per row
  uint32_t ngroups;  // of all rows
  int vec_in, vec_out;
};

// 16 bf16 of a row from column k, packed: two 16-byte loads where the whole piece lies in the row, else one by one (zeros
// past the end, which leave the group's maximum as it is).
struct Piece {
  uint32_t w[kQtPer / 2];
};

__device__ __forceinline__ void load16(const __nv_bfloat16* row, int k, int K, bool vec, Piece& v) {
  if (vec && k + kQtPer <= K) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 u = reinterpret_cast<const uint4*>(row + k)[j];
      v.w[4 * j] = u.x, v.w[4 * j + 1] = u.y, v.w[4 * j + 2] = u.z, v.w[4 * j + 3] = u.w;
    }
  } else {
    const uint16_t* src = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int i = 0; i < kQtPer; ++i) {
      const uint32_t h = k + i < K ? src[k + i] : 0u;
      v.w[i / 2] = i % 2 ? v.w[i / 2] | (h << 16) : h;
    }
  }
}

template <bool SILU>
__global__ void __launch_bounds__(256, SILU ? 6 : 8) fp8_quantize_kernel(const QtParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t group = blockIdx.x * (blockDim.x / kQtLanes) + threadIdx.x / kQtLanes;
  if (group / (32 / kQtLanes) * (32 / kQtLanes) >= p.ngroups) return;  // a whole warp leaves or stays
  const bool live = group < p.ngroups;
  const uint32_t m = live ? group / p.kb : 0;
  const uint32_t g = live ? group - m * p.kb : 0;
  const int k = static_cast<int>(g) * kFp8Block + static_cast<int>(threadIdx.x % kQtLanes) * kQtPer;
  const __nv_bfloat16* row = p.x + static_cast<int64_t>(m) * p.ldx;
  Piece x, up;
  load16(row, k, live ? p.K : 0, p.vec_in, x);
  if (SILU) load16(row + p.K, k, live ? p.K : 0, p.vec_in, up);
  float v[kQtPer];
#pragma unroll
  for (int i = 0; i < kQtPer; i += 2) {
    v[i] = bf16_lo(x.w[i / 2]);
    v[i + 1] = bf16_hi(x.w[i / 2]);
    if (SILU) {
      const float2 s = sigmoid2(v[i], v[i + 1]);
      v[i] = v[i] * s.x * bf16_lo(up.w[i / 2]);
      v[i + 1] = v[i + 1] * s.y * bf16_hi(up.w[i / 2]);
    }
  }
  float a = kFp8AmaxFloor;
#pragma unroll
  for (int i = 0; i < kQtPer; ++i) a = max_nan(a, fabsf(v[i]));
#pragma unroll
  for (int off = 1; off < kQtLanes; off <<= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, off));
  if (!live) return;
  const float inv = __fdiv_rn(kE4m3Max, a);
  if (threadIdx.x % kQtLanes == 0) p.scale[static_cast<int64_t>(m) * p.lds + g] = __fdiv_rn(a, kE4m3Max);
  uint8_t* out = p.q + static_cast<int64_t>(m) * p.ldq + k;
  uint32_t o[kQtPer / 4];
#pragma unroll
  for (int i = 0; i < kQtPer / 4; ++i)
    o[i] = f32x4_to_e4m3x4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
  if (p.vec_out && k + kQtPer <= p.K) {
    *reinterpret_cast<uint4*>(out) = make_uint4(o[0], o[1], o[2], o[3]);
  } else {
#pragma unroll
    for (int i = 0; i < kQtPer; ++i)
      if (k + i < p.K) out[i] = static_cast<uint8_t>(o[i / 4] >> (8 * (i % 4)));
  }
}

}  // namespace
}  // namespace qf

using namespace qf;

extern "C" int qf_fp8_quantize(const void* x, int64_t ldx, int M, int K, int silu_mul, void* q, int64_t ldq,
                               float* scale, int64_t lds, unsigned flags, void* stream) {
  if (M < 0 || K < 0) return fail(QF_ERR_SHAPE, "negative size");
  if (M == 0 || K == 0) return QF_OK;
  if (K > QF_FP8_MAX_K) return fail(QF_ERR_SHAPE, "K too large");
  if (!x || !q || !scale) return fail(QF_ERR_INVALID, "null pointer");
  const int64_t kb = (K + kFp8Block - 1) / kFp8Block;
  const int64_t width = silu_mul ? 2 * static_cast<int64_t>(K) : K;
  if (M > 1 && (ldx < width || ldq < K || lds < kb)) return fail(QF_ERR_STRIDE, "row stride smaller than the row");
  if (reinterpret_cast<uintptr_t>(x) % 2 || reinterpret_cast<uintptr_t>(scale) % 4)
    return fail(QF_ERR_ALIGN, "x must be 2-byte and scale 4-byte aligned");
  if (kb * M >= (int64_t{1} << 31)) return fail(QF_ERR_SHAPE, "more than 2^31 groups");
  int rc = require_b200(nullptr, nullptr);
  if (rc) return rc;
  QtParams p = {};
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.ldx = ldx;
  p.q = static_cast<uint8_t*>(q);
  p.ldq = ldq;
  p.scale = scale;
  p.lds = lds;
  p.K = K;
  p.kb = static_cast<uint32_t>(kb);
  p.ngroups = static_cast<uint32_t>(kb * M);
  p.vec_in = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (M == 1 || ldx % 8 == 0) && (!silu_mul || K % 8 == 0);
  p.vec_out = reinterpret_cast<uintptr_t>(q) % 16 == 0 && (M == 1 || ldq % 16 == 0);
  // few groups: one-warp CTAs, so that a single token's row spreads over the SMs
  const unsigned threads = p.ngroups <= 4096 ? 32 : 256;
  const unsigned per = threads / kQtLanes;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.ngroups + per - 1) / per);
  cfg.blockDim = dim3(threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  const cudaError_t e = silu_mul ? cudaLaunchKernelEx(&cfg, fp8_quantize_kernel<true>, p)
                                 : cudaLaunchKernelEx(&cfg, fp8_quantize_kernel<false>, p);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}
