// qf_norm.cu -- the residual update between two blocks of a decoder layer with the norms on both sides of it, in one
// pass over a token row.
//
// Mathematics, per token row of H elements, all in fp32:
//   u = x, or x * rsqrt(mean(x^2) + eps) * (post_weight + offset)      (the norm after the block)
//   v = u * act(gate), act one of 1 / identity / sigmoid / silu         (the block's gate)
//   r' = residual + alpha * v                                           (stored, rounded to the residual's type)
//   h = r' * rsqrt(mean(r'^2) + eps) * (pre_weight + offset)            (the norm before the next block; r' unrounded)
//   h stored as bf16, or quantized in groups of 128 as qf_fp8_quant.cu does (h unrounded in between).
//
// Bound by memory for many rows and by two block-wide sums for one.  A CTA takes a row, a thread C pieces of eight
// consecutive elements, everything stays in registers between the loads and the stores, and each sum is one
// shuffle tree and one barrier.  CTAs walk the rows with the weights kept in registers (packed bf16), which saves
// reading them from L2 once per row.  Sixteen threads hold a group of 128, so the quantizer's maximum is four shuffles.
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

struct NormParams {
  const __nv_bfloat16* x;
  int64_t ldx;
  const void* residual;   // null: zeros
  int64_t ldr;
  const __nv_bfloat16* gate;  // null: none; element (m, h) at m * gate_sm + h * gate_sh
  int64_t gate_sm, gate_sh;
  const __nv_bfloat16* post;  // null: no norm after the block
  const __nv_bfloat16* pre;   // null: no h
  void* residual_out;         // null: not stored
  int64_t ldro;
  void* out;
  int64_t ldo;
  float* scale;
  int64_t lds;
  float alpha, eps, offset;
  int act;
  int M, H;
};

// Sum over the CTA, the same order on every thread: shuffle tree, then the warps' sums one after the other.
__device__ __forceinline__ float cta_sum(float s, float* red) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.f;
  const int nw = blockDim.x >> 5;
  for (int i = 0; i < nw; ++i) s += red[i];
  return s;
}

template <bool VEC> __device__ __forceinline__ void load8_bf16(const __nv_bfloat16* src, int n, float (&v)[8]) {
  if (VEC) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (n >= 8) u = *reinterpret_cast<const uint4*>(src);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16_lo(w[i]);
      v[2 * i + 1] = bf16_hi(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? __bfloat162float(src[i]) : 0.f;
  }
}

template <bool VEC> __device__ __forceinline__ void load8_f32(const float* src, int n, float (&v)[8]) {
  if (VEC) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (n >= 8) {
      a = reinterpret_cast<const float4*>(src)[0];
      b = reinterpret_cast<const float4*>(src)[1];
    }
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? src[i] : 0.f;
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return reinterpret_cast<const uint32_t&>(h);
}

template <bool VEC> __device__ __forceinline__ void store8_bf16(__nv_bfloat16* dst, int n, const float (&v)[8]) {
  if (VEC) {
    if (n >= 8)
      *reinterpret_cast<uint4*>(dst) =
          make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) dst[i] = __float2bfloat16_rn(v[i]);
  }
}

template <bool VEC> __device__ __forceinline__ void store8_f32(float* dst, int n, const float (&v)[8]) {
  if (VEC) {
    if (n >= 8) {
      reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) dst[i] = v[i];
  }
}

__device__ __forceinline__ float activate(float g, int act) {
  if (act == QF_GATE_NONE) return g;
  const float s = __fdiv_rn(1.f, 1.f + expf(-g));
  return act == QF_GATE_SIGMOID ? s : g * s;
}

// VEC: H and every row stride a multiple of eight elements and every pointer 16-byte aligned, so that a piece is whole
// or absent and moves in 16-byte accesses.  R32: the residual is fp32.  QUANT: h leaves as e4m3 groups.
template <int C, bool VEC, bool R32, bool QUANT>
__global__ void __launch_bounds__(512) residual_norm_kernel(const NormParams p) {
  __shared__ float red[2][2][32];
  pdl_launch_dependents();
  pdl_wait();
  const int T = blockDim.x;
  uint32_t wpost[C][4], wpre[C][4];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int e = (c * T + static_cast<int>(threadIdx.x)) * 8;
    float t[8] = {};
    if (p.post) load8_bf16<VEC>(p.post + e, p.H - e, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) wpost[c][i] = pack_bf16(t[2 * i], t[2 * i + 1]);
    if (p.pre) load8_bf16<VEC>(p.pre + e, p.H - e, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) wpre[c][i] = pack_bf16(t[2 * i], t[2 * i + 1]);
  }
  const float inv_h = 1.f / static_cast<float>(p.H);
  int parity = 0;
  for (int m = blockIdx.x; m < p.M; m += gridDim.x, parity ^= 1) {
    float v[C][8];
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * T + static_cast<int>(threadIdx.x)) * 8;
      load8_bf16<VEC>(p.x + static_cast<int64_t>(m) * p.ldx + e, p.H - e, v[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(v[c][i], v[c][i], s);
    }
    if (p.post) {
      const float n = rsqrtf(fmaf(cta_sum(s, red[parity][0]), inv_h, p.eps));
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[c][2 * i] *= n * (bf16_lo(wpost[c][i]) + p.offset);
          v[c][2 * i + 1] *= n * (bf16_hi(wpost[c][i]) + p.offset);
        }
    }
    s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * T + static_cast<int>(threadIdx.x)) * 8;
      if (p.gate) {
        float g[8];
        const __nv_bfloat16* src = p.gate + static_cast<int64_t>(m) * p.gate_sm;
        if (p.gate_sh) {
          load8_bf16<VEC>(src + e, p.H - e, g);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] *= activate(g[i], p.act);
        } else {
          const float a = activate(__bfloat162float(*src), p.act);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] *= a;
        }
      }
      float r[8] = {};
      if (p.residual) {
        if (R32)
          load8_f32<VEC>(static_cast<const float*>(p.residual) + static_cast<int64_t>(m) * p.ldr + e, p.H - e, r);
        else
          load8_bf16<VEC>(static_cast<const __nv_bfloat16*>(p.residual) + static_cast<int64_t>(m) * p.ldr + e, p.H - e,
                          r);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[c][i] = fmaf(p.alpha, v[c][i], r[i]);
        // elements past the row must not enter the sum (a gate of infinity there would not be zero times x)
        if (e + i >= p.H) v[c][i] = 0.f;
        s = fmaf(v[c][i], v[c][i], s);
      }
      if (p.residual_out) {
        if (R32)
          store8_f32<VEC>(static_cast<float*>(p.residual_out) + static_cast<int64_t>(m) * p.ldro + e, p.H - e, v[c]);
        else
          store8_bf16<VEC>(static_cast<__nv_bfloat16*>(p.residual_out) + static_cast<int64_t>(m) * p.ldro + e, p.H - e,
                           v[c]);
      }
    }
    if (!p.pre) continue;
    const float n = rsqrtf(fmaf(cta_sum(s, red[parity][1]), inv_h, p.eps));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * T + static_cast<int>(threadIdx.x)) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[c][2 * i] *= n * (bf16_lo(wpre[c][i]) + p.offset);
        v[c][2 * i + 1] *= n * (bf16_hi(wpre[c][i]) + p.offset);
      }
      if (!QUANT) {
        store8_bf16<VEC>(static_cast<__nv_bfloat16*>(p.out) + static_cast<int64_t>(m) * p.ldo + e, p.H - e, v[c]);
        continue;
      }
      float a = kFp8AmaxFloor;
#pragma unroll
      for (int i = 0; i < 8; ++i) a = max_nan(a, e + i < p.H ? fabsf(v[c][i]) : 0.f);
#pragma unroll
      for (int off = 1; off < kFp8Block / 8; off <<= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, off));
      const float inv = __fdiv_rn(kE4m3Max, a);
      if (e < p.H && e % kFp8Block == 0)
        p.scale[static_cast<int64_t>(m) * p.lds + e / kFp8Block] = __fdiv_rn(a, kE4m3Max);
      const uint32_t lo = f32x4_to_e4m3x4(v[c][0] * inv, v[c][1] * inv, v[c][2] * inv, v[c][3] * inv);
      const uint32_t hi = f32x4_to_e4m3x4(v[c][4] * inv, v[c][5] * inv, v[c][6] * inv, v[c][7] * inv);
      uint8_t* dst = static_cast<uint8_t*>(p.out) + static_cast<int64_t>(m) * p.ldo + e;
      if (VEC) {
        if (e + 8 <= p.H) *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i < p.H) dst[i] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i % 4)));
      }
    }
  }
}

template <int C, bool VEC> cudaError_t launch_norm(const cudaLaunchConfig_t& cfg, const NormParams& p, bool r32, bool quant) {
  if (r32) return quant ? cudaLaunchKernelEx(&cfg, residual_norm_kernel<C, VEC, true, true>, p)
                        : cudaLaunchKernelEx(&cfg, residual_norm_kernel<C, VEC, true, false>, p);
  return quant ? cudaLaunchKernelEx(&cfg, residual_norm_kernel<C, VEC, false, true>, p)
               : cudaLaunchKernelEx(&cfg, residual_norm_kernel<C, VEC, false, false>, p);
}

bool aligned(const void* ptr, size_t n) { return reinterpret_cast<uintptr_t>(ptr) % n == 0; }

}  // namespace
}  // namespace qf

using namespace qf;

extern "C" int qf_residual_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, int residual_dtype,
                                const void* gate, int64_t gate_sm, int64_t gate_sh, int gate_act, const void* post_weight,
                                const void* pre_weight, float weight_offset, float residual_scale, float eps,
                                void* residual_out, int64_t ldro, void* out, int64_t ldo, float* out_scale, int64_t lds,
                                int M, int H, unsigned flags, void* stream) {
  if (M < 0 || H < 0) return fail(QF_ERR_SHAPE, "negative size");
  if (H > QF_NORM_MAX_H) return fail(QF_ERR_SHAPE, "rows wider than 16384 elements");
  if (residual_dtype != QF_DTYPE_BF16 && residual_dtype != QF_DTYPE_F32)
    return fail(QF_ERR_DTYPE, "residual must be bf16 or fp32");
  if (gate_act < QF_GATE_NONE || gate_act > QF_GATE_SILU) return fail(QF_ERR_INVALID, "unknown gate activation");
  if (!(eps >= 0.f) || eps > 3.4e38f) return fail(QF_ERR_INVALID, "eps must be finite and >= 0");
  if (M == 0 || H == 0) return QF_OK;
  const bool quant = out_scale != nullptr;
  const bool r32 = residual_dtype == QF_DTYPE_F32;
  if (!x || (!out && !residual_out) || (!pre_weight) != (!out) || (quant && !out))
    return fail(QF_ERR_INVALID, "null pointer (out goes with pre_weight; one of out and residual_out is needed)");
  if (gate && gate_sh != 0 && gate_sh != 1) return fail(QF_ERR_STRIDE, "the gate's column stride must be 0 or 1");
  if (M > 1 && (ldx < H || (residual && ldr < H) || (residual_out && ldro < H) || (out && ldo < H) ||
                (quant && lds < (H + kFp8Block - 1) / kFp8Block)))
    return fail(QF_ERR_STRIDE, "row stride smaller than the row");
  if (gate && gate_sm < 0) return fail(QF_ERR_STRIDE, "negative gate stride");
  const size_t rb = r32 ? 4 : 2;
  if (!aligned(x, 2) || !aligned(residual, rb) || !aligned(residual_out, rb) || !aligned(gate, 2) ||
      !aligned(post_weight, 2) || !aligned(pre_weight, 2) || (!quant && !aligned(out, 2)) || !aligned(out_scale, 4))
    return fail(QF_ERR_ALIGN, "pointers must be aligned to their element");
  int sms = 0;
  int rc = require_b200(nullptr, &sms);
  if (rc) return rc;
  NormParams p = {};
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.ldx = ldx;
  p.residual = residual;
  p.ldr = ldr;
  p.gate = static_cast<const __nv_bfloat16*>(gate);
  p.gate_sm = gate_sm;
  p.gate_sh = gate_sh;
  p.post = static_cast<const __nv_bfloat16*>(post_weight);
  p.pre = static_cast<const __nv_bfloat16*>(pre_weight);
  p.residual_out = residual_out;
  p.ldro = ldro;
  p.out = out;
  p.ldo = ldo;
  p.scale = out_scale;
  p.lds = lds;
  p.alpha = residual_scale;
  p.eps = eps;
  p.offset = weight_offset;
  p.act = gate_act;
  p.M = M;
  p.H = H;
  auto rows16 = [&](const void* ptr, int64_t ld) { return !ptr || (aligned(ptr, 16) && (M == 1 || ld % 8 == 0)); };
  const bool vec = H % 8 == 0 && rows16(x, ldx) && rows16(residual, ldr) && rows16(residual_out, ldro) &&
                   rows16(out, ldo) && (!gate || gate_sh == 0 || rows16(gate, gate_sm)) && aligned(post_weight, 16) &&
                   aligned(pre_weight, 16);
  // pieces per thread: the fewest that keep the CTA at 512 threads
  const int pieces = (H + 7) / 8;
  const int C = pieces <= 512 ? 1 : pieces <= 1024 ? 2 : 4;
  const int threads = ((pieces + C - 1) / C + 31) / 32 * 32;
  const int per_sm = 2048 / threads < 1 ? 1 : (2048 / threads > 8 ? 8 : 2048 / threads);
  const long long grid = static_cast<long long>(sms) * per_sm;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(M < grid ? M : grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  cudaError_t e;
  if (vec)
    e = C == 1 ? launch_norm<1, true>(cfg, p, r32, quant) : C == 2 ? launch_norm<2, true>(cfg, p, r32, quant)
                                                                    : launch_norm<4, true>(cfg, p, r32, quant);
  else
    e = C == 1 ? launch_norm<1, false>(cfg, p, r32, quant) : C == 2 ? launch_norm<2, false>(cfg, p, r32, quant)
                                                                    : launch_norm<4, false>(cfg, p, r32, quant);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}
