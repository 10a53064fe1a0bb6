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
// shuffle tree and one barrier.  Where there are many rows, CTAs walk over them with the weights kept in registers
// (packed bf16, which saves reading them from L2 once per row) and the next rows arriving in shared memory.  Sixteen
// threads hold a group of 128, so the quantizer's maximum is four shuffles.
// Measured (B200): 8192 x 5120 with fp32 residual, full gate and both norms 94 us in a graph, 97..102 through the call
// (5.8..6.2 TB/s); with bf16 residual and quantized output alone 65 us (4.5 TB/s: the phases of a row, load, sum, scale and
// quantize, follow one another on the few CTAs of an SM); one row 3.3 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <mutex>
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
  int stages;  // rows ahead (kAhead)
  long long wait_clocks;  // limit of a thread's wait for a row ahead
};

__device__ int g_norm_err;  // sticky: QF_ERR_TIMEOUT once such a wait ran out (read by qf_residual_norm_status)

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

__device__ __forceinline__ float2 activate2(float a, float b, int act) {
  if (act == QF_GATE_NONE) return make_float2(a, b);
  const float2 s = sigmoid2(a, b);
  return act == QF_GATE_SIGMOID ? s : make_float2(a * s.x, b * s.y);
}

// How a kernel reads its rows.
//   kAny: element by element, for any sizes, strides and alignments;
//   kWide: 16-byte loads (H and every row stride a multiple of eight elements, every pointer 16-byte aligned);
//   kAhead: the same rows by bulk copies into shared memory, `stages` rows ahead, where a CTA walks over several rows:
//     what a thread could hold of the next row in registers is too little in flight (8192 x 5120 with fp32 residual and
//     gate: 157 us with the next row in registers).
enum RowMode { kAny, kWide, kAhead };

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo(w[i]);
    v[2 * i + 1] = bf16_hi(w[i]);
  }
}

constexpr long long kRowWaitClocks = 8000000000ll;  // about 4 s
constexpr int kMaxRowStages = 4;
constexpr long long kNormSmem = 226 * 1024;  // shared memory of an SM, of which a CTA takes this for itself:
constexpr long long kNormFixed = 1792;      // the system's KiB and the static arrays
// What a CTA has for the rows ahead with `per_sm` of them on an SM.
constexpr long long norm_ring(int per_sm) { return kNormSmem / per_sm - kNormFixed; }

// R32: the residual is fp32.  QUANT: h leaves as e4m3 groups.
template <int C, int MAX_T, int MODE, bool R32, bool QUANT>
__global__ void __launch_bounds__(MAX_T, MAX_T == 512 ? 1 : C == 1 ? 3 : 2) residual_norm_kernel(const NormParams p) {
  constexpr bool VEC = MODE != kAny;
  __shared__ float red[2][2][32];
  __shared__ uint64_t full[kMaxRowStages];
  extern __shared__ __align__(128) uint8_t ring[];
  pdl_launch_dependents();
  const int T = blockDim.x;
  const bool gate_row = p.gate && p.gate_sh;  // a gate value for each element, not one for the row
  const int off_r = 2 * p.H, off_g = off_r + (p.residual ? (R32 ? 4 : 2) * p.H : 0);
  const int stage_bytes = off_g + (gate_row ? 2 * p.H : 0);
  if (MODE == kAhead) {
    if (threadIdx.x == 0) {
      for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1);
      fence_mbar_init();
    }
    __syncthreads();
  }
  pdl_wait();
  auto copy_row = [&](long long m, int s) {  // by one thread
    uint8_t* dst = ring + s * stage_bytes;
    mbar_arrive_expect_tx(&full[s], stage_bytes);
    bulk_load(dst, p.x + m * p.ldx, 2 * p.H, &full[s]);
    if (p.residual)
      bulk_load(dst + off_r, static_cast<const uint8_t*>(p.residual) + m * p.ldr * (R32 ? 4 : 2),
                off_g - off_r, &full[s]);
    if (gate_row) bulk_load(dst + off_g, p.gate + m * p.gate_sm, 2 * p.H, &full[s]);
  };
  if (MODE == kAhead && threadIdx.x == 0)
    for (int s = 0; s < p.stages; ++s)
      if (const long long m = blockIdx.x + static_cast<long long>(s) * gridDim.x; m < p.M) copy_row(m, s);
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
  int parity = 0, stage = 0;
  uint32_t phase = 0;
  int left_at = -1;  // kAhead: the row at which this thread left the ring
  // unsigned: below 2^31 rows and CTAs, the step past the last row stays within 32 bits (a signed index would not)
  for (uint32_t m = blockIdx.x; m < static_cast<uint32_t>(p.M); m += gridDim.x, parity ^= 1) {
    // where this row's operands are: in the ring, or in global memory
    const __nv_bfloat16* x = p.x + static_cast<int64_t>(m) * p.ldx;
    const uint8_t* res = static_cast<const uint8_t*>(p.residual);
    if (p.residual) res += static_cast<int64_t>(m) * p.ldr * (R32 ? 4 : 2);
    const __nv_bfloat16* gate = p.gate + (p.gate ? static_cast<int64_t>(m) * p.gate_sm : 0);
    if (MODE == kAhead && left_at < 0) {
      // A thread whose wait runs out leaves the ring for good and reads this and all later rows from global memory (no
      // thread but itself writes the elements it reads): the phases of a barrier that it has not seen complete would no
      // longer tell it anything.  The others go on: a stage is only filled again by thread 0, after it saw the stage's last
      // copy arrive, so what they wait for is that copy or one that is never issued.
      bool have = p.wait_clocks ? mbar_try_wait(&full[stage], phase)   // which may suspend the thread for a while
                                : mbar_test_wait(&full[stage], phase);
      if (!have)
        for (const long long t0 = clock64(); !have && clock64() - t0 < p.wait_clocks;)
          have = mbar_try_wait(&full[stage], phase);
      if (have) {
        const uint8_t* src = ring + stage * stage_bytes;
        x = reinterpret_cast<const __nv_bfloat16*>(src);
        res = src + off_r;
        if (gate_row) gate = reinterpret_cast<const __nv_bfloat16*>(src + off_g);
      } else {
        left_at = static_cast<int>(m);
        atomicExch(&g_norm_err, QF_ERR_TIMEOUT);
      }
    }
    float v[C][8], r[C][8];
    uint4 g4[C];
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * T + static_cast<int>(threadIdx.x)) * 8;
      load8_bf16<VEC>(x + e, p.H - e, v[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(v[c][i], v[c][i], s), r[c][i] = 0.f;
      if (MODE == kWide) {  // everything of the row on its way at once
        if (p.residual) {
          if (R32)
            load8_f32<true>(reinterpret_cast<const float*>(res) + e, p.H - e, r[c]);
          else
            load8_bf16<true>(reinterpret_cast<const __nv_bfloat16*>(res) + e, p.H - e, r[c]);
        }
        g4[c] = make_uint4(0, 0, 0, 0);
        if (gate_row && e < p.H) g4[c] = *reinterpret_cast<const uint4*>(gate + e);
      }
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
    float row_gate = 1.f;
    if (p.gate && !p.gate_sh) {
      const float g = __bfloat162float(*gate);
      row_gate = activate2(g, g, p.act).x;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int e = (c * T + static_cast<int>(threadIdx.x)) * 8;
      if (gate_row) {
        float g[8];
        if (MODE == kWide)
          unpack8(g4[c], g);
        else
          load8_bf16<VEC>(gate + e, p.H - e, g);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float2 a = activate2(g[i], g[i + 1], p.act);
          v[c][i] *= a.x;
          v[c][i + 1] *= a.y;
        }
      } else if (p.gate) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] *= row_gate;
      }
      if (MODE != kWide && p.residual) {
        if (R32)
          load8_f32<VEC>(reinterpret_cast<const float*>(res) + e, p.H - e, r[c]);
        else
          load8_bf16<VEC>(reinterpret_cast<const __nv_bfloat16*>(res) + e, p.H - e, r[c]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[c][i] = fmaf(p.alpha, v[c][i], r[c][i]);
        // elements past the row must not enter the sum (a gate of infinity there would not be zero times x); with wide
        // loads a piece is in the row or not as a whole
        if ((VEC ? e : e + i) < p.H) s = fmaf(v[c][i], v[c][i], s);
      }
      if (p.residual_out) {
        if (R32)
          store8_f32<VEC>(static_cast<float*>(p.residual_out) + static_cast<int64_t>(m) * p.ldro + e, p.H - e, v[c]);
        else
          store8_bf16<VEC>(static_cast<__nv_bfloat16*>(p.residual_out) + static_cast<int64_t>(m) * p.ldro + e, p.H - e,
                           v[c]);
      }
    }
    float n = 0.f;
    if (p.pre)
      n = rsqrtf(fmaf(cta_sum(s, red[parity][1]), inv_h, p.eps));
    else if (MODE == kAhead)
      __syncthreads();
    if (MODE == kAhead && left_at < 0) {
      // behind that barrier every thread has read the stage
      const long long next = m + static_cast<long long>(p.stages) * gridDim.x;
      if (threadIdx.x == 0 && next < p.M) copy_row(next, stage);
      if (++stage == p.stages) stage = 0, phase ^= 1;
    }
    if (!p.pre) continue;
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
      for (int i = 0; i < 8; ++i)
        if ((VEC ? e : e + i) < p.H) a = max_nan(a, fabsf(v[c][i]));
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
  if (MODE == kAhead && threadIdx.x == 0 && left_at >= 0) {
    // the copies still under way land before the shared memory is given up: those of the rows from left_at on for which
    // there was a stage
    for (int s = 0; s < p.stages && left_at + static_cast<long long>(s) * gridDim.x < p.M; ++s) {
      const long long t0 = clock64();
      while (!mbar_try_wait(&full[stage], phase) && clock64() - t0 < kRowWaitClocks) {
      }
      if (++stage == p.stages) stage = 0, phase ^= 1;
    }
  }
}

// Launches one instance: with several rows to a CTA and rows that bulk copies take, as kAhead.
template <int C, int MAX_T, bool R32, bool QUANT>
cudaError_t launch_norm(NormParams p, bool vec, int threads, int dev, int sms, bool pdl, cudaStream_t st) {
  // resident CTAs per SM by registers, asked once per CTA size
  static std::mutex mu;
  static int resident[64][17] = {};
  int per_sm;
  {
    std::lock_guard<std::mutex> lk(mu);
    int& known = resident[dev][threads / 32];
    if (known == 0) {
      cudaError_t e = cudaFuncSetAttribute(residual_norm_kernel<C, MAX_T, kAhead, R32, QUANT>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(norm_ring(1)));
      if (e == cudaSuccess)
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&known, residual_norm_kernel<C, MAX_T, kAhead, R32, QUANT>,
                                                          threads, 0);
      if (e != cudaSuccess) {
        known = 0;
        return e;
      }
      if (known > 16) known = 16;
      if (known < 1) known = 1;
    }
    per_sm = known;
  }
  const int per_element = 2 + (p.residual ? (R32 ? 4 : 2) : 0) + (p.gate && p.gate_sh ? 2 : 0);
  const long long bytes = static_cast<long long>(p.H) * per_element;
  while (per_sm > 1 && norm_ring(per_sm) / bytes < 2) --per_sm;
  p.stages = static_cast<int>(norm_ring(per_sm) / bytes < kMaxRowStages ? norm_ring(per_sm) / bytes : kMaxRowStages);
  const bool ahead = vec && p.stages >= 2 && p.M > 2 * sms * per_sm;
  const long long grid = static_cast<long long>(sms) * per_sm;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.M < grid || !ahead ? p.M : grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = ahead ? static_cast<size_t>(p.stages * bytes) : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  if (ahead) return cudaLaunchKernelEx(&cfg, residual_norm_kernel<C, MAX_T, kAhead, R32, QUANT>, p);
  return vec ? cudaLaunchKernelEx(&cfg, residual_norm_kernel<C, MAX_T, kWide, R32, QUANT>, p)
             : cudaLaunchKernelEx(&cfg, residual_norm_kernel<C, MAX_T, kAny, R32, QUANT>, p);
}

template <int C, int MAX_T>
cudaError_t launch_norm(const NormParams& p, bool r32, bool quant, bool vec, int threads, int dev, int sms, bool pdl,
                        cudaStream_t st) {
  if (r32) return quant ? launch_norm<C, MAX_T, true, true>(p, vec, threads, dev, sms, pdl, st)
                        : launch_norm<C, MAX_T, true, false>(p, vec, threads, dev, sms, pdl, st);
  return quant ? launch_norm<C, MAX_T, false, true>(p, vec, threads, dev, sms, pdl, st)
               : launch_norm<C, MAX_T, false, false>(p, vec, threads, dev, sms, pdl, st);
}

// Limit of a wait for a row ahead.  QF_NORM_WAIT_CLOCKS (read only with QF_TEST_OVERRIDES=1, once per process) replaces
// it: with 0 the tests run the path of a wait that ran out.
long long row_wait_clocks() {
  static const long long v = [] {
    const char* t = std::getenv("QF_TEST_OVERRIDES");
    const char* e = std::getenv("QF_NORM_WAIT_CLOCKS");
    return t && std::strcmp(t, "1") == 0 && e ? std::atoll(e) : kRowWaitClocks;
  }();
  return v;
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
  int dev = 0, sms = 0;
  int rc = require_b200(&dev, &sms);
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
  p.wait_clocks = row_wait_clocks();
  auto rows16 = [&](const void* ptr, int64_t ld) { return !ptr || (aligned(ptr, 16) && (M == 1 || ld % 8 == 0)); };
  const bool vec = H % 8 == 0 && rows16(x, ldx) && rows16(residual, ldr) && rows16(residual_out, ldro) &&
                   rows16(out, ldo) && (!gate || gate_sh == 0 || rows16(gate, gate_sm)) && aligned(post_weight, 16) &&
                   aligned(pre_weight, 16);
  // pieces per thread: the fewest that keep the CTA at 320 threads, so that two are resident and one works while the
  // other is at a barrier; wider rows, of which shared memory holds too few for two CTAs anyway, take up to 512 threads
  // (4096 x 8192, fp32 residual and gate: 84 us with two pieces on 512 threads, 116 with four on 256)
  const int pieces = (H + 7) / 8;
  const int C = pieces <= 320 ? 1 : pieces <= 1024 ? 2 : 4;
  const int threads = ((pieces + C - 1) / C + 31) / 32 * 32;
  const bool pdl = (flags & QF_FLAG_PDL) != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (C == 1)
    e = launch_norm<1, 320>(p, r32, quant, vec, threads, dev, sms, pdl, st);
  else if (C == 2)
    e = threads <= 320 ? launch_norm<2, 320>(p, r32, quant, vec, threads, dev, sms, pdl, st)
                       : launch_norm<2, 512>(p, r32, quant, vec, threads, dev, sms, pdl, st);
  else
    e = launch_norm<4, 512>(p, r32, quant, vec, threads, dev, sms, pdl, st);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}

extern "C" int qf_residual_norm_status(void* stream, int* status) {
  return read_error_word(&g_norm_err, stream, status);
}
