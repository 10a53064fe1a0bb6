// qf_rope.cu -- norms of queries and keys for each head with the position rotation in the same pass, and optionally the
// keys and values straight into the 4-bit cache.
//
// Mathematics, per token and head (a row of D values x), fp32 inside:
//   y = x, or x * rsqrt(mean(x^2) + eps) * (weight + offset)
//   the first R values turn by the token's angles: with (cos_i, sin_i) = the table's row of the token's position,
//   a = y[i], b = y[i + R / 2] (or y[2 i], y[2 i + 1]):  a' = a cos_i - b sin_i,  b' = b cos_i + a sin_i
//   the result is rounded to bf16 once; a key that goes into the cache is quantized from those bf16 values.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/qf_b200.h"
#include "qf_fp8.cuh"
#include "qf_host.h"
#include "qf_kv4.cuh"
#include "qf_ptx.cuh"

namespace qf {
namespace {

struct RopeParams {
  const __nv_bfloat16* x[3];  // queries, keys, values (values only with a cache)
  int64_t xt[3], xh[3];
  const __nv_bfloat16* weight[2];  // null: no norm
  __nv_bfloat16* out[2];           // out[1] null: keys go to the cache
  int64_t ot[2], oh[2];
  const int64_t* positions;
  const void* cos_sin;  // null: no rotation
  int64_t cs_row;
  int64_t max_pos;
  const int64_t* slots;
  Kv4View cache;
  float offset, eps, inv_d;
  int heads[2];
  int D, rot;
  int rows;       // of a token
  uint32_t total;  // rows of all tokens
  int cs_f32, interleaved;
};

constexpr int kRopeWarps = 4;

__global__ void __launch_bounds__(kRopeWarps * 32) rope_any_kernel(const RopeParams p) {
  __shared__ float row_buf[kRopeWarps][QF_ROPE_MAX_D];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  float* buf = row_buf[threadIdx.x >> 5];
  const uint32_t row = blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
  if (row >= p.total) return;
  const int64_t token = row / p.rows;
  int head = row % p.rows, side = 0;
  if (head >= p.heads[0]) head -= p.heads[0], side = 1;
  if (side == 1 && head >= p.heads[1]) head -= p.heads[1], side = 2;
  const __nv_bfloat16* x = p.x[side] + token * p.xt[side] + head * p.xh[side];
  float sum = 0.f;
  for (int e = lane; e < p.D; e += 32) {
    const float v = __bfloat162float(x[e]);
    buf[e] = v;
    sum = fmaf(v, v, sum);
  }
  if (side < 2 && p.weight[side]) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const float n = rsqrtf(fmaf(sum, p.inv_d, p.eps));
    for (int e = lane; e < p.D; e += 32) buf[e] *= n * (__bfloat162float(p.weight[side][e]) + p.offset);
  }
  __syncwarp();
  if (side < 2 && p.cos_sin) {
    const int half = p.rot / 2;
    const int64_t pos = p.positions[token];
    const bool known = pos >= 0 && pos < p.max_pos;
    for (int i = lane; i < half; i += 32) {
      float c = __int_as_float(0x7fffffff), s = c;
      if (known) {
        const int64_t at = pos * p.cs_row + i;
        if (p.cs_f32) {
          c = static_cast<const float*>(p.cos_sin)[at], s = static_cast<const float*>(p.cos_sin)[at + half];
        } else {
          c = __bfloat162float(static_cast<const __nv_bfloat16*>(p.cos_sin)[at]);
          s = __bfloat162float(static_cast<const __nv_bfloat16*>(p.cos_sin)[at + half]);
        }
      }
      const int ia = p.interleaved ? 2 * i : i, ib = p.interleaved ? 2 * i + 1 : i + half;
      const float a = buf[ia], b = buf[ib];
      buf[ia] = a * c - b * s;
      buf[ib] = b * c + a * s;
    }
    __syncwarp();
  }
  if (side < 2 && p.out[side]) {
    __nv_bfloat16* o = p.out[side] + token * p.ot[side] + head * p.oh[side];
    for (int e = lane; e < p.D; e += 32) o[e] = __float2bfloat16_rn(buf[e]);
    return;
  }
  const int64_t slot = p.slots[token];
  if (slot < 0) return;
  const int64_t page = slot / p.cache.page_size, off = slot % p.cache.page_size;
  if (page >= p.cache.num_pages) return;
  const Kv4View& v = p.cache;
  const int kv = side - 1;
  uint8_t* codes = v.codes[kv] + page * v.page + head * v.head + off * v.slot;
  __nv_bfloat16* scale = v.scale[kv] + page * v.spage + head * v.shead + off * v.sslot;
  for (int g = 0; g < p.D / kKv4Group; ++g) {
    const float a = __bfloat162float(__float2bfloat16_rn(buf[g * kKv4Group + 2 * lane]));
    const float b = __bfloat162float(__float2bfloat16_rn(buf[g * kKv4Group + 2 * lane + 1]));
    float hi = max_nan(a, b), lo = max_nan(-a, -b);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      lo = max_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    float s, c;
    kv4_scale(-lo, hi, s, c);
    codes[g * (kKv4Group / 2) + lane] = static_cast<uint8_t>(kv4_code(a, s, c) | kv4_code(b, s, c) << 4);
    if (lane == 0) reinterpret_cast<__nv_bfloat162*>(scale)[g] = __floats2bfloat162_rn(s, c);
  }
}

bool aligned(const void* ptr, size_t n) { return reinterpret_cast<uintptr_t>(ptr) % n == 0; }

}  // namespace
}  // namespace qf

using namespace qf;

extern "C" int qf_qk_norm_rope(const void* q, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_t, int64_t sk_h,
                               const void* q_weight, const void* k_weight, float weight_offset, float eps,
                               const int64_t* positions, const void* cos_sin, int64_t s_cs, int cos_sin_dtype,
                               int64_t max_positions, int rot, int interleaved, void* q_out, int64_t so_t, int64_t so_h,
                               void* k_out, int64_t sp_t, int64_t sp_h, const void* v, int64_t sv_t, int64_t sv_h,
                               const int64_t* slots, const qf_kv4_cache* cache, int tokens, int num_heads,
                               int num_kv_heads, int head_size, unsigned flags, void* stream) {
  if (tokens < 0 || num_heads < 0 || num_kv_heads < 0 || head_size < 1) return fail(QF_ERR_SHAPE, "sizes");
  if (head_size > QF_ROPE_MAX_D) return fail(QF_ERR_SHAPE, "heads wider than 512");
  if (!(eps >= 0.f) || eps > 3.4e38f) return fail(QF_ERR_INVALID, "eps must be finite and >= 0");
  if (cos_sin_dtype != QF_DTYPE_BF16 && cos_sin_dtype != QF_DTYPE_F32)
    return fail(QF_ERR_DTYPE, "the table of angles must be bf16 or fp32");
  if (rot < 0 || rot % 2 || rot > head_size) return fail(QF_ERR_SHAPE, "the rotated part must be even and within the head");
  if (max_positions < 0) return fail(QF_ERR_SHAPE, "negative size");
  const int64_t rows = num_heads + static_cast<int64_t>(num_kv_heads) * (cache ? 2 : 1);
  if (rows * tokens > INT32_MAX) return fail(QF_ERR_SHAPE, "more than 2^31 - 1 rows");
  const int64_t st[] = {sq_t, sq_h, sk_t, sk_h, so_t, so_h, sp_t, sp_h, sv_t, sv_h, s_cs};
  for (int64_t s : st)
    if (s < 0) return fail(QF_ERR_STRIDE, "negative stride");
  RopeParams p = {};
  if (cache) {
    const int rc = kv4_view(cache, &p.cache);
    if (rc) return rc;
    if (cache->num_heads != num_kv_heads || cache->head_size != head_size)
      return fail(QF_ERR_SHAPE, "the cache has other heads");
  }
  if (rows * tokens == 0) return QF_OK;
  if ((num_heads && (!q || !q_out)) || (num_kv_heads && !k) || (rot && (!positions || (max_positions && !cos_sin))) ||
      (cache ? !v || !slots || k_out : num_kv_heads && !k_out))
    return fail(QF_ERR_INVALID, "null pointer (a cache comes with v and slots and without k_out)");
  const void* two[] = {q, k, v, q_out, k_out, q_weight, k_weight};
  for (const void* t : two)
    if (!aligned(t, 2)) return fail(QF_ERR_ALIGN, "pointers must be aligned to their element");
  if (!aligned(cos_sin, cos_sin_dtype == QF_DTYPE_F32 ? 4 : 2) || !aligned(positions, 8) || !aligned(slots, 8))
    return fail(QF_ERR_ALIGN, "pointers must be aligned to their element");
  const int rc = require_b200(nullptr, nullptr);
  if (rc) return rc;
  p.x[0] = static_cast<const __nv_bfloat16*>(q), p.xt[0] = sq_t, p.xh[0] = sq_h;
  p.x[1] = static_cast<const __nv_bfloat16*>(k), p.xt[1] = sk_t, p.xh[1] = sk_h;
  p.x[2] = static_cast<const __nv_bfloat16*>(v), p.xt[2] = sv_t, p.xh[2] = sv_h;
  p.weight[0] = static_cast<const __nv_bfloat16*>(q_weight);
  p.weight[1] = static_cast<const __nv_bfloat16*>(k_weight);
  p.out[0] = static_cast<__nv_bfloat16*>(q_out), p.ot[0] = so_t, p.oh[0] = so_h;
  p.out[1] = static_cast<__nv_bfloat16*>(k_out), p.ot[1] = sp_t, p.oh[1] = sp_h;
  p.positions = positions;
  p.rot = rot;
  p.cos_sin = rot ? cos_sin : nullptr;
  p.cs_row = s_cs;
  p.max_pos = max_positions;
  p.cs_f32 = cos_sin_dtype == QF_DTYPE_F32;
  p.interleaved = interleaved != 0;
  p.slots = slots;
  p.offset = weight_offset;
  p.eps = eps;
  p.inv_d = 1.f / static_cast<float>(head_size);
  p.heads[0] = num_heads, p.heads[1] = num_kv_heads;
  p.D = head_size;
  p.rows = static_cast<int>(rows);
  p.total = static_cast<uint32_t>(rows * tokens);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.total + kRopeWarps - 1) / kRopeWarps);
  cfg.blockDim = dim3(kRopeWarps * 32);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, rope_any_kernel, p);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}
