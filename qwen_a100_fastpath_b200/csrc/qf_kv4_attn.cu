// qf_kv4_attn.cu -- attention of uniform decode and verification batches over the paged cache held in 4 bits (qf_kv4.cuh has
// the format).
//
// Mathematics: O = softmax(scale q K^T + mask) V in one pass over the keys with a running maximum and sum in fp32, over the
// bf16 values that the cache stands for.
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

struct Kv4AttnParams {
  const __nv_bfloat16* q;
  int64_t qt, qh;
  __nv_bfloat16* out;
  int64_t ot, oh;
  Kv4View cache;
  const int32_t* table;
  int64_t table_row;
  const int32_t* lens;
  int max_pages, reqs, q_len, heads, group, D;
  float scale_log2;
};

constexpr int kSimpleThreads = 128;

// The value of dimension d of the slot at (codes, scale).
__device__ __forceinline__ float kv4_value(const uint8_t* codes, const __nv_bfloat16* scale, int d) {
  const float n = static_cast<float>(((codes[d / 2] >> (4 * (d & 1))) & 15) + 16);
  const float s = __bfloat162float(scale[2 * (d / kKv4Group)]), c = __bfloat162float(scale[2 * (d / kKv4Group) + 1]);
  return __bfloat162float(__float2bfloat16_rn(fmaf(n, s, c)));
}

// One CTA per query token and head; a thread a key of each 128, then two dimensions of the sum.
__global__ void __launch_bounds__(kSimpleThreads) kv4_attn_simple_kernel(const Kv4AttnParams p) {
  __shared__ float q[256], w[kSimpleThreads], red[kSimpleThreads / 32];
  __shared__ int64_t at[kSimpleThreads], sat[kSimpleThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, token = blockIdx.x, head = blockIdx.y;
  const int b = token / p.q_len, qi = token % p.q_len, kv = head / p.group;
  for (int d = tid; d < p.D; d += kSimpleThreads) q[d] = __bfloat162float(p.q[token * p.qt + head * p.qh + d]);
  const int64_t keys = min(static_cast<int64_t>(p.lens[b]) - p.q_len + qi + 1,
                           static_cast<int64_t>(p.max_pages) * p.cache.page_size);
  float top = -INFINITY, sum = 0.f, acc[2] = {0.f, 0.f};
  for (int64_t k0 = 0; k0 < keys; k0 += kSimpleThreads) {
    const int64_t key = k0 + tid;
    float x = -INFINITY;
    __syncthreads();  // the last keys have been read
    at[tid] = -1;
    if (key < keys) {
      const int32_t page = p.table[b * p.table_row + key / p.cache.page_size];
      if (page >= 0 && page < p.cache.num_pages) {
        const int64_t off = key % p.cache.page_size;
        at[tid] = page * p.cache.page + kv * p.cache.head + off * p.cache.slot;
        sat[tid] = page * p.cache.spage + kv * p.cache.shead + off * p.cache.sslot;
        x = 0.f;
        for (int d = 0; d < p.D; ++d)
          x = fmaf(q[d], kv4_value(p.cache.codes[0] + at[tid], p.cache.scale[0] + sat[tid], d), x);
        x *= p.scale_log2;
      }
    }
    float m = x;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, off));
    __syncthreads();
    if (tid % 32 == 0) red[tid / 32] = m;
    __syncthreads();
    for (int i = 0; i < kSimpleThreads / 32; ++i) m = max_nan(m, red[i]);
    const float next = max_nan(top, m);
    if (next == -INFINITY) continue;
    w[tid] = at[tid] < 0 ? 0.f : exp2f(x - next);
    __syncthreads();
    const float old = exp2f(top - next);
    top = next;
    sum *= old, acc[0] *= old, acc[1] *= old;
    const int n = static_cast<int>(min(keys - k0, static_cast<int64_t>(kSimpleThreads)));
    for (int j = 0; j < n; ++j) {
      if (at[j] < 0) continue;
      sum += w[j];
      for (int i = 0; i < 2; ++i)
        if (tid + i * kSimpleThreads < p.D)
          acc[i] = fmaf(w[j], kv4_value(p.cache.codes[1] + at[j], p.cache.scale[1] + sat[j], tid + i * kSimpleThreads),
                        acc[i]);
    }
  }
  for (int i = 0; i < 2; ++i)
    if (tid + i * kSimpleThreads < p.D)
      p.out[token * p.ot + head * p.oh + tid + i * kSimpleThreads] = __float2bfloat16_rn(sum == 0.f ? 0.f : acc[i] / sum);
}

}  // namespace
}  // namespace qf

using namespace qf;

extern "C" size_t qf_kv4_attn_workspace_bytes(int num_reqs, int q_len, int num_heads, int num_kv_heads, int head_size) {
  (void)num_reqs, (void)q_len, (void)num_heads, (void)num_kv_heads, (void)head_size;
  return 256;
}

extern "C" int qf_kv4_attn(const void* q, int64_t sq_t, int64_t sq_h, const qf_kv4_cache* cache,
                           const int32_t* block_table, int64_t s_bt, int max_pages, const int32_t* seq_lens, void* out,
                           int64_t so_t, int64_t so_h, int num_reqs, int q_len, int num_heads, float scale, void* ws,
                           size_t ws_bytes, unsigned flags, void* stream) {
  Kv4AttnParams p = {};
  int rc = kv4_view(cache, &p.cache);
  if (rc) return rc;
  if (num_reqs < 0 || q_len < 1 || num_heads < 0 || max_pages < 0) return fail(QF_ERR_SHAPE, "sizes");
  if (num_heads % cache->num_heads) return fail(QF_ERR_SHAPE, "query heads must be a multiple of the cache's heads");
  if (static_cast<int64_t>(q_len) * (num_heads / cache->num_heads) > 64)
    return fail(QF_ERR_SHAPE, "more than 64 query rows for a key head");
  if (static_cast<int64_t>(num_reqs) * q_len > INT32_MAX / 64 || num_heads > 65535)
    return fail(QF_ERR_SHAPE, "too many query rows");
  if (!(scale > -3.4e38f && scale < 3.4e38f)) return fail(QF_ERR_INVALID, "scale must be finite");
  if (num_reqs == 0 || num_heads == 0) return QF_OK;
  if (!q || !out || !seq_lens || (max_pages && !block_table)) return fail(QF_ERR_INVALID, "null pointer");
  if (sq_t < 0 || sq_h < 0 || so_t < 0 || so_h < 0 || s_bt < 0) return fail(QF_ERR_STRIDE, "negative stride");
  if (sq_t % 8 || sq_h % 8 || so_t % 8 || so_h % 8 || reinterpret_cast<uintptr_t>(q) % 16 ||
      reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(block_table) % 4 ||
      reinterpret_cast<uintptr_t>(seq_lens) % 4 || reinterpret_cast<uintptr_t>(ws) % 256)
    return fail(QF_ERR_ALIGN, "query and out 16-byte aligned with strides multiples of eight, workspace 256-byte aligned");
  if (!ws || ws_bytes < qf_kv4_attn_workspace_bytes(num_reqs, q_len, num_heads, cache->num_heads, cache->head_size))
    return fail(QF_ERR_WORKSPACE, "workspace missing or too small");
  rc = require_b200(nullptr, nullptr);
  if (rc) return rc;
  p.q = static_cast<const __nv_bfloat16*>(q), p.qt = sq_t, p.qh = sq_h;
  p.out = static_cast<__nv_bfloat16*>(out), p.ot = so_t, p.oh = so_h;
  p.table = block_table, p.table_row = s_bt, p.max_pages = max_pages;
  p.lens = seq_lens;
  p.reqs = num_reqs, p.q_len = q_len, p.heads = num_heads, p.group = num_heads / cache->num_heads;
  p.D = cache->head_size;
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(num_reqs * q_len), static_cast<unsigned>(num_heads));
  cfg.blockDim = dim3(kSimpleThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_attn_simple_kernel, p);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}
