// qf_kv4.cu -- writes keys and values into a paged cache held in 4 bits, and reads them back (qf_kv4.cuh has the format).
//
// Both are bound by memory: a token and head of D values is 2 D bytes on one side and D / 2 + D / 16 on the other.  A thread
// takes eight values (16 bytes of bf16, one word of nibbles), eight threads a group, whose extremes are three shuffles.
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

int kv4_view(const qf_kv4_cache* c, Kv4View* v) {
  if (!c) return fail(QF_ERR_INVALID, "null cache");
  if (c->num_pages < 0 || c->page_size < 1 || c->num_heads < 1) return fail(QF_ERR_SHAPE, "cache sizes");
  if (c->head_size != 64 && c->head_size != 128 && c->head_size != 256)
    return fail(QF_ERR_SHAPE, "head size must be 64, 128 or 256");
  const bool any = c->num_pages > 0;
  if (any && (!c->k || !c->v || !c->k_scale || !c->v_scale)) return fail(QF_ERR_INVALID, "null pointer in the cache");
  const int64_t st[] = {c->page_stride, c->head_stride, c->slot_stride};
  const int64_t ss[] = {c->scale_page_stride, c->scale_head_stride, c->scale_slot_stride};
  const int pair = 2 * (c->head_size / kKv4Group);
  for (int i = 0; i < 3; ++i) {
    if (st[i] < 0 || ss[i] < 0) return fail(QF_ERR_STRIDE, "negative stride in the cache");
    if (st[i] % 16 || ss[i] % pair) return fail(QF_ERR_ALIGN, "cache strides");
  }
  const void* codes[] = {c->k, c->v};
  const void* scales[] = {c->k_scale, c->v_scale};
  for (int i = 0; i < 2; ++i)
    if (reinterpret_cast<uintptr_t>(codes[i]) % 16 || reinterpret_cast<uintptr_t>(scales[i]) % (2 * pair))
      return fail(QF_ERR_ALIGN, "cache pointers");
  v->codes[0] = static_cast<uint8_t*>(c->k);
  v->codes[1] = static_cast<uint8_t*>(c->v);
  v->scale[0] = static_cast<__nv_bfloat16*>(c->k_scale);
  v->scale[1] = static_cast<__nv_bfloat16*>(c->v_scale);
  v->page = st[0], v->head = st[1], v->slot = st[2];
  v->spage = ss[0], v->shead = ss[1], v->sslot = ss[2];
  v->num_pages = c->num_pages, v->page_size = c->page_size, v->heads = c->num_heads;
  return QF_OK;
}

namespace {

struct Kv4IoParams {
  Kv4View cache;
  __nv_bfloat16* x[2];  // keys and values: read, or written by the reader
  int64_t xt[2], xh[2];
  const int64_t* slots;
  uint32_t items;       // pieces of eight values
  int pieces;           // of a head
};

// Where a slot is: false if it is none of the cache's.
__device__ __forceinline__ bool place(const Kv4View& c, int64_t slot, int64_t& page, int64_t& off) {
  if (slot < 0) return false;
  page = slot / c.page_size;
  off = slot - page * c.page_size;
  return page < c.num_pages;
}

constexpr int kIoThreads = 256;

// Items: (token, keys or values, head, piece), the piece innermost; eight in a row share a group and a warp.
__global__ void __launch_bounds__(kIoThreads) kv4_write_kernel(const Kv4IoParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t i = blockIdx.x * kIoThreads + threadIdx.x;
  const uint32_t at = i < p.items ? i : p.items - 1;
  const int piece = at % p.pieces;
  uint32_t rest = at / p.pieces;
  const int head = rest % p.cache.heads;
  rest /= p.cache.heads;
  const int side = rest & 1;
  const int64_t token = rest >> 1;
  const uint4 u = *reinterpret_cast<const uint4*>(p.x[side] + token * p.xt[side] + head * p.xh[side] + 8 * piece);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) x[2 * j] = bf16_lo(w[j]), x[2 * j + 1] = bf16_hi(w[j]);
  float hi = x[0], lo = -x[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) hi = max_nan(hi, x[j]), lo = max_nan(lo, -x[j]);
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) {
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
    lo = max_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
  }
  float s, c;
  kv4_scale(-lo, hi, s, c);
  uint32_t code = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) code |= kv4_code(x[j], s, c) << (4 * j);
  int64_t page, off;
  if (i >= p.items || !place(p.cache, p.slots[token], page, off)) return;
  const Kv4View& v = p.cache;
  reinterpret_cast<uint32_t*>(v.codes[side] + page * v.page + head * v.head + off * v.slot)[piece] = code;
  if (piece % 8 == 0)
    reinterpret_cast<__nv_bfloat162*>(v.scale[side] + page * v.spage + head * v.shead + off * v.sslot)[piece / 8] =
        __floats2bfloat162_rn(s, c);
}

__global__ void __launch_bounds__(kIoThreads) kv4_read_kernel(const Kv4IoParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t i = blockIdx.x * kIoThreads + threadIdx.x;
  if (i >= p.items) return;
  const int piece = i % p.pieces;
  uint32_t rest = i / p.pieces;
  const int head = rest % p.cache.heads;
  rest /= p.cache.heads;
  const int side = rest & 1;
  const int64_t token = rest >> 1;
  uint4 r = make_uint4(0, 0, 0, 0);
  int64_t page, off;
  if (place(p.cache, p.slots[token], page, off)) {
    const Kv4View& v = p.cache;
    const uint32_t w = reinterpret_cast<const uint32_t*>(v.codes[side] + page * v.page + head * v.head + off * v.slot)[piece];
    const uint32_t sc = reinterpret_cast<const uint32_t*>(v.scale[side] + page * v.spage + head * v.shead +
                                                          off * v.sslot)[piece / 8];
    const uint32_t ss = dup_lo(sc), cc = dup_hi(sc);
    // pairs of nibbles (k, k + 4) -> values in order
    const uint32_t a = kv4_pair<0>(w, ss, cc), b = kv4_pair<1>(w, ss, cc), c = kv4_pair<2>(w, ss, cc),
                   d = kv4_pair<3>(w, ss, cc);
    r = make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), __byte_perm(a, b, 0x7632),
                   __byte_perm(c, d, 0x7632));
  }
  *reinterpret_cast<uint4*>(p.x[side] + token * p.xt[side] + head * p.xh[side] + 8 * piece) = r;
}

int kv4_io(const void* k, int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_t, int64_t sv_h, const int64_t* slots,
           int tokens, const qf_kv4_cache* cache, unsigned flags, void* stream, bool write) {
  Kv4IoParams p = {};
  int rc = kv4_view(cache, &p.cache);
  if (rc) return rc;
  if (tokens < 0) return fail(QF_ERR_SHAPE, "negative size");
  if (tokens == 0) return QF_OK;
  if (!k || !v || !slots) return fail(QF_ERR_INVALID, "null pointer");
  p.pieces = cache->head_size / 8;
  const int64_t items = 2ll * tokens * cache->num_heads * p.pieces;
  if (items > INT32_MAX) return fail(QF_ERR_SHAPE, "more than 2^31 - 1 pieces of eight values");
  const int64_t st[] = {sk_t, sk_h, sv_t, sv_h};
  for (int64_t s : st) {
    if (s < 0) return fail(QF_ERR_STRIDE, "negative stride");
    if (s % 8) return fail(QF_ERR_ALIGN, "key and value strides must be multiples of eight elements");
  }
  if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16 ||
      reinterpret_cast<uintptr_t>(slots) % 8)
    return fail(QF_ERR_ALIGN, "keys and values must be 16-byte aligned, slots aligned to their element");
  rc = require_b200(nullptr, nullptr);
  if (rc) return rc;
  p.x[0] = static_cast<__nv_bfloat16*>(const_cast<void*>(k));
  p.x[1] = static_cast<__nv_bfloat16*>(const_cast<void*>(v));
  p.xt[0] = sk_t, p.xh[0] = sk_h, p.xt[1] = sv_t, p.xh[1] = sv_h;
  p.slots = slots;
  p.items = static_cast<uint32_t>(items);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((items + kIoThreads - 1) / kIoThreads));
  cfg.blockDim = dim3(kIoThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  const cudaError_t e = write ? cudaLaunchKernelEx(&cfg, kv4_write_kernel, p) : cudaLaunchKernelEx(&cfg, kv4_read_kernel, p);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}

}  // namespace
}  // namespace qf

using namespace qf;

extern "C" int qf_kv4_write(const void* k, int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_t, int64_t sv_h,
                            const int64_t* slots, int tokens, const qf_kv4_cache* cache, unsigned flags, void* stream) {
  return kv4_io(k, sk_t, sk_h, v, sv_t, sv_h, slots, tokens, cache, flags, stream, true);
}

extern "C" int qf_kv4_read(void* k, int64_t sk_t, int64_t sk_h, void* v, int64_t sv_t, int64_t sv_h, const int64_t* slots,
                           int tokens, const qf_kv4_cache* cache, unsigned flags, void* stream) {
  return kv4_io(k, sk_t, sk_h, v, sv_t, sv_h, slots, tokens, cache, flags, stream, false);
}
