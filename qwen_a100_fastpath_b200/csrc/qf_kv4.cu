// qf_kv4.cu -- writes keys and values into a paged cache held in 4 bits, and reads them back (qf_kv4.cuh has the format).
//
// Both are bound by memory: a token and head of D values is 2 D bytes on one side and D / 2 + D / 16 on the other.  A thread
// takes eight values (16 bytes of bf16, one word of nibbles) of several tokens, eight threads a group, whose extremes are
// three shuffles of a packed word.  In fact the logic pipe is the writer's limit (unpacking, clamps, addresses: 57 % busy, IPC
// 2.8): 8192 tokens of 8 heads of 128 written and read back 24.4 us in a graph (3.5 TB/s; floor 13), 64 tokens of 4 heads of
// 256 3.7 us.  Steps at the first size: a piece of one token to a thread 43 us; which piece found once for four tokens 38;
// 32-bit page and slot strides and one reciprocal a group 32; quotients of pairs and packed extremes 26.8; four CTAs on an SM
// 24.4 (five 26.3).
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
  if (st[0] > UINT32_MAX || st[2] > UINT32_MAX || ss[0] > UINT32_MAX / 2 || ss[2] > UINT32_MAX / 2)
    return fail(QF_ERR_STRIDE, "a cache's pages and slots must lie less than 2^32 bytes apart");
  v->codes[0] = static_cast<uint8_t*>(c->k);
  v->codes[1] = static_cast<uint8_t*>(c->v);
  v->scale[0] = static_cast<uint8_t*>(c->k_scale);
  v->scale[1] = static_cast<uint8_t*>(c->v_scale);
  v->page = static_cast<uint32_t>(st[0]), v->head = st[1], v->slot = static_cast<uint32_t>(st[2]);
  v->spage = static_cast<uint32_t>(2 * ss[0]), v->shead = 2 * ss[1], v->sslot = static_cast<uint32_t>(2 * ss[2]);
  kv4_divisor(c->page_size, &v->div_mul, &v->div_shift);
  v->num_pages = c->num_pages, v->page_size = c->page_size, v->heads = c->num_heads;
  return QF_OK;
}

namespace {

struct Kv4IoParams {
  Kv4View cache;
  __nv_bfloat16* x[2];  // keys and values: read, or written by the reader
  int64_t xt[2], xh[2];
  const int64_t* slots;
  int tokens;
  int items;            // pieces of eight values of a token: (keys or values, head, piece), the piece innermost
  int per_pass;         // tokens that a CTA takes at a time
  int passes;           // up to kIoTokens
};

constexpr int kIoThreads = 256;
constexpr int kIoTokens = 4;

// A CTA takes passes * per_pass tokens, a thread the same piece of `passes` of them: which piece that is, and of which head,
// is found out once, and the passes' loads are under way together.  Eight threads in a row share a group and a warp.
template <int D, bool WRITE> __global__ void __launch_bounds__(kIoThreads, 4) kv4_io_kernel(const Kv4IoParams p) {
  constexpr int kPieces = D / 8;
  pdl_launch_dependents();
  pdl_wait();
  const Kv4View& v = p.cache;
  const int local = p.items >= kIoThreads ? 0 : threadIdx.x / p.items;
  if (local >= p.per_pass) return;  // (whole groups of eight)
  const uint32_t group = 0xffu << (threadIdx.x & 24);
  for (int item = threadIdx.x - local * p.items; item < p.items; item += kIoThreads) {
    const int piece = item % kPieces, hh = item / kPieces, side = hh >= v.heads, head = hh - side * v.heads;
    __nv_bfloat16* const x = p.x[side] + head * p.xh[side] + 8 * piece;
    uint8_t* const codes = v.codes[side] + head * v.head + 4 * piece;
    uint8_t* const scale = v.scale[side] + head * v.shead + 4 * (piece / 8);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (p.passes * p.per_pass) + local;
    int64_t slot[kIoTokens];
    uint4 u[kIoTokens];
#pragma unroll
    for (int i = 0; i < kIoTokens; ++i) {
      const int64_t token = first + i * p.per_pass;
      slot[i] = -1;
      if (i < p.passes && token < p.tokens) {
        slot[i] = p.slots[token];
        if (WRITE) u[i] = *reinterpret_cast<const uint4*>(x + token * p.xt[side]);
      }
    }
    uint32_t page[kIoTokens], off[kIoTokens];
    bool ok[kIoTokens];
#pragma unroll
    for (int i = 0; i < kIoTokens; ++i) ok[i] = v.place(slot[i], page[i], off[i]);
    if (WRITE) {
#pragma unroll
      for (int i = 0; i < kIoTokens; ++i) {
        if (!ok[i]) continue;  // (the same for the eight threads of a group)
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[2 * j] = bf16_lo(w[j]), f[2 * j + 1] = bf16_hi(w[j]);
        const uint32_t ends = kv4_extremes(w[0], w[1], w[2], w[3], group);
        float s, c;
        kv4_scale(-bf16_hi(ends), bf16_lo(ends), s, c);
        *reinterpret_cast<uint32_t*>(codes + v.codes_at(page[i], off[i])) = kv4_codes(f, s, c);
        if (piece % 8 == 0)
          *reinterpret_cast<__nv_bfloat162*>(scale + v.scale_at(page[i], off[i])) = __floats2bfloat162_rn(s, c);
      }
    } else {
      uint32_t w[kIoTokens], sc[kIoTokens];
#pragma unroll
      for (int i = 0; i < kIoTokens; ++i)
        if (ok[i]) {
          w[i] = *reinterpret_cast<const uint32_t*>(codes + v.codes_at(page[i], off[i]));
          sc[i] = *reinterpret_cast<const uint32_t*>(scale + v.scale_at(page[i], off[i]));
        }
#pragma unroll
      for (int i = 0; i < kIoTokens; ++i) {
        const int64_t token = first + i * p.per_pass;
        if (i >= p.passes || token >= p.tokens) continue;
        uint4 r = make_uint4(0, 0, 0, 0);
        if (ok[i]) {
          const uint32_t ss = dup_lo(sc[i]), cc = dup_hi(sc[i]);
          // pairs of nibbles (k, k + 4) -> values in order
          const uint32_t a = kv4_pair<0>(w[i], ss, cc), b = kv4_pair<1>(w[i], ss, cc), c = kv4_pair<2>(w[i], ss, cc),
                         d = kv4_pair<3>(w[i], ss, cc);
          r = make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), __byte_perm(a, b, 0x7632),
                         __byte_perm(c, d, 0x7632));
        }
        *reinterpret_cast<uint4*>(x + token * p.xt[side]) = r;
      }
    }
  }
}

template <bool WRITE> cudaError_t launch_io(const cudaLaunchConfig_t& cfg, const Kv4IoParams& p, int head_size) {
  return head_size == 64    ? cudaLaunchKernelEx(&cfg, kv4_io_kernel<64, WRITE>, p)
         : head_size == 128 ? cudaLaunchKernelEx(&cfg, kv4_io_kernel<128, WRITE>, p)
                            : cudaLaunchKernelEx(&cfg, kv4_io_kernel<256, WRITE>, p);
}

int kv4_io(const void* k, int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_t, int64_t sv_h, const int64_t* slots,
           int tokens, const qf_kv4_cache* cache, unsigned flags, void* stream, bool write) {
  Kv4IoParams p = {};
  int rc = kv4_view(cache, &p.cache);
  if (rc) return rc;
  if (tokens < 0) return fail(QF_ERR_SHAPE, "negative size");
  if (tokens == 0) return QF_OK;
  if (!k || !v || !slots) return fail(QF_ERR_INVALID, "null pointer");
  const int64_t items = 2ll * cache->num_heads * (cache->head_size / 8);
  if (items * tokens > INT32_MAX) return fail(QF_ERR_SHAPE, "more than 2^31 - 1 pieces of eight values");
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
  p.tokens = tokens;
  p.items = static_cast<int>(items);
  p.per_pass = items >= kIoThreads ? 1 : static_cast<int>(kIoThreads / items);
  // several passes where there are CTAs enough for the SMs all the same (64 tokens of 4 heads of 256: one pass 3.7 us, four 6.9)
  p.passes = tokens / p.per_pass >= 4 * kIoTokens * 148 ? kIoTokens : 1;
  const int per_cta = p.passes * p.per_pass;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((tokens + static_cast<int64_t>(per_cta) - 1) / per_cta));
  cfg.blockDim = dim3(kIoThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  const cudaError_t e = write ? launch_io<true>(cfg, p, cache->head_size) : launch_io<false>(cfg, p, cache->head_size);
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
