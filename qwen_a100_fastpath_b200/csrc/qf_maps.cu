// qf_maps.cu -- the maps of a step on a paged cache, from the requests' lengths on the GPU: where each request's tokens
// begin, its length after the step, the position and the cache slot of every token, and the pages a request grows into, taken
// from a list of free ones in the requests' order.
//
// With q and past the lengths of request r (negative ones count as zero; all sums stop at 2^31 - 1):
//   seq = past + q;  start = sum of the q before;  pages taken = pages(seq) - pages(past), pages(n) = min(ceil(n / page), W);
//   entry col of r's table is its old one below pages(past), and free[head + taken before + col - pages(past)] from there on
//   (-1 behind the list's end);  token i of the step belongs to the last r with start[r] <= i;  slot = entry * page + offset.
//
// The work is a scan over the requests (two sums) and 16 bytes for each token, so that the call is bound by latency: a
// launch, one round trip for the lengths, the scan, a search, one round trip for a table entry.  Every CTA makes the scan on
// its own in shared memory instead of waiting for one that does; a token on a new page computes its entry from the scan,
// so that no CTA reads what another writes.  The entries themselves are written page by page, whatever the number of tokens
// and of places for them: 64 contexts of 100000 tokens, opened without a place for any, are 400000 entries and 31 us (a token
// at a time it was 25000 turns of one CTA).  Measured: 2.1 us for one request, 3.5 for 256 requests and 8192 tokens, 8.0 for
// 1024 requests and 131072 tokens (in a graph; with the entries written by the tokens 5.1 and 7.8; the call's host time is 7.9).
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/qf_b200.h"
#include "qf_host.h"
#include "qf_ptx.cuh"

namespace qf {
namespace {

struct MapsParams {
  const int32_t *q_lens, *past_lens;
  int32_t* table;
  int64_t table_row;
  const int32_t *free_pages, *free_head;
  int32_t *query_start, *seq_lens, *free_head_out;
  int64_t *positions, *slots;
  int reqs, width, page, num_free, tokens;
  int grow;  // new pages come from free_pages (which may be empty)
};

constexpr int kMapThreads = 256;
constexpr size_t kMapStatic = 1024;  // no less than the kernel's static shared memory
constexpr uint32_t kMapMax = 0x7fffffffu;

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kMapMax); }

__global__ void __launch_bounds__(kMapThreads) maps_kernel(const MapsParams p) {
  extern __shared__ uint32_t sm[];
  uint32_t* start = sm;                      // [reqs + 1]
  uint32_t* first = start + p.reqs + 1;      // [reqs + 1]: pages taken before request r
  uint32_t* past = first + p.reqs + 1;
  __shared__ uint2 warp_sum[kMapThreads / 32];
  static_assert(sizeof(warp_sum) <= kMapStatic, "counted with the dynamic part against the default limit");
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto pages = [&](uint32_t n) { return min((n + static_cast<uint32_t>(p.page) - 1u) / p.page, static_cast<uint32_t>(p.width)); };
  uint32_t base_q = 0, base_p = 0;
  for (int r0 = 0; r0 < p.reqs; r0 += kMapThreads) {
    const int r = r0 + tid;
    uint32_t q = 0, before = 0, taken = 0;
    if (r < p.reqs) {
      q = max(p.q_lens[r], 0);
      before = max(p.past_lens[r], 0);
      taken = pages(sat_add(before, q)) - pages(before);
    }
    uint32_t sq = q, sp = taken;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t a = __shfl_up_sync(0xffffffffu, sq, off), b = __shfl_up_sync(0xffffffffu, sp, off);
      if (lane >= off) sq = sat_add(sq, a), sp = sat_add(sp, b);
    }
    if (lane == 31) warp_sum[warp] = make_uint2(sq, sp);
    __syncthreads();
    uint32_t wq = base_q, wp = base_p;
    for (int w = 0; w < kMapThreads / 32; ++w) {
      const uint2 t = warp_sum[w];
      if (w < warp) wq = sat_add(wq, t.x), wp = sat_add(wp, t.y);
      base_q = sat_add(base_q, t.x), base_p = sat_add(base_p, t.y);
    }
    sq = sat_add(sq, wq), sp = sat_add(sp, wp);
    if (r < p.reqs) {
      start[r + 1] = sq;
      first[r + 1] = sp;
      past[r] = before;
      if (blockIdx.x == 0) {
        p.query_start[r + 1] = static_cast<int32_t>(sq);
        p.seq_lens[r] = static_cast<int32_t>(sat_add(before, q));
      }
    }
    __syncthreads();
  }
  if (tid == 0) start[0] = first[0] = 0;
  const uint32_t head = p.free_head ? max(p.free_head[0], 0) : 0;
  if (blockIdx.x == 0 && tid == 0) {
    p.query_start[0] = 0;
    if (p.free_head_out) p.free_head_out[0] = static_cast<int32_t>(sat_add(head, base_p));
  }
  __syncthreads();
  // the last request whose tokens (or pages) begin at or before v
  auto holder = [&](const uint32_t* begin, uint32_t v) {
    int lo = 0, hi = p.reqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (begin[mid] <= v) lo = mid; else hi = mid - 1;
    }
    return lo;
  };
  // the new page `taken` places behind the list's head
  auto new_page = [&](uint32_t taken) {
    const uint64_t from = static_cast<uint64_t>(head) + taken;
    return from < static_cast<uint64_t>(p.num_free) ? p.free_pages[from] : -1;
  };
  const uint64_t self = blockIdx.x * static_cast<uint64_t>(kMapThreads) + tid, threads = static_cast<uint64_t>(gridDim.x) * kMapThreads;
  const uint32_t total = base_q, opened = p.grow ? base_p : 0;
  for (uint64_t j = self; j < static_cast<uint32_t>(p.tokens); j += threads) {
    const uint32_t i = static_cast<uint32_t>(j);
    int64_t pos = 0, slot = -1;
    if (i < total) {
      const int r = holder(start, i);
      pos = static_cast<int64_t>(past[r]) + (i - start[r]);
      const uint32_t at = static_cast<uint32_t>(min(pos, static_cast<int64_t>(kMapMax)));
      const uint32_t col = at / p.page, off = at - col * p.page;
      if (col < static_cast<uint32_t>(p.width)) {
        const uint32_t old = pages(past[r]);
        const int32_t page = p.grow && col >= old ? new_page(first[r] + (col - old)) : p.table[r * p.table_row + col];
        if (page >= 0) slot = static_cast<int64_t>(page) * p.page + off;
      }
    }
    p.positions[i] = pos, p.slots[i] = slot;
  }
  // (from the last thread on: the first ones have had a token more where those do not come out even)
  for (uint64_t j = threads - 1 - self; j < opened; j += threads) {
    const uint32_t i = static_cast<uint32_t>(j);
    const int r = holder(first, i);
    p.table[r * p.table_row + pages(past[r]) + (i - first[r])] = new_page(i);
  }
}

}  // namespace
}  // namespace qf

using namespace qf;

extern "C" int qf_step_maps(const int32_t* query_lens, const int32_t* past_lens, int num_reqs, int32_t* block_table,
                            int64_t s_bt, int max_pages, int page_size, const int32_t* free_pages, int num_free,
                            const int32_t* free_head, int32_t* query_start, int32_t* seq_lens, int64_t* positions,
                            int64_t* slots, int num_tokens, int32_t* free_head_out, unsigned flags, void* stream) {
  if (num_reqs < 0 || max_pages < 0 || num_free < 0 || num_tokens < 0) return fail(QF_ERR_SHAPE, "negative size");
  if (num_reqs > QF_MAPS_MAX_REQS) return fail(QF_ERR_SHAPE, "more than 16384 requests");
  if (page_size < 1) return fail(QF_ERR_SHAPE, "pages hold at least one slot");
  if (!query_start || (num_reqs && (!query_lens || !past_lens || !seq_lens || (max_pages && !block_table))) ||
      (num_tokens && (!positions || !slots)))
    return fail(QF_ERR_INVALID, "null pointer");
  if (!free_head != !free_head_out || (num_free && !free_pages) || (free_pages && !free_head))
    return fail(QF_ERR_INVALID, "free_pages, free_head and free_head_out go together");
  if (num_reqs > 1 && s_bt < max_pages) return fail(QF_ERR_STRIDE, "row stride smaller than the row");
  const void* four[] = {query_lens, past_lens, block_table, free_pages, free_head, query_start, seq_lens, free_head_out};
  for (const void* t : four)
    if (reinterpret_cast<uintptr_t>(t) % 4) return fail(QF_ERR_ALIGN, "pointers must be aligned to their element");
  if (reinterpret_cast<uintptr_t>(positions) % 8 || reinterpret_cast<uintptr_t>(slots) % 8)
    return fail(QF_ERR_ALIGN, "pointers must be aligned to their element");
  int dev = 0, sms = 0;
  const int rc = require_b200(&dev, &sms);
  if (rc) return rc;
  MapsParams p = {query_lens, past_lens, block_table, s_bt, free_pages, free_head,
                  query_start, seq_lens, free_head_out, positions, slots, num_reqs, max_pages, page_size, num_free,
                  num_tokens, free_head != nullptr};
  const size_t smem = (3 * static_cast<size_t>(num_reqs) + 2) * 4;
  if (smem + kMapStatic > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(maps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (3 * QF_MAPS_MAX_REQS + 2) * 4);
    if (e != cudaSuccess) return fail(QF_ERR_LAUNCH, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  }
  // four tokens a thread; how many pages open is known on the device only: at most 64 entries a thread, until all SMs are in use
  const int64_t entries = p.grow ? static_cast<int64_t>(num_reqs) * max_pages : 0;
  const int64_t for_tokens = (static_cast<int64_t>(num_tokens) + 4 * kMapThreads - 1) / (4 * kMapThreads);
  const int64_t for_pages = (entries + 64 * kMapThreads - 1) / (64 * kMapThreads);
  const int64_t ctas = for_tokens > for_pages ? for_tokens : for_pages;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas < 1 ? 1 : ctas > sms ? sms : ctas));
  cfg.blockDim = dim3(kMapThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, maps_kernel, p);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}
