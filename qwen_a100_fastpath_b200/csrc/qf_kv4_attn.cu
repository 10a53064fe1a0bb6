// qf_kv4_attn.cu -- attention of uniform decode and verification batches over the paged cache held in 4 bits (qf_kv4.cuh has
// the format).
//
// Mathematics: O = softmax(scale q K^T + mask) V in one pass over the keys, with a reference m and a sum l for each query row
// in fp32: a tile's weights are p = 2^(x - m) with x in units of log2, and where m has to rise O and l are first scaled by
// 2^(m_old - m).  Parts of a row's keys that different CTAs hold are joined by their m and l afterwards.
//
// Bound by memory for few rows (D / 2 + D / 16 bytes for each key and value), by taking the nibbles apart and the matrix
// instructions for many.  The R = q_len * group query rows of a key head are one tile, so that its cache is read once.  The
// tokens are the 16-row operand of mma.sync, the query rows the 8-column one, in both products: S^T = K Q^T and
// O^T = V^T P^T.  Decoding has 1 to 64 rows, often 6 or 8, and pads them to a multiple of 8 and not of 16 (or of tcgen05's
// 64 or 128, whose operands would besides have to go through shared memory as bf16, 4 bytes a value written and read for the
// half byte that came); the operand with 16 rows is the one that is unpacked, straight into registers.
//
// A nibble row of a token is both operands as it lies.  For K, ldmatrix gives a thread eight dimensions of token g (and
// g + 8), and the order of the dimensions within the sum is free as long as the query has the same.  For V, the transposed
// ldmatrix of 16-bit elements (four dimensions each) gives a thread the same four dimensions of two neighbouring tokens in
// the two halves of a register, which is what the 16-bit operand wants: token pairs; each of the four nibble places is a
// tile of 16 dimensions.
//
// A CTA of four warps takes 64 tokens at a time: each warp scores 16 of them against all rows, the weights (bf16) are
// exchanged in shared memory, and each warp adds up 64 of the head's dimensions (over all tokens for D = 256, over half or a
// quarter of them for 128 and 64).  The weights are relative to a reference, not to the running maximum: bf16 and fp32 have
// the same range of exponents, so that the precision of a weight does not depend on where the reference lies.  It is set 32
// above the first tile's maximum, and set anew, with the exchange that this needs, only where a score has come within 16 of
// it.  So weights are at most 2^-16, and the sums over 2^17 keys of the largest values that the cache keeps (2^126) stay below
// 2^128; the row's largest weight is at least 2^-32, so that means of values down to 2^-90 lose nothing to fp32's range either.
// (Set at the first maximum itself, the weights reached 2^16, and sums of values from 2^112 on could become infinite.)
//
// Codes and scales arrive by cp.async, kAhead tiles ahead; the pages are looked up a tile before that.  The CTAs split all
// tiles of all requests and heads evenly, whatever the lengths; a CTA's part may begin or end inside a (request, head), and
// a second kernel joins those.
//
// Measured (in a graph, the cache from DRAM): 100000 keys x 2 requests, 4 heads of 256, 30 rows 116 us (2.0 TB/s, 212 TFLOP/s;
// floor 35), 38400 keys, 18 rows 31 us (floor 6.8), 64 requests of 1 to 8192 keys, 8 heads of 128, 8 rows 36 us (floor 12),
// 700 keys 9.8 us.  What bounds it: neither DRAM (a third) nor the tensor pipe (48 %) nor issue (IPC 1.9 of 4), but how few
// warps (12 an SM with 30 rows, 168 registers each) have to cover the latencies of a tile's phases.  At the first size without
// the matrix instructions 121 us, without the unpacking 104, without the copies 111, without the first two 100.  Of a tile's
// 5300 to 6000 clocks the scores take 1600 to 1900, the values 1400 to 1900, its copies 600 to 700, the bookkeeping before it 500
// to 900, the weights 350.
// Not kept, at the four sizes or the first: scores of the next tile beside this one's values in one block of code 120; the
// loops over groups rolled 121; five or six CTAs an SM with one row tile 54 (50 then); pages of a tile or more by every thread
// itself, without places in shared memory 121.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/qf_b200.h"
#include "qf_fp8.cuh"
#include "qf_host.h"
#include "qf_kv4.cuh"
#include "qf_ptx.cuh"

namespace qf {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxSms = 160;    // the workspace is sized without asking the device

struct AttnParams {
  const __nv_bfloat16* q;
  int64_t qt, qh;
  __nv_bfloat16* out;
  int64_t ot, oh;
  // the cache: keys' codes and scales, and how many bytes further the values' are; strides in bytes
  const uint8_t *codes, *scales;
  int64_t value_codes, value_scales, head, shead;
  uint32_t page, slot, spage, sslot;
  int num_pages, page_size, heads;
  const int32_t* table;
  int64_t table_row;
  const int32_t* lens;
  int64_t width;  // keys that a row of the table can place
  int reqs, q_len, group, rows;
  uint32_t div_mul, div_shift;  // by the page size
  float scale_log2;
  // workspace
  int4* joins;      // [grid]: the (request, head) that begins in a CTA's share and ends in a later one's
  float2* part_ml;  // [2 * grid][rows]: reference and sum
  float* part_o;    // [2 * grid][rows][D]
};

// Blocks of 16 tokens of a warp in a tile, and CTAs of an SM.  Two blocks halve a tile's fixed share of time, where registers
// and shared memory allow it: D = 128 with 8 rows 43.6 -> 38.6 us (the ragged batch above, then), with 16 rows 97 -> 74 (16
// requests of 8192 keys), D = 64 with 8 rows 76 -> 66; with 16 rows D = 64 loses, 53 -> 65 (64 requests of 4096 keys).
constexpr int token_blocks(int d, int nq) { return (d == 128 && nq <= 2) || (d == 64 && nq == 1) ? 2 : 1; }
constexpr int ctas_per_sm(int d, int nq) { return nq == 1 ? 4 : nq <= 4 ? 3 : 2; }

template <int D, int NQ> struct Geo {
  static constexpr int kBlocks = token_blocks(D, NQ), kTile = 64 * kBlocks;  // tokens
  static constexpr int kWords = kTile / 32;                // of a bit for each token
  static constexpr int kRow = D / 2;                       // bytes of a token's codes
  static constexpr int kScale = D / 16;                    // bytes of a token's scales
  static constexpr int kSide = kTile * (kRow + kScale);    // bytes of a tile's keys, or values
  // A tile's keys are done with when its weights are exchanged, its values a tile later.
  static constexpr int kAhead = D == 64 && kBlocks == 1 ? 3 : 2, kKeyStages = kAhead, kValueStages = kAhead + 1;
  static constexpr int kCtas = ctas_per_sm(D, NQ);
  static constexpr int kPRow = 2 * kTile + 16;             // bytes of a query row's weights, one chunk of padding
  static constexpr int kQBytes = 4096 * NQ;                // the query's fragments; at a part's end the warps' sums
  static constexpr int kPBytes = 8 * NQ * kPRow;
  static constexpr int kOffV = kKeyStages * kSide;
  static constexpr int kOffQ = kOffV + kValueStages * kSide;
  static constexpr int kOffP = kOffQ + kQBytes;
  static constexpr int kSmem = kOffP + kPBytes;
  static constexpr int kDimWarps = D / 64, kTokenWarps = 4 / kDimWarps;
};

// ---- small PTX forms ----
// 16, 8 or 4 bytes from global to shared memory without registers; zeros where !there (nothing is read then).
template <int N> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool there) {
  const int n = there ? N : 0;
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(N) : "memory");
}
// As mma_bf16_m16n8k16, free to be moved among other instructions.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two 8x8 tiles of 16-bit elements into shared memory, transposed: lane l gives the address of row l % 8 of tile l / 8.
__device__ __forceinline__ void stsm_x2_trans(uint32_t addr, uint32_t r0, uint32_t r1) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1, %2};" ::"r"(addr), "r"(r0), "r"(r1) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Where the 16-byte chunk c of a token's codes lies in its tile: eight neighbouring tokens' chunks c are in different banks.
template <int ROW> __device__ __forceinline__ uint32_t chunk_at(uint32_t token, uint32_t c) {
  constexpr int kPerLine = 128 / ROW;  // tokens in 128 bytes
  return token * ROW + ((c ^ ((token / kPerLine) & (ROW / 16 - 1))) << 4);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return reinterpret_cast<const uint32_t&>(h);
}

// Tiles of a request, for each head: at least one, which writes the zeros of a request without keys.
__device__ __forceinline__ int keys_of(const AttnParams& p, int len) {
  return static_cast<int>(min(static_cast<int64_t>(max(len, 0)), p.width));
}
template <int TILE> __device__ __forceinline__ int tiles_of(const AttnParams& p, int len) {
  return max((keys_of(p, len) - 1) / TILE + 1, 1);
}

// What a (request, head) costs besides its tiles, in tiles: the query, the first reference, the output.  The CTAs' shares are
// even in these units: positions v below kStart in front of a (request, head)'s first tile, tile v - kStart behind.  (Ragged
// batch above, then: 69 us without, 51.8 with 1, 50.4 with 2, 52.9 with 4.)
constexpr int kStart = 2;

// A walk over tiles in the order (request, head, tile).
template <int TILE> struct Cursor {
  int b, h, tile, tiles, len;
  __device__ __forceinline__ void next(const AttnParams& p) {
    if (++tile < tiles) return;
    tile = 0;
    if (++h < p.heads) return;
    h = 0;
    if (++b < p.reqs) len = p.lens[b], tiles = tiles_of<TILE>(p, len);
  }
};

constexpr float kNoRef = -3e38f;  // stands for the reference of a row that has seen no key, in a part that is joined
constexpr float kAbove = 32.f;    // of the maximum, where a reference is set
constexpr float kNear = -16.f;    // a score that comes nearer has it set anew

// Positions 0 to total - 1 split evenly: CTA i begins at start(i), position v is in CTA holder(v)'s share.
struct Shares {
  uint32_t each, more;  // the first `more` CTAs have one more than `each`
  __device__ __forceinline__ Shares(uint32_t total, uint32_t ctas) : each(total / ctas), more(total - each * ctas) {}
  __device__ __forceinline__ uint32_t start(uint32_t i) const { return each * i + min(i, more); }
  __device__ __forceinline__ uint32_t holder(uint32_t v) const {
    const uint32_t big = (each + 1) * more;
    return v < big ? v / (each + 1) : more + (v - big) / each;
  }
};

// Where a token's keys are.
struct __align__(16) Place {
  const uint8_t *codes, *scales;
};

template <int D, int NQ>
__global__ void __launch_bounds__(kThreads, Geo<D, NQ>::kCtas) kv4_attn_kernel(const AttnParams p) {
  using G = Geo<D, NQ>;
  constexpr int kTile = G::kTile, kBlocks = G::kBlocks, kWords = G::kWords;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Place places[kTile];               // of the tile that is copied next
  __shared__ __align__(16) uint32_t there[G::kAhead + 1][kWords];  // a bit for each token of a tile
  __shared__ float red[4][8 * NQ];
  __shared__ uint32_t bad[2][4][kWords];       // tokens whose values' group is not finite, of a tile with masked rows
  __shared__ uint32_t scan[4], bounds[2];
  __shared__ int found[4];
  __shared__ uint8_t row_query[8 * NQ];        // qi of a row
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t sm = smem_u32(smem);
  for (int r = tid; r < 8 * NQ; r += kThreads) row_query[r] = r < p.rows ? r / p.group : 0;

  // ---- this CTA's part: a scan over the requests, twice (for the sum, then for where the part begins and ends) ----
  uint32_t total = 0, begin = 0, end = 0, n = 0;
  uint32_t ctas = 1;
  int len = 0;
  for (int pass = 0; pass < 2; ++pass) {
    uint32_t base = 0;
    for (int b0 = 0; b0 < p.reqs; b0 += kThreads) {
      const int b = b0 + tid;
      if (pass == 0 || p.reqs > kThreads) {
        if (b < p.reqs) len = p.lens[b];
        n = b < p.reqs ? tiles_of<kTile>(p, len) + kStart : 0;
      }
      uint32_t sum = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += a;
      }
      __syncthreads();
      if (lane == 31) scan[warp] = sum;
      __syncthreads();
      uint32_t before = base + sum - n;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (w < warp) before += scan[w];
        base += scan[w];
      }
      if (pass == 0 || !n) continue;
      before *= p.heads;
      const uint32_t after = before + n * p.heads;
      // tiles before a position: all those before the request, those of its heads before, those before it
      const uint32_t tiles = before - kStart * p.heads * b;
      if (before <= begin && begin < after) {
        const uint32_t h = (begin - before) / n, rest = begin - before - h * n;
        const uint32_t tile = rest > kStart ? rest - kStart : 0;
        found[0] = b, found[1] = h, found[2] = tile, found[3] = len;
        bounds[0] = tiles + h * (n - kStart) + tile;
      }
      if (before < end && end <= after) {
        const uint32_t h = (end - before) / n, rest = end - before - h * n;
        bounds[1] = tiles + h * (n - kStart) + (rest > kStart ? rest - kStart : 0);
      }
    }
    if (pass == 0) {
      total = base * p.heads;
      ctas = min(total, gridDim.x);
      if (blockIdx.x >= ctas) {
        if (tid == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
      }
      const Shares shares(total, ctas);
      begin = shares.start(blockIdx.x), end = shares.start(blockIdx.x + 1);
    }
  }
  __syncthreads();
  const int count = static_cast<int>(bounds[1] - bounds[0]);
  if (count == 0) {
    if (tid == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }
  Cursor<kTile> cur;
  cur.b = found[0], cur.h = found[1], cur.tile = found[2], cur.len = found[3];
  cur.tiles = tiles_of<kTile>(p, cur.len);

  // the query's fragments: a thread's eight dimensions of a row in the order in which the nibbles come apart
  auto query = [&] {
    constexpr int kAll = D / 32 * NQ * 32, kBatch = 4;
    for (int e0 = tid; e0 < kAll; e0 += kBatch * kThreads) {
      uint4 u[kBatch];  // on their way together
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int e = e0 + k * kThreads, l5 = e & 31, j = (e >> 5) % NQ, c = (e >> 5) / NQ;
        const int r = 8 * j + (l5 >> 2);
        u[k] = make_uint4(0, 0, 0, 0);
        if (e < kAll && r < p.rows) {
          const int qi = row_query[r], hq = cur.h * p.group + r - qi * p.group;
          u[k] = *reinterpret_cast<const uint4*>(p.q + (static_cast<int64_t>(cur.b) * p.q_len + qi) * p.qt + hq * p.qh +
                                                 32 * c + 8 * (l5 & 3));
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (e0 + k * kThreads < kAll)
          reinterpret_cast<uint4*>(smem + G::kOffQ)[e0 + k * kThreads] =
              make_uint4(__byte_perm(u[k].x, u[k].z, 0x5410), __byte_perm(u[k].x, u[k].z, 0x7632),
                         __byte_perm(u[k].y, u[k].w, 0x5410), __byte_perm(u[k].y, u[k].w, 0x7632));
    }
  };

  // ---- copies: the threads of tokens look pages up, then all threads copy ----
  Cursor<kTile> ahead = cur;  // of the tile whose pages are looked up next
  struct Look {
    int32_t entry;
    uint32_t off;  // in the page
    int h;
  };
  auto look = [&](int i) {  // tile i's page of this thread's token; and on to the next tile
    Look r = {-1, 0, 0};
    if (tid >= kTile || i >= count) return r;
    const uint32_t pos = ahead.tile * kTile + tid;
    if (static_cast<int>(pos) < keys_of(p, ahead.len)) {
      const uint32_t col = (__umulhi(pos, p.div_mul) + pos) >> p.div_shift;
      r.entry = p.table[ahead.b * p.table_row + col];
      r.off = pos - col * p.page_size;
    }
    r.h = ahead.h;
    if (i + 1 < count) ahead.next(p);
    return r;
  };
  auto place = [&](const Look& r, Place* to, int value_slot) {
    if (tid >= kTile) return;
    const bool ok = static_cast<uint32_t>(r.entry) < static_cast<uint32_t>(p.num_pages);
    const uint32_t e = ok ? r.entry : 0, off = ok ? r.off : 0;  // (a place that is not read, all the same within the cache)
    to[tid].codes = p.codes + r.h * p.head + static_cast<uint64_t>(e) * p.page + static_cast<uint64_t>(off) * p.slot;
    to[tid].scales = p.scales + r.h * p.shead + static_cast<uint64_t>(e) * p.spage + static_cast<uint64_t>(off) * p.sslot;
    const uint32_t bits = __ballot_sync(0xffffffffu, ok);
    if (lane == 0) there[value_slot][warp] = bits;
  };
  constexpr int kChunks = G::kRow / 16, kRows = kThreads / kChunks;
  static_assert(kRows / (128 / G::kRow) % (G::kRow / 16) == 0, "a thread's rows have their chunks in the same places");
  const int copy_row = tid / kChunks, copy_chunk = tid % kChunks;
  const uint32_t copy_at = chunk_at<G::kRow>(copy_row, copy_chunk);
  auto copy = [&](int i, const Place* from, int key_slot, int value_slot) {
    if (i < count) {
      const uint32_t keys = sm + key_slot * G::kSide, vals = sm + G::kOffV + value_slot * G::kSide;
      // everything that is read from shared memory first
      const uint8_t* codes[kTile / kRows];
      const uint8_t* scales[kBlocks];
      uint32_t words[kWords];
#pragma unroll
      for (int j = 0; j < kTile / kRows; ++j) codes[j] = from[j * kRows + copy_row].codes + 16 * copy_chunk;
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) scales[j] = from[(j * kThreads + tid) % kTile].scales;
#pragma unroll
      for (int k = 0; k < kWords; ++k) words[k] = there[value_slot][k];
#pragma unroll
      for (int j = 0; j < kTile / kRows; ++j) {
        const int token = j * kRows + copy_row;
        const uint32_t word = kRows <= 32 ? words[j * kRows / 32] : copy_row < 32 ? words[2 * j] : words[(2 * j + 1) % kWords];
        const bool ok = word >> (token % 32) & 1;
        copy_async<16>(keys + copy_at + j * kRows * G::kRow, codes[j], ok);
        copy_async<16>(vals + copy_at + j * kRows * G::kRow, codes[j] + p.value_codes, ok);
      }
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        const int token = (j * kThreads + tid) % kTile, side = (j * kThreads + tid) / kTile;
        uint32_t word = words[0];
#pragma unroll
        for (int k = 1; k < kWords; ++k) word = warp % kWords == k ? words[k] : word;  // a warp's tokens are those of a word
        copy_async<G::kScale>((side ? vals : keys) + kTile * G::kRow + token * G::kScale,
                              scales[j] + (side ? p.value_scales : 0), word >> lane & 1);
      }
    }
    cp_async_commit();
  };
  Look next;  // of the tile kAhead tiles ahead
  {
    // (the later ones' where the weights will be)
    static_assert((G::kAhead - 1) * kTile * sizeof(Place) <= G::kPBytes, "places fit where the weights will be");
    auto places_of = [&](int i) { return i == 0 ? places : reinterpret_cast<Place*>(smem + G::kOffP) + (i - 1) * kTile; };
    Look first[G::kAhead];  // all on their way at once, with the query
#pragma unroll
    for (int i = 0; i < G::kAhead; ++i) first[i] = look(i);
    next = look(G::kAhead);
    query();
#pragma unroll
    for (int i = 0; i < G::kAhead; ++i) place(first[i], places_of(i), i);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G::kAhead; ++i) copy(i, places_of(i), i, i);
  }

  // ---- a part of one (request, head) after the other ----
  float o[4][NQ][4];  // [nibble place][rows' tile][fragment]: O^T of this warp's 64 dimensions
  float ref[NQ][2], l[NQ][2];
  const int dim_warp = warp % G::kDimWarps, token_warp = warp / G::kDimWarps;
  uint32_t unset = 0;  // a bit for each ref of a row that has seen no key (its ref is 0)
  bool fresh = true;
  int first_tile = 0;
  int key_stage = 0, value_stage = 0;   // of tile i
  for (int i = 0; i < count; ++i) {
    if (__builtin_expect(fresh, 0)) {
      if (i > 0) query();
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        ref[j][0] = ref[j][1] = l[j][0] = l[j][1] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k][j][0] = o[k][j][1] = o[k][j][2] = o[k][j][3] = 0.f;
      }
      unset = (1u << 2 * NQ) - 1;
      first_tile = cur.tile;
      fresh = false;
      if (i == 0) cp_async_wait<G::kAhead - 1>();
      __syncthreads();
    }
    const uint32_t keys = sm + key_stage * G::kSide, vals = sm + G::kOffV + value_stage * G::kSide;
    const int pos0 = cur.tile * kTile;
    const bool masked_rows = pos0 + kTile - 1 > cur.len - p.q_len;  // some row does not see some token of the tile
    uint32_t words[kWords];
#pragma unroll
    for (int k = 0; k < kWords; ++k) words[k] = there[value_stage][k];
    uint32_t all_there = words[0], ok_bits = words[0];
#pragma unroll
    for (int k = 1; k < kWords; ++k) all_there &= words[k], ok_bits = kBlocks * warp / 2 == k ? words[k] : ok_bits;
    ok_bits >>= 16 * (kBlocks * warp % 2);  // this warp's tokens
    const int value_free = value_stage == 0 ? G::kValueStages - 1 : value_stage - 1;  // the last tile's
    if (i + G::kAhead < count) place(next, places, value_free);
    next = look(i + G::kAhead + 1);
    if (__builtin_expect(masked_rows, 0) && tid < kTile) {
      // values that are not finite may be hidden from some rows only: they leave the product (a weight of zero would not
      // keep them out), and the rows that see one get their NaN afterwards.  A group's values are finite if those of its least
      // and its greatest nibble are.  (The writer makes no others but NaN; in a group from elsewhere that could hold an infinity
      // every value counts as NaN here.)
#pragma unroll
      for (int gr = 0; gr < D / 64; ++gr) {
        const uint32_t at = vals + kTile * G::kRow + tid * G::kScale + 4 * gr;
        const uint32_t sc = lds32(at);
        const float s = bf16_lo(sc), c = bf16_hi(sc);
        constexpr float kEnd = 3.39617752923046e38f;  // 2^128 - 2^119, from which on a sum rounds to an infinite bf16 number
        const bool is_bad = !(fabsf(fmaf(16.f, s, c)) < kEnd && fabsf(fmaf(31.f, s, c)) < kEnd);
        if (is_bad) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(0u) : "memory");
        const uint32_t bits = __ballot_sync(0xffffffffu, is_bad);
        if (lane == 0) bad[i & 1][gr][warp] = bits;
      }
    }

    // ---- scores of this warp's tokens ----
    float x[kBlocks][NQ][4];
#pragma unroll
    for (int blk = 0; blk < kBlocks; ++blk) {
      // sums of their own for every second half group where there are few to take turns
      constexpr int kChains = NQ <= 2 ? 2 : 1;
      float y[kChains][NQ][4];
#pragma unroll
      for (int c = 0; c < kChains; ++c)
#pragma unroll
        for (int j = 0; j < NQ; ++j) y[c][j][0] = y[c][j][1] = y[c][j][2] = y[c][j][3] = 0.f;
      const uint32_t token0 = 16 * (kBlocks * warp + blk);
      const uint32_t scales = keys + kTile * G::kRow + (token0 + g) * G::kScale;
#pragma unroll
      for (int gr = 0; gr < D / 64; ++gr) {
        uint32_t w[4];
        // ldmatrix: lanes 0-15 a chunk's rows, 16-31 the next chunk's
        ldsm_x4(keys + chunk_at<G::kRow>(token0 + (lane & 15), 2 * gr + (lane >> 4)), w[0], w[1], w[2], w[3]);
        const uint32_t sa = lds32(scales + 4 * gr), sb = lds32(scales + 8 * G::kScale + 4 * gr);
        const uint32_t ssa = dup_lo(sa), cca = dup_hi(sa), ssb = dup_lo(sb), ccb = dup_hi(sb);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 q[NQ];
#pragma unroll
          for (int j = 0; j < NQ; ++j) q[j] = reinterpret_cast<const uint4*>(smem + G::kOffQ)[((2 * gr + h) * NQ + j) * 32 + lane];
          const uint32_t a0 = kv4_pair<0>(w[2 * h], ssa, cca), a1 = kv4_pair<0>(w[2 * h + 1], ssb, ccb);
          const uint32_t a2 = kv4_pair<1>(w[2 * h], ssa, cca), a3 = kv4_pair<1>(w[2 * h + 1], ssb, ccb);
          const uint32_t b0 = kv4_pair<2>(w[2 * h], ssa, cca), b1 = kv4_pair<2>(w[2 * h + 1], ssb, ccb);
          const uint32_t b2 = kv4_pair<3>(w[2 * h], ssa, cca), b3 = kv4_pair<3>(w[2 * h + 1], ssb, ccb);
#pragma unroll
          for (int j = 0; j < NQ; ++j) mma(y[0][j], a0, a1, a2, a3, q[j].x, q[j].y);
#pragma unroll
          for (int j = 0; j < NQ; ++j) mma(y[kChains - 1][j], b0, b1, b2, b3, q[j].z, q[j].w);
        }
      }
      // distances to the reference: the weights are 2^x from here on
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[blk][j][e] = fmaf(kChains == 2 ? y[0][j][e] + y[kChains - 1][j][e] : y[0][j][e], p.scale_log2, -ref[j][e & 1]);
    }
    if (__builtin_expect(masked_rows || ~all_there, 0)) {
#pragma unroll
      for (int blk = 0; blk < kBlocks; ++blk) {
        const int ta = 16 * (kBlocks * warp + blk) + g;
        const bool oka = ok_bits >> (16 * blk + g) & 1, okb = ok_bits >> (16 * blk + g + 8) & 1;
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int last = cur.len - p.q_len + row_query[8 * j + 2 * t + e] - pos0;  // the last token that the row sees
            if (!(oka && ta <= last)) x[blk][j][e] = -INFINITY;
            if (!(okb && ta + 8 <= last)) x[blk][j][2 + e] = -INFINITY;
          }
      }
    }
    // the largest of a row's distances in this thread
    auto highest = [&](int j, int e) {
      float v = fmaxf(x[0][j][e], x[0][j][2 + e]);
#pragma unroll
      for (int blk = 1; blk < kBlocks; ++blk) v = fmaxf(v, fmaxf(x[blk][j][e], x[blk][j][2 + e]));
      return v;
    };
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NQ; ++j) top = fmaxf(top, fmaxf(highest(j, 0), highest(j, 1)));
    if (__builtin_expect(unset != 0, 0))
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (unset >> (2 * j + e) & 1 && highest(j, e) > -INFINITY) top = INFINITY;
    // (all warps have read this tile's keys and the last one's values, whose stages are filled again now)
    const bool raise = __syncthreads_or(top > kNear);
    copy(i + G::kAhead, places, key_stage, value_free);
    float scale_o[NQ][2];
    if (__builtin_expect(raise, 0)) {
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float v[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          v[e] = highest(j, e);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) v[e] = fmaxf(v[e], __shfl_xor_sync(0xffffffffu, v[e], off));
        }
        if (g == 0) *reinterpret_cast<float2*>(&red[warp][8 * j + 2 * t]) = make_float2(v[0], v[1]);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float v[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 r = *reinterpret_cast<const float2*>(&red[k][8 * j + 2 * t]);
          v[0] = fmaxf(v[0], r.x), v[1] = fmaxf(v[1], r.y);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t bit = 1u << (2 * j + e);
          // a row's first reference goes by its maximum so far, whatever its sign; later ones only rise
          const float rise = !(unset & bit) ? fmaxf(v[e] + kAbove, 0.f) : v[e] == -INFINITY ? 0.f : v[e] + kAbove;
          scale_o[j][e] = unset & bit ? 1.f : ex2_approx(-rise);  // (sums of an unset row are zero, or NaN for good)
          if (v[e] > -INFINITY) unset &= ~bit;
          l[j][e] *= scale_o[j][e];
          ref[j][e] += rise;
#pragma unroll
          for (int blk = 0; blk < kBlocks; ++blk) x[blk][j][e] -= rise, x[blk][j][2 + e] -= rise;
        }
      }
    }
#pragma unroll
    for (int blk = 0; blk < kBlocks; ++blk)
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float(&w)[4] = x[blk][j];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = ex2_approx(w[e]);
        l[j][0] += w[0] + w[2], l[j][1] += w[1] + w[3];
        stsm_x2_trans(sm + G::kOffP + (8 * j + (lane & 7)) * G::kPRow + 2 * (16 * (kBlocks * warp + blk) + (lane & 8)),
                      pack2(w[0], w[1]), pack2(w[2], w[3]));
      }
    cp_async_wait<G::kAhead - 1>();  // the next tile
    __syncthreads();                 // weights; and the next tile for all warps

    // ---- O^T += V^T P^T: 64 dimensions of this warp ----
    if (__builtin_expect(raise, 0))
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[k][j][e] *= scale_o[j][e & 1];
    constexpr int kValueBlocks = kTile / 16 / G::kTokenWarps;
    uint32_t pb[NQ][4];
#pragma unroll
    for (int kb = 0; kb < kValueBlocks; ++kb) {
      const int token0 = 16 * (token_warp * kValueBlocks + kb);
      uint32_t w[4];
      ldsm_x4_trans(vals + chunk_at<G::kRow>(token0 + (lane & 15), 2 * dim_warp + (lane >> 4)), w[0], w[1],
                    w[2], w[3]);
      const uint32_t scales = vals + kTile * G::kRow + (token0 + 2 * t) * G::kScale + 4 * dim_warp;
      const uint32_t s0 = lds32(scales), s1 = lds32(scales + G::kScale), s2 = lds32(scales + 8 * G::kScale),
                     s3 = lds32(scales + 9 * G::kScale);
      const uint32_t ssa = __byte_perm(s0, s1, 0x5410), cca = __byte_perm(s0, s1, 0x7632);
      const uint32_t ssb = __byte_perm(s2, s3, 0x5410), ccb = __byte_perm(s2, s3, 0x7632);
      if constexpr (kValueBlocks > 1) {
        if (kb % 2 == 0)  // this block's weights and the next one's
#pragma unroll
          for (int j = 0; j < NQ; ++j)
            ldsm_x4(sm + G::kOffP + (8 * j + (lane & 7)) * G::kPRow + 2 * (token0 + (lane & 24)), pb[j][0], pb[j][1], pb[j][2],
                    pb[j][3]);
      } else {
        const uint8_t* weights = smem + G::kOffP + g * G::kPRow + 2 * (token0 + 2 * t);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          pb[j][0] = *reinterpret_cast<const uint32_t*>(weights + 8 * j * G::kPRow);
          pb[j][1] = *reinterpret_cast<const uint32_t*>(weights + 8 * j * G::kPRow + 16);
        }
      }
      auto times = [&](auto place_k) {
        constexpr int K = decltype(place_k)::value;
        const uint32_t a0 = kv4_pair<K>(w[0], ssa, cca), a1 = kv4_pair<K>(w[2], ssa, cca);
        const uint32_t a2 = kv4_pair<K>(w[1], ssb, ccb), a3 = kv4_pair<K>(w[3], ssb, ccb);
#pragma unroll
        for (int j = 0; j < NQ; ++j) mma(o[K][j], a0, a1, a2, a3, pb[j][2 * (kb % 2)], pb[j][2 * (kb % 2) + 1]);
      };
      times(std::integral_constant<int, 0>{}), times(std::integral_constant<int, 1>{});
      times(std::integral_constant<int, 2>{}), times(std::integral_constant<int, 3>{});
    }
    if (__builtin_expect(masked_rows, 0)) {
#pragma unroll
      for (int k = 0; k < kWords; ++k)
        if (const uint32_t bits = bad[i & 1][dim_warp][k])
          for (int j = 0; j < NQ; ++j)
            for (int e = 0; e < 2; ++e) {
              const int last = cur.len - p.q_len + row_query[8 * j + 2 * t + e] - pos0 - 32 * k;
              if (last >= 0 && (bits & (last >= 31 ? ~0u : (2u << last) - 1)))
                for (int m = 0; m < 4; ++m) o[m][j][e] = o[m][j][2 + e] = __int_as_float(0x7fffffff);
            }
    }

    // ---- the end of a (request, head), or of this CTA's share of it ----
    const bool last_tile = cur.tile + 1 == cur.tiles;
    if (__builtin_expect(last_tile || i + 1 == count, 0)) {
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], off);
      if (g == 0)
#pragma unroll
        for (int j = 0; j < NQ; ++j)
          *reinterpret_cast<float2*>(&red[warp][8 * j + 2 * t]) = make_float2(l[j][0], l[j][1]);
      // the token warps' sums, in halves
      float4* sums = reinterpret_cast<float4*>(smem + G::kOffQ);
#pragma unroll
      for (int half = G::kTokenWarps / 2; half >= 1; half /= 2) {
        if (half < G::kTokenWarps / 2) __syncthreads();
        if (token_warp >= half && token_warp < 2 * half)
#pragma unroll
          for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              sums[(((token_warp - half) * G::kDimWarps + dim_warp) * NQ * 4 + j * 4 + k) * 32 + lane] =
                  make_float4(o[k][j][0], o[k][j][1], o[k][j][2], o[k][j][3]);
        __syncthreads();
        if (token_warp < half)
#pragma unroll
          for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float4 v = sums[((token_warp * G::kDimWarps + dim_warp) * NQ * 4 + j * 4 + k) * 32 + lane];
              o[k][j][0] += v.x, o[k][j][1] += v.y, o[k][j][2] += v.z, o[k][j][3] += v.w;
            }
      }
      if (G::kTokenWarps == 1) __syncthreads();  // the sums l
      if (token_warp == 0) {
        const bool whole = first_tile == 0 && last_tile;
        // a share that begins with the CTA's is its first, else its last
        const int64_t part = 2 * static_cast<int64_t>(blockIdx.x) + (i + 1 - (cur.tile + 1 - first_tile) == 0 ? 0 : 1);
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * j + 2 * t + e;
            if (r >= p.rows) continue;
            const float sum = red[0][r] + red[1][r] + red[2][r] + red[3][r];
            const int d = 64 * dim_warp + 4 * g;
            if (whole) {
              const float n = sum == 0.f ? 0.f : 1.f / sum;  // no key: zeros
              const int qi = row_query[r], hq = cur.h * p.group + r - qi * p.group;
              __nv_bfloat16* dst = p.out + (static_cast<int64_t>(cur.b) * p.q_len + qi) * p.ot + hq * p.oh + d;
              *reinterpret_cast<uint2*>(dst) =
                  make_uint2(pack2(o[0][j][e] * n, o[1][j][e] * n), pack2(o[2][j][e] * n, o[3][j][e] * n));
              *reinterpret_cast<uint2*>(dst + 32) = make_uint2(pack2(o[0][j][2 + e] * n, o[1][j][2 + e] * n),
                                                               pack2(o[2][j][2 + e] * n, o[3][j][2 + e] * n));
            } else {
              float* dst = p.part_o + (part * p.rows + r) * D + d;
              *reinterpret_cast<float4*>(dst) = make_float4(o[0][j][e], o[1][j][e], o[2][j][e], o[3][j][e]);
              *reinterpret_cast<float4*>(dst + 32) =
                  make_float4(o[0][j][2 + e], o[1][j][2 + e], o[2][j][2 + e], o[3][j][2 + e]);
              if (dim_warp == 0 && g == 0) p.part_ml[part * p.rows + r] = make_float2(unset >> (2 * j + e) & 1 ? kNoRef : ref[j][e], sum);
            }
          }
      }
      if (i + 1 == count && tid == 0) {
        // the CTA that begins a (request, head) which others end names it for the join
        const bool open = first_tile == 0 && !last_tile;
        const uint32_t last = end - 1 + (cur.tiles - 1 - cur.tile);  // the position of its last tile
        p.joins[blockIdx.x] = open ? make_int4(cur.b, cur.h, Shares(total, ctas).holder(last), cur.tile + 1 == count ? 0 : 1)
                                   : make_int4(-1, 0, 0, 0);
      }
      fresh = true;
      __syncthreads();  // the query's place and `red` are free again
    }
    if (i + 1 < count) cur.next(p);
    if (++key_stage == G::kKeyStages) key_stage = 0;
    if (++value_stage == G::kValueStages) value_stage = 0;
  }
}

// Joins the parts of each (request, head) that several CTAs held.  Work is a (join, row, 64 dimensions), 16 threads with four
// dimensions each; several such groups share the parts of one where there are many (a long context), or take one each where
// there are few (a batch).  A CTA takes a round of work of one join at a time.
constexpr int kJoinThreads = 256, kJoinDims = 64, kJoinGroups = kJoinThreads / (kJoinDims / 4), kJoinEarly = 8;
constexpr int kMaxCtas = 4;  // of an SM

// Groups that share a piece of work.
__device__ __forceinline__ int join_share(int parts) {
  int n = 1;
  while (n < kJoinGroups && n * 4 < parts) n *= 2;
  return n;
}

__global__ void __launch_bounds__(kJoinThreads) kv4_join_kernel(const AttnParams p, int grid, int D) {
  __shared__ int4 list[kMaxSms * kMaxCtas];
  __shared__ int rounds[kMaxSms * kMaxCtas + 1];  // before each join
  __shared__ int2 warp_sum[kJoinThreads / 32];
  __shared__ float weight[kJoinGroups][kMaxSms * kMaxCtas / 4];
  __shared__ float4 sums[kJoinGroups][kJoinDims / 4];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pieces = D / kJoinDims, work = p.rows * pieces;
  constexpr int kLists = (kMaxSms * kMaxCtas + kJoinThreads - 1) / kJoinThreads;
  int4 joins[kLists];  // all on their way at once
#pragma unroll
  for (int i = 0; i < kLists; ++i) {
    joins[i] = make_int4(-1, 0, 0, 0);
    if (i * kJoinThreads + tid < grid) joins[i] = p.joins[i * kJoinThreads + tid];
  }
  int n = 0, total = 0;
#pragma unroll
  for (int i = 0; i < kLists; ++i) {
    const int from = i * kJoinThreads + tid;
    const int4 join = joins[i];
    const bool named = join.x >= 0;
    const int share = join_share(join.z - from + 1);
    int2 sum = make_int2(named, named ? (work * share + kJoinGroups - 1) / kJoinGroups : 0);
    const int2 own = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, sum.x, off), c = __shfl_up_sync(0xffffffffu, sum.y, off);
      if (lane >= off) sum.x += a, sum.y += c;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    int at = n + sum.x - own.x, before = total + sum.y - own.y;
    for (int w = 0; w < kJoinThreads / 32; ++w) {
      const int2 v = warp_sum[w];
      if (w < warp) at += v.x, before += v.y;
      n += v.x, total += v.y;
    }
    if (named) {
      // (request and head, the CTA that begins it, the last one, whether its part is the first's last share)
      list[at] = make_int4(join.x * p.heads + join.y, from, join.z, join.w);
      rounds[at] = before;
    }
    __syncthreads();
  }
  const int col = tid % (kJoinDims / 4), group = tid / (kJoinDims / 4);
  for (int round = blockIdx.x; round < total; round += gridDim.x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (rounds[mid] <= round) lo = mid; else hi = mid - 1;
    }
    const int4 join = list[lo];
    const int parts = join.z - join.y + 1, share = join_share(parts);
    const int item = (round - rounds[lo]) * (kJoinGroups / share) + group / share, sub = group % share;
    const bool active = item < work;
    const int piece = item % pieces, r = active ? item / pieces : 0;
    // part k is CTA join.y + k's first, or its last where the (request, head) begins inside its share
    auto row_of = [&](int k) { return (2 * static_cast<int64_t>(join.y + k) + (k == 0 ? join.w : 0)) * p.rows + r; };
    auto load = [&](int k) {
      return *reinterpret_cast<const float4*>(p.part_o + row_of(k) * D + kJoinDims * piece + 4 * col);
    };
    float4 early[kJoinEarly];  // this group's parts sub, sub + share, ..., on their way while the weights are made
#pragma unroll
    for (int e = 0; e < kJoinEarly; ++e) {
      early[e] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (active && sub + e * share < parts) early[e] = load(sub + e * share);
    }
    // the weights of the row (every group that shares it makes them all, and keeps its own)
    float top = kNoRef, sum = 0.f;
    float2 ml[kJoinEarly];
#pragma unroll
    for (int e = 0; e < kJoinEarly; ++e) {
      const int k = col + e * (kJoinDims / 4);
      ml[e] = make_float2(kNoRef, 0.f);
      if (k < parts) ml[e] = p.part_ml[row_of(k)];
    }
#pragma unroll
    for (int e = 0; e < kJoinEarly; ++e) top = fmaxf(top, ml[e].x);
    for (int k = col + kJoinEarly * (kJoinDims / 4); k < parts; k += kJoinDims / 4) top = fmaxf(top, p.part_ml[row_of(k)].x);
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    auto weigh = [&](int k, const float2& v) {
      const float w = ex2_approx(v.x - top);
      if (k % share == sub) weight[group][k / share] = w;
      sum = fmaf(v.y, w, sum);
    };
#pragma unroll
    for (int e = 0; e < kJoinEarly; ++e)
      if (const int k = col + e * (kJoinDims / 4); k < parts) weigh(k, ml[e]);
    for (int k = col + kJoinEarly * (kJoinDims / 4); k < parts; k += kJoinDims / 4) weigh(k, p.part_ml[row_of(k)]);
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    __syncwarp();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, float w) {
      acc.x = fmaf(v.x, w, acc.x), acc.y = fmaf(v.y, w, acc.y), acc.z = fmaf(v.z, w, acc.z), acc.w = fmaf(v.w, w, acc.w);
    };
    if (active) {
#pragma unroll
      for (int e = 0; e < kJoinEarly; ++e)
        if (sub + e * share < parts) add(early[e], weight[group][e]);
#pragma unroll 4
      for (int k = sub + kJoinEarly * share; k < parts; k += share) add(load(k), weight[group][k / share]);
    }
    if (share > 1) {
      sums[group][col] = acc;
      __syncthreads();
      if (sub == 0)
        for (int k = 1; k < share; ++k) add(sums[group + k][col], 1.f);
      __syncthreads();
    }
    if (active && sub == 0) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int b = join.x / p.heads, h = join.x - b * p.heads;
      const int qi = r / p.group, hq = h * p.group + r - qi * p.group;
      __nv_bfloat16* dst = p.out + (static_cast<int64_t>(b) * p.q_len + qi) * p.ot + hq * p.oh + kJoinDims * piece + 4 * col;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(acc.x * inv, acc.y * inv), pack2(acc.z * inv, acc.w * inv));
    }
    __syncwarp();
  }
}

int tiles_of_rows(int rows) {
  const int n = (rows + 7) / 8;
  return n == 5 ? 6 : n == 7 ? 8 : n;
}

template <int D, int NQ> cudaError_t launch(const AttnParams& p, int grid, int dev, int sms, bool pdl, cudaStream_t st) {
  using G = Geo<D, NQ>;
  static std::mutex mu;
  static bool set[64] = {};
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!set[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(kv4_attn_kernel<D, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
      if (e != cudaSuccess) return e;
      set[dev] = true;
    }
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = G::kSmem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_attn_kernel<D, NQ>, p);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * sms));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel, p, grid, D);
}

template <int D> cudaError_t launch(const AttnParams& p, int grid, int dev, int sms, bool pdl, cudaStream_t st) {
  switch (tiles_of_rows(p.rows)) {
    case 1: return launch<D, 1>(p, grid, dev, sms, pdl, st);
    case 2: return launch<D, 2>(p, grid, dev, sms, pdl, st);
    case 3: return launch<D, 3>(p, grid, dev, sms, pdl, st);
    case 4: return launch<D, 4>(p, grid, dev, sms, pdl, st);
    case 6: return launch<D, 6>(p, grid, dev, sms, pdl, st);
    default: return launch<D, 8>(p, grid, dev, sms, pdl, st);
  }
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace qf

using namespace qf;

extern "C" size_t qf_kv4_attn_workspace_bytes(int num_reqs, int q_len, int num_heads, int num_kv_heads, int head_size) {
  if (num_reqs <= 0 || q_len <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_size <= 0) return 256;
  const int64_t rows = static_cast<int64_t>(q_len) * (num_heads / num_kv_heads);
  const size_t parts = 2 * static_cast<size_t>(kMaxSms) * ctas_per_sm(head_size, tiles_of_rows(static_cast<int>(rows < 64 ? rows : 64)));
  return up256(parts / 2 * sizeof(int4)) + up256(parts * rows * 8) + parts * rows * head_size * 4;
}

extern "C" int qf_kv4_attn(const void* q, int64_t sq_t, int64_t sq_h, const qf_kv4_cache* cache,
                           const int32_t* block_table, int64_t s_bt, int max_pages, const int32_t* seq_lens, void* out,
                           int64_t so_t, int64_t so_h, int num_reqs, int q_len, int num_heads, float scale, void* ws,
                           size_t ws_bytes, unsigned flags, void* stream) {
  AttnParams p = {};
  Kv4View c;
  int rc = kv4_view(cache, &c);
  if (rc) return rc;
  if (num_reqs < 0 || q_len < 1 || num_heads < 0 || max_pages < 0) return fail(QF_ERR_SHAPE, "sizes");
  if (num_heads % cache->num_heads) return fail(QF_ERR_SHAPE, "query heads must be a multiple of the cache's heads");
  if (static_cast<int64_t>(q_len) * (num_heads / cache->num_heads) > 64)
    return fail(QF_ERR_SHAPE, "more than 64 query rows for a key head");
  if (static_cast<int64_t>(num_reqs) * q_len > INT32_MAX / 64 || num_heads > 65535 ||
      static_cast<int64_t>(num_reqs) * cache->num_heads > INT32_MAX)
    return fail(QF_ERR_SHAPE, "too many query rows");
  const int64_t tiles = static_cast<int64_t>(max_pages) * cache->page_size / 64 + 4;
  if (static_cast<int64_t>(num_reqs) * cache->num_heads > INT32_MAX / (tiles < INT32_MAX ? tiles : INT32_MAX))
    return fail(QF_ERR_SHAPE, "more keys than 2^31 tiles of 64 (requests, heads and the table's width together)");
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
  int dev = 0, sms = 0;
  rc = require_b200(&dev, &sms);
  if (rc) return rc;
  p.q = static_cast<const __nv_bfloat16*>(q), p.qt = sq_t, p.qh = sq_h;
  p.out = static_cast<__nv_bfloat16*>(out), p.ot = so_t, p.oh = so_h;
  p.table = block_table, p.table_row = s_bt;
  p.width = static_cast<int64_t>(max_pages) * cache->page_size;
  if (p.width > INT32_MAX - 1024) p.width = INT32_MAX - 1024;  // positions stay 32-bit numbers
  p.codes = c.codes[0], p.scales = c.scale[0];
  p.value_codes = c.codes[1] - c.codes[0], p.value_scales = c.scale[1] - c.scale[0];
  p.head = c.head, p.shead = c.shead;
  p.page = c.page, p.slot = c.slot, p.spage = c.spage, p.sslot = c.sslot;
  p.div_mul = c.div_mul, p.div_shift = c.div_shift;
  if (c.num_pages == 0) {  // nothing is read, but addresses are formed
    p.codes = p.scales = static_cast<const uint8_t*>(q);
    p.value_codes = p.value_scales = 0;
  }
  p.num_pages = c.num_pages, p.page_size = c.page_size, p.heads = c.heads;
  p.lens = seq_lens;
  p.reqs = num_reqs, p.q_len = q_len, p.group = num_heads / cache->num_heads, p.rows = q_len * p.group;
  p.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  if (sms > kMaxSms) sms = kMaxSms;
  const int grid = sms * ctas_per_sm(cache->head_size, tiles_of_rows(p.rows));
  const size_t parts = 2 * static_cast<size_t>(kMaxSms) * ctas_per_sm(cache->head_size, tiles_of_rows(p.rows));
  uint8_t* w = static_cast<uint8_t*>(ws);
  p.joins = reinterpret_cast<int4*>(w);
  w += up256(parts / 2 * sizeof(int4));
  p.part_ml = reinterpret_cast<float2*>(w);
  w += up256(parts * p.rows * 8);
  p.part_o = reinterpret_cast<float*>(w);
  const bool pdl = (flags & QF_FLAG_PDL) != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = cache->head_size == 64    ? launch<64>(p, grid, dev, sms, pdl, st)
                        : cache->head_size == 128 ? launch<128>(p, grid, dev, sms, pdl, st)
                                                  : launch<256>(p, grid, dev, sms, pdl, st);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}
