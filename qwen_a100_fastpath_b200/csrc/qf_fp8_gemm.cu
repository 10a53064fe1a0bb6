// qf_fp8_gemm.cu -- e4m3 x e4m3 product with one fp32 scale for each 128 elements along k (and each 128 output
// channels of the weight).
//
// Mathematics: y[m, n] = sum_g sa[m, g] * sw[n / 128, g] * P_g[m, n], P_g = sum over the 128 k of group g of
// a[m, k] * w[n, k].  Products of e4m3 values are exact in fp32; each P_g is summed by the tensor cores in fp32 and
// folded into fp32 sums with one multiply-add per group and output.
//
// fp8_tile_kernel (more than 16 token rows): 128 token rows x BN channels on tcgen05 kind::f8f6f4, one tensor-memory
// accumulator per k group; two producer and two issuing warps feed it from a ring of TMA stages (128-byte rows, 128-byte
// swizzle), eight warps add each finished accumulator, times its scales, to fp32 sums in registers while the next
// groups are multiplied.  With fewer tiles than SMs a cluster shares a tile's groups and adds its parts over distributed
// shared memory, in rank order.  What bounds it over many groups: one of 64 / 128 / 256 channels takes a CTA
// 0.30 / 0.38 / 0.52 us, of which shared memory's 128 bytes a clock (copies in, operands out: 2 x (16 KiB + BN * 128)) are
// 0.20 / 0.26 / 0.39 and the rest, the same at every width, is about one barrier wait.  A short share of groups costs
// more (starts and the join of a split).  Measured (us, B200, in a graph): 72 x 10240 x 5120 18.2 (40 tiles x 3 CTAs; 17.8
// with its weights in L2); 333 x 2600 x 1160 7.9; 2048 x 5120 x 8192 119 (three rounds of tiles, the last of 24); 4096 x
// 34816 x 5120 767 (1.90 PFLOP/s; 915 in a loop under the power cap).
//
// fp8_rows_kernel (up to 16): bound by the weights' bytes.  A CTA takes tiles of 16 or 32 weight rows, a producer copies
// four or eight k groups of them and of the token rows per stage into a ring (one TMA copy each: a copy costs its issuer
// and the TMA unit the same whatever it moves), and each of four warps multiplies one or two of the stage's groups with
// mma.sync m16n8k32 (weights as the 16-row operand, so that 8 token columns are not padded to a tcgen05 tile); the
// warps' sums are added in shared memory in warp order.  Three CTAs per SM hold rings of 144 to 192 KiB together, token rows
// included.  Measured (us, B200, in a graph): 1 x 5120 x 8192 10.5; 5 x 34816 x 5120 29.9 (6.0 TB/s); 1 x 5120 x 17408
// 18.7; 16 x 10240 x 5120 14.8.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/qf_b200.h"
#include "qf_fp8.cuh"
#include "qf_host.h"
#include "qf_ptx.cuh"

namespace qf {
namespace {

constexpr int kRowWarps = 4;

struct Fp8Params {
  const uint8_t* a;
  int64_t lda;
  const float* sa;
  int64_t sa_m, sa_g;
  const uint8_t* w;
  int64_t ldw;
  const float* sw;
  int64_t sw_n, sw_g;
  const __nv_bfloat16* bias;
  void* y;
  int64_t ldy;
  int y_f32;
  int M, N, K, kb;
};

constexpr long long kFp8WaitClocks = 8000000000ll;  // about 4 s; the global timer would cost each poll its read

__device__ int g_fp8_err;  // sticky: QF_ERR_TIMEOUT once a bounded wait expired (read by qf_fp8_status)

__device__ __forceinline__ bool fp8_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (*abort_flag) return false;
    if (mbar_try_wait(bar, parity)) return true;
    if (clock64() - t0 > kFp8WaitClocks) {
      atomicExch(&g_fp8_err, QF_ERR_TIMEOUT);
      *abort_flag = 1;
      return false;
    }
  }
}

// The same by a whole warp, which goes on together: at once, or with lane 0's bounded wait.
__device__ __forceinline__ bool fp8_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  int have = 0;
  if ((threadIdx.x & 31) == 0) have = fp8_wait(bar, parity, abort_flag) ? 1 : 0;
  return __shfl_sync(0xffffffffu, have, 0) != 0;
}

// ---------------------------------------------------------------------------------------------- few token rows
constexpr int kRowPerSm = 3;

// A tile of 16 * MT weight rows and 8 * NT tokens; a stage holds G k groups for each warp: [group][weight rows]
// [128 bytes], then [group][token rows][128 bytes].
template <int NT, int MT, int G> struct RowGeo {
  static constexpr int kRows = 16 * MT;
  static constexpr int kGroups = kRowWarps * G;
  static constexpr int kWBytes = kGroups * kRows * kFp8Block;
  static constexpr int kABytes = kGroups * 8 * NT * kFp8Block;
  static constexpr int kStage = kWBytes + kABytes;
  static constexpr int kSum = kRowWarps * NT * MT * 128;     // floats of the warps' sums
  static constexpr int kStages = (224 * 1024 / kRowPerSm - 2048 - kSum * 4) / kStage;
  static constexpr int kSmemBytes = kStages * kStage + kSum * 4 + 1024;
  static_assert(kStages >= 2 && kSmemBytes <= 227 * 1024 / kRowPerSm - 1024, "shared memory");
};

// 16 bytes of an operand row from column k; bytes past K read as zero and are not touched.
__device__ __forceinline__ uint4 load_chunk(const uint8_t* row, int k, int K) {
  if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) w[i / 4] |= static_cast<uint32_t>(row[k + i]) << (8 * (i % 4));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Scales of a warp's k group: the weight block's, tokens' 2t and 2t + 1 of each 8.
template <int NT> struct RowScales {
  float sw, sa[NT][2];
};

// One finished output, with its bias.
__device__ __forceinline__ void store_row_sum(const Fp8Params& p, int n, int m, float v) {
  if (n >= p.N || m >= p.M) return;
  if (p.bias) v += __bfloat162float(p.bias[n]);
  const int64_t at = static_cast<int64_t>(m) * p.ldy + n;
  if (p.y_f32)
    static_cast<float*>(p.y)[at] = v;
  else
    static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
}

template <int NT, int MT, int G>
__global__ void __launch_bounds__(kRowWarps * 32 + 32, kRowPerSm)
    fp8_rows_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                    const Fp8Params p, int ntiles) {
  using C = RowGeo<NT, MT, G>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[C::kStages], empty[C::kStages];
  __shared__ volatile int abort_flag, leave;
  float* red = reinterpret_cast<float*>(ring + C::kStages * C::kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.y * (8 * NT);
  const int kfull = p.K / kFp8Block;  // groups that are copied; a shorter last one is read where it is used
  const int nst = (kfull + C::kGroups - 1) / C::kGroups;
  if (threadIdx.x == 0) {
    if (nst > 0) {  // without a whole k group there are no maps
      prefetch_tensormap(&tmap_w);
      prefetch_tensormap(&tmap_a);
    }
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kRowWarps);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_launch_dependents();
  if (warp == kRowWarps) {
    if (lane == 0) {
      const uint64_t pol_w = policy_evict_first();
      const uint64_t pol_a = policy_evict_last();
      // the first stages' weights into L2 while the kernel before this one ends (no value is read before the wait)
      for (int st = 0; st < min(C::kStages, nst); ++st)
        tma_prefetch_3d(&tmap_w, 0, static_cast<int>(blockIdx.x) * C::kRows, st * C::kGroups);
      pdl_wait();
      int issued = 0, s = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int tile = blockIdx.x; tile < ntiles && ok; tile += gridDim.x) {
        for (int st = 0; st < nst; ++st, ++issued) {
          if (!fp8_wait(&empty[s], phase, &abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* dst = ring + s * C::kStage;
          mbar_arrive_expect_tx(&full[s], C::kStage);
          tma_load_3d(dst, &tmap_w, &full[s], 0, tile * C::kRows, st * C::kGroups, pol_w);
          tma_load_3d(dst + C::kWBytes, &tmap_a, &full[s], 0, m0, st * C::kGroups, pol_a);
          if (++s == C::kStages) s = 0, phase ^= 1;
        }
      }
      // every copy issued lands before the shared memory is given up
      for (int i = issued > C::kStages ? issued - C::kStages : 0; i < issued; ++i) {
        const long long t0 = clock64();
        while (!mbar_try_wait(&full[i % C::kStages], (i / C::kStages) & 1)) {
          if (clock64() - t0 > kFp8WaitClocks) {
            atomicExch(&g_fp8_err, QF_ERR_TIMEOUT);
            abort_flag = 1;
            break;
          }
        }
      }
    }
  } else {
    pdl_wait();
    const int gid = lane >> 2, t = lane & 3;
    // tokens past the end repeat the last one: their products are computed and not stored
    const float* sa_row[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        sa_row[j][i] = p.sa + static_cast<int64_t>(min(m0 + 8 * j + 2 * t + i, p.M - 1)) * p.sa_m;
    // Thread t of a row takes the 16-byte pieces 2t and 2t + 1 of its 128 bytes, at their places under the 128-byte
    // swizzle (piece ^ row % 8): the rows of a quarter warp then fall on different banks.
    const uint32_t base = smem_u32(ring) + static_cast<uint32_t>(gid * 128);
    const uint32_t piece[2] = {static_cast<uint32_t>(((2 * t) ^ gid) * 16), static_cast<uint32_t>(((2 * t + 1) ^ gid) * 16)};
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < ntiles && ok; tile += gridDim.x) {
      const int n0 = tile * C::kRows;
      const float* sw_row = p.sw + static_cast<int64_t>(n0 / kFp8Block) * p.sw_n;
      auto load_scales = [&](RowScales<NT>& r, int g) {
        if (g >= p.kb) return;
        r.sw = sw_row[g * p.sw_g];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) r.sa[j][i] = sa_row[j][i][g * p.sa_g];
      };
      float acc[NT][MT][4] = {};
      auto add = [&](const uint4 (&lo)[MT][2], const uint4 (&hi)[MT][2], const uint4 (&b)[NT][2],
                     const float (&sc)[NT][2]) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            float d[2][4] = {};  // two chains of instructions
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              // the thread's 16 bytes stand for the instruction's k slots of two steps, the same ones in both operands
              mma_e4m3_m16n8k32(d[c], lo[i][c].x, hi[i][c].x, lo[i][c].y, hi[i][c].y, b[j][c].x, b[j][c].y);
              mma_e4m3_m16n8k32(d[c], lo[i][c].z, hi[i][c].z, lo[i][c].w, hi[i][c].w, b[j][c].z, b[j][c].w);
            }
            acc[j][i][0] = fmaf(d[0][0] + d[1][0], sc[j][0], acc[j][i][0]);
            acc[j][i][1] = fmaf(d[0][1] + d[1][1], sc[j][1], acc[j][i][1]);
            acc[j][i][2] = fmaf(d[0][2] + d[1][2], sc[j][0], acc[j][i][2]);
            acc[j][i][3] = fmaf(d[0][3] + d[1][3], sc[j][1], acc[j][i][3]);
          }
        }
      };
      // group i of the warp's G in stage st
      auto group_of = [&](int st, int i) { return st * C::kGroups + i * kRowWarps + warp; };
      auto product = [](const RowScales<NT>& r, float (&sc)[NT][2]) {
#pragma unroll
        for (int j = 0; j < NT; ++j) sc[j][0] = r.sw * r.sa[j][0], sc[j][1] = r.sw * r.sa[j][1];
      };
      auto stage = [&](int st, RowScales<NT> (&r)[G]) {
        // the scales of two stages ahead are on their way before the wait (16 x 10240 x 5120 through the linear layer 16.9
        // us; behind the products 18.4)
        float sc[G][NT][2];
#pragma unroll
        for (int u = 0; u < G; ++u) {
          product(r[u], sc[u]);
          load_scales(r[u], group_of(st + 2, u));
        }
        if (!fp8_wait_warp(&full[s], phase, &abort_flag)) {
          ok = false;
          return;
        }
        uint4 lo[G][MT][2], hi[G][MT][2], b[G][NT][2];
#pragma unroll
        for (int u = 0; u < G; ++u) {
          const uint32_t w_at =
              base + static_cast<uint32_t>(s * C::kStage + (u * kRowWarps + warp) * (C::kRows * kFp8Block));
          const uint32_t a_at =
              base + static_cast<uint32_t>(s * C::kStage + C::kWBytes + (u * kRowWarps + warp) * (8 * NT * kFp8Block));
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              lo[u][i][c] = lds128(w_at + 16 * i * kFp8Block + piece[c]);
              hi[u][i][c] = lds128(w_at + (16 * i + 8) * kFp8Block + piece[c]);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) b[u][j][c] = lds128(a_at + 8 * j * kFp8Block + piece[c]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        if (++s == C::kStages) s = 0, phase ^= 1;
#pragma unroll
        for (int u = 0; u < G; ++u)
          if (group_of(st, u) < kfull) add(lo[u], hi[u], b[u], sc[u]);
      };
      RowScales<NT> r0[G] = {}, r1[G] = {};
#pragma unroll
      for (int u = 0; u < G; ++u) {
        load_scales(r0[u], group_of(0, u));
        load_scales(r1[u], group_of(1, u));
      }
      for (int st = 0; st < nst && ok; st += 2) {
        stage(st, r0);
        if (st + 1 < nst && ok) stage(st + 1, r1);
      }
      if (kfull < p.kb && kfull % kRowWarps == warp) {  // the shorter last group
        const int k = kfull * kFp8Block + 32 * t;
        uint4 lo[MT][2], hi[MT][2], b[NT][2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            lo[i][c] = load_chunk(p.w + static_cast<int64_t>(min(n0 + 16 * i + gid, p.N - 1)) * p.ldw, k + 16 * c, p.K);
            hi[i][c] = load_chunk(p.w + static_cast<int64_t>(min(n0 + 16 * i + gid + 8, p.N - 1)) * p.ldw, k + 16 * c, p.K);
          }
#pragma unroll
          for (int j = 0; j < NT; ++j)
            b[j][c] = load_chunk(p.a + static_cast<int64_t>(min(m0 + 8 * j + gid, p.M - 1)) * p.lda, k + 16 * c, p.K);
        }
        load_scales(r0[0], kfull);
        float sc[NT][2];
        product(r0[0], sc);
        add(lo, hi, b, sc);
      }
      // the warps' sums in warp order
      named_bar_sync(1, kRowWarps * 32);  // the tile before is read
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) red[(((warp * NT + j) * MT + i) * 4 + e) * 32 + lane] = acc[j][i][e];
      if (threadIdx.x == 0) leave = abort_flag;
      named_bar_sync(1, kRowWarps * 32);
      // one reading of the flag for all warps: they leave, or go on, with the same barriers behind them
      ok = !leave;
      for (int e = threadIdx.x; e < NT * MT * 128 && ok; e += kRowWarps * 32) {
        const int r = e % C::kRows, tk = e / C::kRows;
        const int src = (r % 8) * 4 + (tk % 8) / 2, reg = (r % 16 / 8) * 2 + (tk & 1);
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) v += red[(((w * NT + tk / 8) * MT + r / 16) * 4 + reg) * 32 + src];
        store_row_sum(p, n0 + r, m0 + tk, v);
      }
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------- tcgen05 tiles
constexpr int kTileM = 128;
// Scales of kScaleK groups at a time, kScaleBufs chunks in flight, in shared memory.
constexpr int kScaleK = 8, kScaleBufs = 3;

constexpr int kMaxStages = 12;

constexpr int kEpiWarps = 8;  // two for each tensor-memory quarter

template <int BN, bool SPLIT> struct TileGeo {
  static constexpr int EW = kEpiWarps;
  static constexpr int kThreads = 128 + 32 * EW;
  static constexpr int kBBytes = BN * kFp8Block;
  // a stage: the weight tile, then the token rows of the tile (fewer than 128 where the call has fewer)
  static constexpr int kRing = 196 * 1024;
  static constexpr int kTmemCols = 512;
  static constexpr int kAccs = kTmemCols / BN;    // one k group each
  static constexpr int kCols = BN * 4 / EW;       // columns per epilogue thread
  static constexpr int kChunks = kCols / 32;
  static constexpr int kOffBar = kRing;
  static constexpr int kNumBars = 2 * kMaxStages + 2 * kAccs + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kOffScale = kOffMisc + 24;
  // a chunk: [group][epilogue thread], then per epilogue warp [group][one of its two weight blocks]
  static constexpr int kScaleBuf = kScaleK * (32 * EW + 2 * EW);
  static constexpr int kSmemBytes = kOffScale + kScaleBufs * kScaleBuf * 4 + 1024;
  static_assert(kCols % 32 == 0 && kCols <= 128, "columns per epilogue thread");
  static_assert(kRing / (kBBytes + kTileM * kFp8Block) >= 4 && kSmemBytes <= 227 * 1024, "shared memory");
  static_assert(!SPLIT || kTileM * BN * 4 <= kRing, "the partial tile reuses the ring");
};

struct TileParams {
  Fp8Params p;
  int mtiles, ntiles, splits;
  int box_rows;  // token rows copied per tile
  int stages;    // of the ring: weight tile and token rows
  int vec_out;
};

// First output row and column of tile t.  Tiles run down the token rows first (bands of 32 tiles, 4096 rows), so that
// the CTAs of a wave share weight tiles through L2 and a band of activations stays there.
__device__ __forceinline__ void tile_origin(const TileParams& tp, int t, int bn, int* m0, int* n0) {
  if (tp.mtiles == 1) {
    *m0 = 0;
    *n0 = t * bn;
    return;
  }
  const int band = tp.mtiles > 32 ? t / (32 * tp.ntiles) : 0;
  const int rows = min(32, tp.mtiles - 32 * band);
  const int in = t - band * 32 * tp.ntiles;
  *m0 = (32 * band + in % rows) * kTileM;
  *n0 = in / rows * bn;
}

__device__ __forceinline__ void store8(const TileParams& tp, int m, int n, const float (&v)[8]) {
  const Fp8Params& p = tp.p;
  float o[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = v[j] + ((p.bias && n + j < p.N) ? __bfloat162float(p.bias[n + j]) : 0.f);
  const int64_t at = static_cast<int64_t>(m) * p.ldy + n;
  if (p.y_f32) {
    float* y = static_cast<float*>(p.y) + at;
    if (tp.vec_out && n + 8 <= p.N) {
      reinterpret_cast<float4*>(y)[0] = make_float4(o[0], o[1], o[2], o[3]);
      reinterpret_cast<float4*>(y)[1] = make_float4(o[4], o[5], o[6], o[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n + j < p.N) y[j] = o[j];
    }
  } else {
    __nv_bfloat16* y = static_cast<__nv_bfloat16*>(p.y) + at;
    if (tp.vec_out && n + 8 <= p.N) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * j], o[2 * j + 1]);
        w[j] = reinterpret_cast<const uint32_t&>(h);
      }
      *reinterpret_cast<uint4*>(y) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n + j < p.N) y[j] = __float2bfloat16_rn(o[j]);
    }
  }
}

template <int BN, bool SPLIT>
__global__ void __launch_bounds__(128 + 32 * kEpiWarps, 1)
    fp8_tile_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                    const __grid_constant__ TileParams tp) {
  using C = TileGeo<BN, SPLIT>;
  constexpr int A = C::kAccs, EW = kEpiWarps;
  const int S = tp.stages;
  const uint32_t stage_bytes = C::kBBytes + static_cast<uint32_t>(tp.box_rows) * kFp8Block;
  const Fp8Params& p = tp.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;
  uint64_t* acc_empty = acc_full + A;
  uint64_t* mma_done = acc_empty + A;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int ntotal = tp.mtiles * tp.ntiles;
  // with SPLIT the cluster's CTAs take one tile and a share of its k groups each
  const int rank = SPLIT ? static_cast<int>(cluster_rank()) : 0;
  const int first = SPLIT ? static_cast<int>(blockIdx.x) / tp.splits : static_cast<int>(blockIdx.x);
  const int step = SPLIT ? ntotal : static_cast<int>(gridDim.x);
  const int k0 = SPLIT ? static_cast<int>(static_cast<int64_t>(p.kb) * rank / tp.splits) : 0;
  const int k1 = SPLIT ? static_cast<int>(static_cast<int64_t>(p.kb) * (rank + 1) / tp.splits) : p.kb;

  const uint64_t pol_w = policy_evict_normal();
  const uint64_t pol_a = policy_evict_last();
  auto copy_group = [&](int s, int kb, int m0, int n0) {
    uint8_t* dst = smem + s * stage_bytes;
    mbar_arrive_expect_tx(&full[s], stage_bytes);
    tma_load_2d(dst, &tmap_w, &full[s], kb * kFp8Block, n0, pol_w);
    tma_load_2d(dst + C::kBBytes, &tmap_a, &full[s], kb * kFp8Block, m0, pol_a);
  };
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tmap_a);
    prefetch_tensormap(&tmap_w);
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < A; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], EW);  // one arrival per epilogue warp
    }
    mbar_init(mma_done, 2);
    *s_abort = 0;
    fence_mbar_init();
    // the first group is on its way before the CTA meets
    pdl_wait();
    int m0, n0;
    tile_origin(tp, first, BN, &m0, &n0);
    copy_group(0, k0, m0, n0);
  }
  if (warp == 2) tmem_alloc(s_tmem, C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  pdl_launch_dependents();  // after the tensor memory is held: a dependent's CTA could otherwise take it and wait for us
  pdl_wait();

  // where an epilogue thread holds more than 64 sums: 168 registers a thread at launch, and the three warpgroups'
  // 56 + 224 + 224 use what the block has
  if (warp < 4) {
    if (C::kCols > 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // A barrier wait takes a producing or issuing lane some 200 clocks even where the barrier is complete, as long as the
    // matrix instructions of a group: two warps take turns in both roles.
    if (warp < 2) {
      if (lane == 0) {
        int it = 0;
        int s = warp;          // stage and phase of this warp's next turn
        uint32_t phase = 0;
        bool ok = true;
        for (int t = first; t < ntotal && ok; t += step) {
          int m0, n0;
          tile_origin(tp, t, BN, &m0, &n0);
          for (int kb = k0; kb < k1; ++kb, ++it) {
            if ((it & 1) != warp) continue;
            if (it > 0) {  // the first group is under way
              if (!fp8_wait(&empty[s], phase ^ 1, s_abort)) {
                ok = false;
                break;
              }
              copy_group(s, kb, m0, n0);
            }
            s += 2;
            if (s >= S) s -= S, phase ^= 1;
          }
        }
        // every copy issued must land before the shared memory is released
        for (int i = it > S ? it - S : 0; i < it; ++i) {
          if ((i & 1) != warp) continue;
          const long long t0 = clock64();
          while (!mbar_try_wait(&full[i % S], static_cast<uint32_t>(i / S) & 1u)) {
            if (clock64() - t0 > kFp8WaitClocks) {
              atomicExch(&g_fp8_err, QF_ERR_TIMEOUT);
              *s_abort = 1;
              break;
            }
          }
        }
      }
      __syncwarp();
    } else {
      if (lane == 0) {
        constexpr uint32_t idesc = idesc_e4m3(kTileM, BN);
        const uint32_t smem_base = smem_u32(smem);
        int it = 0;
        int s = warp - 2;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = first; t < ntotal && ok; t += step) {
          for (int kb = k0; kb < k1; ++kb, ++it) {
            if ((it & 1) != warp - 2) continue;
            const int b = it % A;
            if (!fp8_wait(&acc_empty[b], ((it / A) & 1) ^ 1, s_abort)) {
              ok = false;
              break;
            }
            tc_fence_after();  // after the epilogue's loads (the copies' own barriers need no fence)
            if (!fp8_wait(&full[s], phase, s_abort)) {
              ok = false;
              break;
            }
            const uint32_t w_addr = smem_base + s * stage_bytes;
            // rows of the tile past box_rows are whatever lies behind them in the ring: their results are not used
            const uint64_t a_desc = smem_desc_k128_sw128(w_addr + C::kBBytes);
            const uint64_t b_desc = smem_desc_k128_sw128(w_addr);
            const uint32_t d = tmem + static_cast<uint32_t>(b * BN);
#pragma unroll
            for (int k = 0; k < kFp8Block / 32; ++k) mma_e4m3(d, a_desc + 2 * k, b_desc + 2 * k, idesc, k != 0);
            mma_commit(&empty[s]);
            mma_commit(&acc_full[b]);
            s += 2;
            if (s >= S) s -= S, phase ^= 1;
          }
        }
        // all issued MMAs complete before the tensor memory can be freed
        mma_commit(mma_done);
        const long long t0 = clock64();
        while (!mbar_try_wait(mma_done, 0)) {
          if (clock64() - t0 > kFp8WaitClocks) {
            atomicExch(&g_fp8_err, QF_ERR_TIMEOUT);
            break;
          }
        }
      }
      __syncwarp();
    }
  } else {
    if (C::kCols > 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int q = warp & 3;                        // tensor-memory lane quarter this warp may read
    const int col0 = (warp - 4) / 4 * C::kCols;    // its columns of the tile
    const int row = 32 * q + lane;
    const int et = threadIdx.x - 128;
    float* s_scale = reinterpret_cast<float*>(smem + C::kOffScale);
    const int nb_last = (p.N - 1) / kFp8Block;

    // Scales: each thread copies its row's, and the warp its two weight blocks', a chunk of groups at a time and two
    // chunks ahead (a cache miss per group would stall every one of them); the copies run on across tiles.
    int lt = first, lk = k0, lch = 0;
    const float* l_sa = nullptr;
    const float* l_sw = nullptr;
    auto load_chunk_of_scales = [&]() {
      if (lt < ntotal) {
        if (lk == k0) {
          int m0, n0;
          tile_origin(tp, lt, BN, &m0, &n0);
          l_sa = p.sa + static_cast<int64_t>(min(m0 + row, p.M - 1)) * p.sa_m;
          const int nb = (n0 + col0 + ((lane & 1) ? C::kCols - 1 : 0)) / kFp8Block;
          l_sw = p.sw + static_cast<int64_t>(min(nb, nb_last)) * p.sw_n;
        }
        const uint32_t dst = smem_u32(s_scale + lch % kScaleBufs * C::kScaleBuf);
#pragma unroll
        for (int i = 0; i < kScaleK; ++i) {
          const int64_t g = min(lk + i, p.kb - 1);
          cp_async4(dst + 4 * (i * 32 * EW + et), l_sa + g * p.sa_g);
        }
        if (lane < 2 * kScaleK) {
          const int64_t g = min(lk + lane / 2, p.kb - 1);
          cp_async4(dst + 4 * (kScaleK * 32 * EW + (warp - 4) * 2 * kScaleK + lane), l_sw + g * p.sw_g);
        }
        lk += kScaleK;
        if (lk >= k1) lk = k0, lt += step;
      }
      cp_async_commit();
      ++lch;
    };
    load_chunk_of_scales();
    load_chunk_of_scales();

    int it = 0, ch = 0;
    bool ok = true;
    for (int t = first; t < ntotal && ok; t += step) {
      int m0, n0;
      tile_origin(tp, t, BN, &m0, &n0);
      const int m = m0 + row;
      // the thread's columns lie in at most two scale blocks; 32 of them in one (n0 and col0 are multiples of 32)
      const int split_col = kFp8Block - (n0 + col0) % kFp8Block;
      uint64_t acc[C::kCols / 2];
#pragma unroll
      for (int j = 0; j < C::kCols / 2; ++j) acc[j] = 0;
      for (int kc = k0; kc < k1 && ok; kc += kScaleK, ++ch) {
        __syncwarp();  // the buffer of the chunk before last is free in every lane
        load_chunk_of_scales();
        cp_async_wait<2>();
        __syncwarp();
        const float* sc = s_scale + ch % kScaleBufs * C::kScaleBuf;
        const float* scw = sc + kScaleK * 32 * EW + (warp - 4) * 2 * kScaleK;
        const int kn = min(kScaleK, k1 - kc);
        for (int i = 0; i < kn; ++i, ++it) {
          const int b = it % A;
          const float sa = sc[i * 32 * EW + et];
          const float s0 = sa * scw[2 * i], s1 = sa * scw[2 * i + 1];
          if (!fp8_wait_warp(&acc_full[b], (it / A) & 1, s_abort)) {  // tcgen05.ld needs the warp whole
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t src = tmem + (static_cast<uint32_t>(32 * q) << 16) + static_cast<uint32_t>(b * BN + col0);
          // the next 32 columns are on their way while these are added
          uint32_t r[2][32];
          tmem_ld_32x32b_x32_async(src, r[0]);
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c) {
            tmem_ld_wait(r[c & 1]);
            if (c + 1 < C::kChunks) {
              tmem_ld_32x32b_x32_async(src + 32 * (c + 1), r[(c + 1) & 1]);
            } else {
              tc_fence_before();
              if (lane == 0) mbar_arrive(&acc_empty[b]);
            }
            const float s = 32 * c < split_col ? s0 : s1;
            const uint64_t s2 = pack_f32x2(s, s);
#pragma unroll
            for (int j = 0; j < 16; ++j)
              fma_f32x2(acc[16 * c + j],
                        pack_f32x2(__uint_as_float(r[c & 1][2 * j]), __uint_as_float(r[c & 1][2 * j + 1])), s2);
          }
        }
      }
      if (!ok) break;
      if (SPLIT) {
        // the ring is idle (every accumulator was read, so every MMA and copy is done): it takes the partial tile,
        // column by column
        float* part = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int j = 0; j < C::kCols / 2; ++j) {
          const float2 v = unpack_f32x2(acc[j]);
          part[(col0 + 2 * j) * kTileM + row] = v.x;
          part[(col0 + 2 * j + 1) * kTileM + row] = v.y;
        }
      } else if (m < p.M) {
#pragma unroll
        for (int j = 0; j < C::kCols / 8; ++j) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_f32x2(acc[4 * j + i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
          }
          store8(tp, m, n0 + col0 + 8 * j, v);
        }
      }
    }
    cp_async_wait<0>();
  }
  tc_fence_before();
  if (SPLIT) {
    cluster_sync();
    // each CTA adds an equal part of the tile over the cluster, in rank order, and stores it
    int m0, n0;
    tile_origin(tp, first, BN, &m0, &n0);
    const int rows = min(kTileM, p.M - m0), pieces = BN / 8;
    const uint32_t part = smem_u32(smem);
    if (!*s_abort) {
      for (int e = rank * C::kThreads + threadIdx.x; e < rows * pieces; e += tp.splits * C::kThreads) {
        const int row = e % rows, c = e / rows * 8;
        if (n0 + c >= p.N) continue;
        float v[8] = {};
        for (int r = 0; r < tp.splits; ++r) {
          const uint32_t src = map_to_rank(part + static_cast<uint32_t>((c * kTileM + row) * 4), r);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] += ld_cluster_f32(src + j * kTileM * 4);
        }
        store8(tp, m0 + row, n0 + c, v);
      }
    }
    cluster_sync();  // no CTA leaves while another reads its part
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, C::kTmemCols);
}

std::mutex g_dev_mu;
int g_dev_sms[64] = {};
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;

int find_encode() {
  std::lock_guard<std::mutex> lk(g_dev_mu);
  if (g_encode) return QF_OK;
  cudaDriverEntryPointQueryResult qres;
  void* fn = nullptr;
  const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
  if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !fn)
    return fail(QF_ERR_DRIVER, "cuTensorMapEncodeTiled entry point not found");
  g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  return QF_OK;
}

// Operand rows, in boxes of one k group.
int encode_rows(CUtensorMap* map, const void* base, int K, int rows, int64_t row_bytes, int box_rows) {
  const int rc = find_encode();
  if (rc) return rc;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(kFp8Block), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(QF_ERR_DRIVER, "cuTensorMapEncodeTiled rejected the tensor (error " + std::to_string(r) + ")");
  return QF_OK;
}

template <int BN, bool SPLIT>
int launch_tiles(TileParams tp, int dev, int sms, int splits, unsigned flags, cudaStream_t st) {
  using C = TileGeo<BN, SPLIT>;
  static bool attr_set[64] = {};
  {
    std::lock_guard<std::mutex> lk(g_dev_mu);
    if (!attr_set[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(fp8_tile_kernel<BN, SPLIT>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
      if (e != cudaSuccess) return fail(QF_ERR_LAUNCH, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
      attr_set[dev] = true;
    }
  }
  const Fp8Params& p = tp.p;
  tp.mtiles = (p.M + kTileM - 1) / kTileM;
  tp.ntiles = (p.N + BN - 1) / BN;
  tp.splits = splits;
  CUtensorMap ta, tw;
  // one row has no stride of its own: any multiple of 16 not below the row does
  const int64_t one = (static_cast<int64_t>(p.K) + 15) / 16 * 16;
  // whole swizzle atoms of eight rows
  tp.box_rows = p.M < kTileM ? (p.M + 7) / 8 * 8 : kTileM;
  tp.stages = C::kRing / (C::kBBytes + tp.box_rows * kFp8Block);
  if (tp.stages > kMaxStages) tp.stages = kMaxStages;
  // the last stage's MMA reads 128 rows from its token rows on: they have to lie in the ring
  while (tp.stages * (C::kBBytes + tp.box_rows * kFp8Block) + (kTileM - tp.box_rows) * kFp8Block > C::kRing) --tp.stages;
  int rc = encode_rows(&ta, p.a, p.K, p.M, p.M > 1 ? p.lda : one, tp.box_rows);
  if (rc) return rc;
  rc = encode_rows(&tw, p.w, p.K, p.N, p.N > 1 ? p.ldw : one, BN);
  if (rc) return rc;
  const int total = tp.mtiles * tp.ntiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(SPLIT ? total * splits : (total < sms ? total : sms)));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (flags & QF_FLAG_PDL) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (SPLIT) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = static_cast<unsigned>(splits);
    attr[na].val.clusterDim.y = 1;
    attr[na++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(na);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_tile_kernel<BN, SPLIT>, ta, tw, tp);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}

// The whole k groups of operand rows as [group][row][128 bytes].
int encode_groups(CUtensorMap* map, const void* base, int K, int rows, int64_t row_bytes, int box_rows, int box_groups) {
  const int rc = find_encode();
  if (rc) return rc;
  cuuint64_t dims[3] = {kFp8Block, static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(K / kFp8Block)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_bytes), kFp8Block};
  cuuint32_t box[3] = {kFp8Block, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(box_groups)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(QF_ERR_DRIVER, "cuTensorMapEncodeTiled rejected the tensor (error " + std::to_string(r) + ")");
  return QF_OK;
}

template <int NT, int MT, int G> int launch_rows(const Fp8Params& p, int dev, int sms, unsigned flags, cudaStream_t st) {
  using C = RowGeo<NT, MT, G>;
  static bool attr_set[64] = {};
  {
    std::lock_guard<std::mutex> lk(g_dev_mu);
    if (!attr_set[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(fp8_rows_kernel<NT, MT, G>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
      if (e != cudaSuccess) return fail(QF_ERR_LAUNCH, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
      attr_set[dev] = true;
    }
  }
  CUtensorMap ta = {}, tw = {};
  if (p.K >= kFp8Block) {
    // one row has no stride of its own: any multiple of 16 not below the row does
    const int64_t one = (static_cast<int64_t>(p.K) + 15) / 16 * 16;
    int rc = encode_groups(&ta, p.a, p.K, p.M, p.M > 1 ? p.lda : one, 8 * NT, C::kGroups);
    if (rc == QF_OK) rc = encode_groups(&tw, p.w, p.K, p.N, p.N > 1 ? p.ldw : one, C::kRows, C::kGroups);
    if (rc) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  // as few CTAs as finish in the same number of rounds: all of them run at once and share the memory evenly, so an SM
  // with one more costs nothing, but a last round for a few would
  const int ntiles = (p.N + C::kRows - 1) / C::kRows;
  const int rounds = (ntiles + sms * kRowPerSm - 1) / (sms * kRowPerSm);
  cfg.gridDim = dim3(static_cast<unsigned>((ntiles + rounds - 1) / rounds),
                     static_cast<unsigned>((p.M + 8 * NT - 1) / (8 * NT)));
  cfg.blockDim = dim3(kRowWarps * 32 + 32);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_rows_kernel<NT, MT, G>, ta, tw, p, ntiles);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}

// Tiles of 32 weight rows halve the token rows copied per weight row and the waits per byte, where there are enough of
// them for two CTAs on every SM (10240 x 5120, 5 tokens: 10.6 us against 12.4; 34816 x 5120: 28.4 against 29.0); fewer
// rows are better spread thin (5120 x 17408, one token: 16 rows 19.1 us, 32 rows 25.5).  With 16 rows a warp takes two
// k groups per stage up to 8 tokens (two stages of 24 KiB; 5120 x 17408, 8 tokens: 18.3 us against 19.6 with one, 8192: 9.8
// against 10.3); above, the token rows of two groups do not fit the registers (16 tokens: 36.5 us against 26.1 with one
// and four stages of 16 KiB).
int rows_any(const Fp8Params& p, int dev, int sms, unsigned flags, cudaStream_t st) {
  const bool wide = (p.N + 31) / 32 >= 2 * sms;
  if (p.M <= 8) return wide ? launch_rows<1, 2, 1>(p, dev, sms, flags, st) : launch_rows<1, 1, 2>(p, dev, sms, flags, st);
  return wide ? launch_rows<2, 2, 1>(p, dev, sms, flags, st) : launch_rows<2, 1, 1>(p, dev, sms, flags, st);
}

// Clusters of `split` CTAs (one per SM) that the device runs at once: a cluster stays within one group of SMs, so this is
// less than SMs / split for some sizes.  Asked once per device.
int resident_clusters(int dev, int sms, int split) {
  if (split == 1) return sms;
  static int known[64][9] = {};
  std::lock_guard<std::mutex> lk(g_dev_mu);
  if (known[dev][split] == 0) {
    using C = TileGeo<128, true>;
    int n = 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(split * sms));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaFuncSetAttribute(fp8_tile_kernel<128, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         C::kSmemBytes);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, fp8_tile_kernel<128, true>, &cfg);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    known[dev][split] = n > 0 ? n : -1;
  }
  return known[dev][split];
}

// Tile width and k split.  Time of a choice in microseconds: whole waves of CTAs, each a start and its groups at the
// measured rate of one CTA over many of them (64 / 128 / 256 channels: 0.30 / 0.38 / 0.52 us), and for a split the join of
// the parts.  It ranks the choices; a split takes longer than it says (72 x 10240 x 5120: 256 channels in three parts, 10.3
// us by this model, 18.2 measured, 17.8 with the weights in L2).
int tiles_any(const TileParams& tp, int dev, int sms, unsigned flags, cudaStream_t st) {
  const Fp8Params& p = tp.p;
  const int mt = (p.M + kTileM - 1) / kTileM;
  int best_bn = 0, best_split = 1;
  double best = 1e30;
  for (int bn = 64; bn <= 256; bn *= 2) {
    const double group = bn == 64 ? 0.30 : bn == 128 ? 0.38 : 0.52;
    const long long tiles = static_cast<long long>(mt) * ((p.N + bn - 1) / bn);
    for (int split = 1; split <= 8 && split <= p.kb; ++split) {
      if (split > 1 && tiles * split > sms) break;  // a split is for the SMs that would idle
      const int at_once = resident_clusters(dev, sms, split);
      if (at_once <= 0) continue;
      const double waves = static_cast<double>((tiles + at_once - 1) / at_once);
      const double t = waves * (((p.kb + split - 1) / split) * group + 0.8) + (split > 1 ? 1.2 + 0.004 * bn : 0.0);
      if (t < best) best = t, best_bn = bn, best_split = split;
    }
  }
  if (best_split > 1) {
    if (best_bn == 64) return launch_tiles<64, true>(tp, dev, sms, best_split, flags, st);
    if (best_bn == 128) return launch_tiles<128, true>(tp, dev, sms, best_split, flags, st);
    return launch_tiles<256, true>(tp, dev, sms, best_split, flags, st);
  }
  if (best_bn == 64) return launch_tiles<64, false>(tp, dev, sms, 1, flags, st);
  if (best_bn == 128) return launch_tiles<128, false>(tp, dev, sms, 1, flags, st);
  return launch_tiles<256, false>(tp, dev, sms, 1, flags, st);
}

}  // namespace

int require_b200(int* dev_out, int* sms) {
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fail(QF_ERR_LAUNCH, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
  if (dev < 0 || dev >= 64) return fail(QF_ERR_INVALID, "device index out of range");
  std::lock_guard<std::mutex> lk(g_dev_mu);
  if (g_dev_sms[dev] == 0) {
    int major = 0, minor = 0, n = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    g_dev_sms[dev] = (major == 10 && minor == 0 && n > 0) ? n : -1;
  }
  if (g_dev_sms[dev] < 0)
    return fail(QF_ERR_ARCH, "libqf_b200 is built for sm_100a (B200); this device is not compute capability 10.0");
  if (dev_out) *dev_out = dev;
  if (sms) *sms = g_dev_sms[dev];
  return QF_OK;
}

int read_error_word(const void* symbol, void* stream, int* status) {
  if (!status) return fail(QF_ERR_INVALID, "null status");
  const int rc = require_b200(nullptr, nullptr);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int v = 0;
  const int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, symbol, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && v != 0) e = cudaMemcpyToSymbolAsync(symbol, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
  if (e == cudaSuccess && v != 0) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return fail(QF_ERR_LAUNCH, cudaGetErrorString(e));
  *status = v;
  return QF_OK;
}

}  // namespace qf

using namespace qf;

extern "C" int qf_fp8_block_gemm(const void* a, int64_t lda, const float* a_scale, int64_t sa_m, int64_t sa_g,
                                 const void* w, int64_t ldw, const float* w_scale, int64_t sw_n, int64_t sw_g,
                                 const void* bias, void* y, int64_t ldy, int y_dtype, int M, int N, int K,
                                 unsigned flags, void* stream) {
  if (M < 0 || N < 0 || K < 0) return fail(QF_ERR_SHAPE, "negative size");
  if (y_dtype != QF_DTYPE_BF16 && y_dtype != QF_DTYPE_F32) return fail(QF_ERR_DTYPE, "y must be bf16 or fp32");
  if (M == 0 || N == 0) return QF_OK;
  if (K == 0) return fail(QF_ERR_SHAPE, "K must be >= 1");
  // tile numbers, and the step of a grid past the last, have 32 bits
  if (K > QF_FP8_MAX_K || N > QF_MAX_N || M > QF_FP8_MAX_M ||
      static_cast<int64_t>((M + kTileM - 1) / kTileM) * ((N + 63) / 64) >= INT32_MAX - 4095)
    return fail(QF_ERR_SHAPE, "M, N or K too large");
  if (!a || !a_scale || !w || !w_scale || !y) return fail(QF_ERR_INVALID, "null pointer");
  if ((M > 1 && lda < K) || (N > 1 && ldw < K) || (M > 1 && ldy < N))
    return fail(QF_ERR_STRIDE, "leading dimension too small");
  if (sa_m < 0 || sa_g < 0 || sw_n < 0 || sw_g < 0) return fail(QF_ERR_STRIDE, "negative scale stride");
  if (reinterpret_cast<uintptr_t>(a) % 16 || (M > 1 && lda % 16) || reinterpret_cast<uintptr_t>(w) % 16 ||
      (N > 1 && ldw % 16))
    return fail(QF_ERR_ALIGN, "a and w must be 16-byte aligned with row strides that are multiples of 16");
  const size_t yb = y_dtype == QF_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a_scale) % 4 || reinterpret_cast<uintptr_t>(w_scale) % 4 ||
      reinterpret_cast<uintptr_t>(bias) % 2 || reinterpret_cast<uintptr_t>(y) % yb)
    return fail(QF_ERR_ALIGN, "scales, bias and y must be aligned to their element");
  int dev = 0, sms = 0;
  const int rc = require_b200(&dev, &sms);
  if (rc) return rc;
  Fp8Params p = {};
  p.a = static_cast<const uint8_t*>(a);
  p.lda = lda;
  p.sa = a_scale;
  p.sa_m = sa_m;
  p.sa_g = sa_g;
  p.w = static_cast<const uint8_t*>(w);
  p.ldw = ldw;
  p.sw = w_scale;
  p.sw_n = sw_n;
  p.sw_g = sw_g;
  p.bias = static_cast<const __nv_bfloat16*>(bias);
  p.y = y;
  p.ldy = ldy;
  p.y_f32 = y_dtype == QF_DTYPE_F32;
  p.M = M;
  p.N = N;
  p.K = K;
  p.kb = (K + kFp8Block - 1) / kFp8Block;
  if (M > 16) {
    TileParams tp = {};
    tp.p = p;
    tp.vec_out = reinterpret_cast<uintptr_t>(y) % 16 == 0 && (M == 1 || ldy * yb % 16 == 0);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return tiles_any(tp, dev, sms, flags, st);
  }
  return rows_any(p, dev, sms, flags, static_cast<cudaStream_t>(stream));
}

extern "C" int qf_fp8_status(void* stream, int* status) { return read_error_word(&g_fp8_err, stream, status); }
