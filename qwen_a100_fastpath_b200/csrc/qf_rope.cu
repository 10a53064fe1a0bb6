// qf_rope.cu -- norms of queries and keys for each head with the position rotation in the same pass, and optionally the
// keys and values straight into the 4-bit cache.
//
// Mathematics, per token and head (a row of D values x), fp32 inside:
//   y = x, or x * rsqrt(mean(x^2) + eps) * (weight + offset)
//   the first R values turn by the token's angles: with (cos_i, sin_i) = the table's row of the token's position,
//   a = y[i], b = y[i + R / 2] (or y[2 i], y[2 i + 1]):  a' = a cos_i - b sin_i,  b' = b cos_i + a sin_i
//   the result is rounded to bf16 once; a key that goes into the cache is quantized from those bf16 values.
//
// Bound by memory on paper (a row is read and written once); in fact by the instructions around the 16 bytes of a lane and by
// the loads in flight: 8192 tokens of 24 + 4 heads of 256 with 64 turned values 49 us in a graph (4.8 TB/s; floor 36), IPC 2.8 of
// 4, half of the logic pipe; 5 tokens into the cache and back 4.2 us.
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
  int rows;        // of a token; kWide: groups of rows
  uint32_t total;  // of all tokens
  int groups[2];   // kWide: of the queries and of the keys
  int chunk;       // kWide: heads of a group
  int cs_f32, interleaved;
};

constexpr int kRopeWarps = 4;

// How rows are read: kAny takes any size, stride and alignment, element by element with the row in shared memory; kWide rows
// whose pointers and strides are multiples of 16 bytes, with heads of up to 256 (a multiple of eight) and a rotated part that
// is a multiple of 16 (of eight where interleaved).  8192 tokens of 24 + 4 heads of 256, 64 of them rotated: 99 us with kAny, 49
// with kWide.  One operand at an odd address takes all to kAny: copying it for kWide costs more (queries at the sizes above, 333
// tokens of 40 + 8 heads of 128 and 5 tokens of 24 + 4 of 256: 99, 7.9 and 2.7 us, with a copy 118, 14.4 and 4.0).

// kWide: L lanes take a row, a lane eight consecutive values in one 16-byte load.  A group of L lanes takes p.chunk heads of
// one side of one token, ROWS at a time, so that the token's angles and the weight are loaded and multiplied once for them
// and ROWS loads are under way.  The other half of a turned pair is another of the L lanes' (a shuffle of the raw bf16 words;
// its weight is loaded beside the lane's own), or the neighbour in the lane's own registers where interleaved (INTER).
// Measured at the size above: four heads to a group and separate products with weight, cosine and sine 75 us; one coefficient
// each for the value and the other one, on packed pairs, 59; eight heads to a group 54; 64 registers, so that eight CTAs
// share an SM, 49 (ten CTAs, with spills, 72; eight rows at a time 53, two 56).
template <int L, int ROWS, bool INTER>
__global__ void __launch_bounds__(kRopeWarps * 32, ROWS == 1 ? 1 : 8) rope_wide_kernel(const RopeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x % L;
  const uint32_t item = blockIdx.x * (kRopeWarps * 32 / L) + threadIdx.x / L;
  // (groups past the end go on with the last one's work, without storing: the shuffles name whole warps)
  const uint32_t at = item < p.total ? item : p.total - 1;
  const uint32_t token = at / p.rows;
  int part = at - token * p.rows, side = 0;
  if (part >= p.groups[0]) part -= p.groups[0], side = 1;
  if (side == 1 && part >= p.groups[1]) part -= p.groups[1], side = 2;
  const int all = side == 0 ? p.heads[0] : p.heads[1], chunk0 = part * p.chunk;
  const int e = 8 * lane;
  const bool in = e < p.D;
  const int heads = min(all, chunk0 + p.chunk);
  const __nv_bfloat16* const x = p.x[side] + static_cast<int64_t>(token) * p.xt[side] + e;
  const int64_t xh = p.xh[side];
  uint4 u[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    u[i] = make_uint4(0, 0, 0, 0);
    if (in && chunk0 + i < heads) u[i] = *reinterpret_cast<const uint4*>(x + (chunk0 + i) * xh);
  }
  const bool normed = side < 2 && p.weight[side], turned = side < 2 && p.cos_sin && e < p.rot;
  const int half = p.rot / 2;
  const int swap = half / 8;  // lanes between the halves of a pair
  const bool upper = !INTER && e >= half;
  constexpr int kAngles = INTER ? 4 : 8;  // of a lane
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) cs[i] = 1.f, sn[i] = 0.f;
  if (turned) {
    const int64_t pos = p.positions[token];
    if (pos >= 0 && pos < p.max_pos) {
      const int64_t row = pos * p.cs_row + (INTER ? e / 2 : upper ? e - half : e);
#pragma unroll
      for (int k = 0; k < kAngles; k += 4) {
        float4 a, b;
        if (p.cs_f32) {
          const float* t = static_cast<const float*>(p.cos_sin) + row + k;
          a = *reinterpret_cast<const float4*>(t), b = *reinterpret_cast<const float4*>(t + half);
        } else {
          const __nv_bfloat16* t = static_cast<const __nv_bfloat16*>(p.cos_sin) + row + k;
          const uint2 c = *reinterpret_cast<const uint2*>(t), d = *reinterpret_cast<const uint2*>(t + half);
          a = make_float4(bf16_lo(c.x), bf16_hi(c.x), bf16_lo(c.y), bf16_hi(c.y));
          b = make_float4(bf16_lo(d.x), bf16_hi(d.x), bf16_lo(d.y), bf16_hi(d.y));
        }
        cs[k] = a.x, cs[k + 1] = a.y, cs[k + 2] = a.z, cs[k + 3] = a.w;
        sn[k] = b.x, sn[k + 1] = b.y, sn[k + 2] = b.z, sn[k + 3] = b.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) cs[k] = sn[k] = __int_as_float(0x7fffffff);
    }
    if (INTER) {
#pragma unroll
      for (int k = 3; k >= 0; --k) cs[2 * k] = cs[2 * k + 1] = cs[k], sn[2 * k] = -sn[k], sn[2 * k + 1] = -sn[2 * k];
    } else if (!upper) {
#pragma unroll
      for (int k = 0; k < 8; ++k) sn[k] = -sn[k];
    }
  }
  // y = n (x w cos + x' w' sin), x' the other of the pair, the sign of the sine taken in above: two coefficients an element
  const int other = turned && !INTER ? (upper ? lane - swap : lane + swap) : lane;
  uint64_t ca[4], cb[4];
  {
    float w[8], w2[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = w2[i] = 1.f;
    if (normed && in) {
      const uint4 a = *reinterpret_cast<const uint4*>(p.weight[side] + e);
      const uint4 b = *reinterpret_cast<const uint4*>(p.weight[side] + 8 * other);
      const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[2 * k] = bf16_lo(wa[k]) + p.offset, w[2 * k + 1] = bf16_hi(wa[k]) + p.offset;
        w2[2 * k] = bf16_lo(wb[k]) + p.offset, w2[2 * k + 1] = bf16_hi(wb[k]) + p.offset;
        if (INTER) {
          const float t = w2[2 * k];
          w2[2 * k] = w2[2 * k + 1], w2[2 * k + 1] = t;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      ca[k] = pack_f32x2(w[2 * k] * cs[2 * k], w[2 * k + 1] * cs[2 * k + 1]);
      // (an infinite weight times the zero that stands for the other of a value that does not turn would be NaN)
      cb[k] = turned ? pack_f32x2(w2[2 * k] * sn[2 * k], w2[2 * k + 1] * sn[2 * k + 1]) : pack_f32x2(0.f, 0.f);
    }
  }
  uint32_t page = 0, off = 0;
  const bool cached = side > 0 && !p.out[1] && p.cache.place(p.slots[token], page, off);
  const uint32_t keep = turned ? ~0u : 0u;  // values that do not turn have no other (an infinity times zero would be NaN)
  __nv_bfloat16* const out = side < 2 && p.out[side] ? p.out[side] + static_cast<int64_t>(token) * p.ot[side] + e : nullptr;
  const int64_t oh = side < 2 ? p.oh[side] : 0;
  const bool sums_needed = p.weight[0] || p.weight[1], to_cache = !p.out[1], stores = in && item < p.total;
  // (the same number of turns for all lanes of a warp: its groups may be of different sides)
  for (int turn = 0; turn < p.chunk; turn += ROWS) {
    const int head0 = chunk0 + turn;
    if (turn > 0)
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (in && head0 + i < heads) u[i] = *reinterpret_cast<const uint4*>(x + (head0 + i) * xh);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const uint32_t raw[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
      uint64_t v2[4], sums = pack_f32x2(0.f, 0.f);
      uint32_t r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t a = pack_f32x2(bf16_lo(raw[k]), bf16_hi(raw[k]));
        fma_f32x2(sums, a, a);
        // the other half of a turned pair: another lane's words, or this one's with its halves exchanged
        const uint32_t x2 = keep & (INTER ? __byte_perm(raw[k], raw[k], 0x1032)
                                          : __shfl_sync(0xffffffffu, raw[k], other, L));
        v2[k] = mul_f32x2(pack_f32x2(bf16_lo(x2), bf16_hi(x2)), cb[k]);
        fma_f32x2(v2[k], a, ca[k]);
      }
      const float2 both = unpack_f32x2(sums);
      float n = 1.f;
      if (sums_needed) {
        float sum = both.x + both.y;
#pragma unroll
        for (int d = L / 2; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (normed) n = rsqrtf(fmaf(sum, p.inv_d, p.eps));
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 y = unpack_f32x2(mul_f32x2(v2[k], pack_f32x2(n, n)));
        const __nv_bfloat162 h = __floats2bfloat162_rn(y.x, y.y);
        r[k] = reinterpret_cast<const uint32_t&>(h);
      }
      const bool store = stores && head0 + i < heads;
      if (out && store) *reinterpret_cast<uint4*>(out + (head0 + i) * oh) = make_uint4(r[0], r[1], r[2], r[3]);
      if (!to_cache) continue;
      // into the cache, from the rounded values (all lanes go along: a warp may hold groups of queries too)
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[2 * k] = bf16_lo(r[k]), v[2 * k + 1] = bf16_hi(r[k]);
      const uint32_t ends = kv4_extremes(r[0], r[1], r[2], r[3], 0xffffffffu);
      if (!cached || !store) continue;
      float s, c;
      kv4_scale(-bf16_hi(ends), bf16_lo(ends), s, c);
      const Kv4View& view = p.cache;
      const int kv = side - 1, head = head0 + i;
      *reinterpret_cast<uint32_t*>(view.codes[kv] + head * view.head + view.codes_at(page, off) + e / 2) =
          kv4_codes(v, s, c);
      if (lane % 8 == 0)
        reinterpret_cast<__nv_bfloat162*>(view.scale[kv] + head * view.shead + view.scale_at(page, off))[lane / 8] =
            __floats2bfloat162_rn(s, c);
    }
  }
}

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
  uint32_t page, off;
  const Kv4View& v = p.cache;
  if (!v.place(p.slots[token], page, off)) return;
  const int kv = side - 1;
  uint8_t* codes = v.codes[kv] + head * v.head + v.codes_at(page, off);
  uint8_t* scale = v.scale[kv] + head * v.shead + v.scale_at(page, off);
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
    const Kv4Coder code(s, c);
    const uint32_t n0 = code.slow(a) & 15u, n1 = code.slow(b) & 15u;
    codes[g * (kKv4Group / 2) + lane] = static_cast<uint8_t>(n0 | n1 << 4);
    if (lane == 0) reinterpret_cast<__nv_bfloat162*>(scale)[g] = __floats2bfloat162_rn(s, c);
  }
}

template <bool INTER> cudaError_t launch_wide(const cudaLaunchConfig_t& cfg, const RopeParams& p, int lanes, bool many) {
  if (many)
    return lanes == 8    ? cudaLaunchKernelEx(&cfg, rope_wide_kernel<8, 4, INTER>, p)
           : lanes == 16 ? cudaLaunchKernelEx(&cfg, rope_wide_kernel<16, 4, INTER>, p)
                         : cudaLaunchKernelEx(&cfg, rope_wide_kernel<32, 4, INTER>, p);
  return lanes == 8    ? cudaLaunchKernelEx(&cfg, rope_wide_kernel<8, 1, INTER>, p)
         : lanes == 16 ? cudaLaunchKernelEx(&cfg, rope_wide_kernel<16, 1, INTER>, p)
                       : cudaLaunchKernelEx(&cfg, rope_wide_kernel<32, 1, INTER>, p);
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
  // (a table of no positions is never read, but it still turns: every position is outside it)
  p.cos_sin = !rot ? nullptr : max_positions ? cos_sin : static_cast<const void*>(positions);
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
  auto wide_rows = [](const void* ptr, int64_t st_t, int64_t st_h) {
    return !ptr || (aligned(ptr, 16) && st_t % 8 == 0 && st_h % 8 == 0);
  };
  const bool wide = head_size % 8 == 0 && head_size <= 256 && rot % (interleaved ? 8 : 16) == 0 &&
                    wide_rows(q, sq_t, sq_h) && wide_rows(k, sk_t, sk_h) && wide_rows(q_out, so_t, so_h) &&
                    wide_rows(k_out, sp_t, sp_h) && wide_rows(v, sv_t, sv_h) && aligned(q_weight, 16) &&
                    aligned(k_weight, 16) && (!p.cos_sin || (aligned(cos_sin, 16) && s_cs % 8 == 0));
  const int lanes = head_size <= 64 ? 8 : head_size <= 128 ? 16 : 32;
  // eight heads to a group, four at a time, where that leaves groups enough for the SMs (about 900 threads each); a head to a
  // group below, where the first load's latency counts and not the angles' share
  const bool many = wide && p.total / 8 * lanes >= 1u << 17;
  p.chunk = many ? 8 : 1;
  cudaLaunchConfig_t cfg = {};
  if (wide) {
    const auto groups = [&](int heads) { return (heads + p.chunk - 1) / p.chunk; };
    p.groups[0] = groups(num_heads), p.groups[1] = groups(num_kv_heads);
    p.rows = p.groups[0] + p.groups[1] * (cache ? 2 : 1);
    p.total = static_cast<uint32_t>(p.rows) * static_cast<uint32_t>(tokens);
  }
  const uint32_t per_cta = wide ? kRopeWarps * 32 / lanes : kRopeWarps;
  cfg.gridDim = dim3((p.total + per_cta - 1) / per_cta);
  cfg.blockDim = dim3(kRopeWarps * 32);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  cudaError_t e;
  if (!wide)
    e = cudaLaunchKernelEx(&cfg, rope_any_kernel, p);
  else if (interleaved)
    e = launch_wide<true>(cfg, p, lanes, many);
  else
    e = launch_wide<false>(cfg, p, lanes, many);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}
