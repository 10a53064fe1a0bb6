// qf_fp8_gemm.cu -- e4m3 x e4m3 product with one fp32 scale for each 128 elements along k (and each 128 output
// channels of the weight).
//
// Mathematics: y[m, n] = sum_g sa[m, g] * sw[n / 128, g] * P_g[m, n], P_g = sum over the 128 k of group g of
// a[m, k] * w[n, k].  Products of e4m3 values are exact in fp32; each P_g is summed by the tensor cores in fp32 and
// folded into fp32 sums with one multiply-add per group and output.
//
// fp8_rows_kernel: a CTA of eight warps takes 16 weight rows and 8 * NT tokens, warp w the groups w, w + 8, ...; the
// weights go from global memory straight into the registers of mma.sync m16n8k32 (weights as the 16-row operand), the
// warps' sums are added in shared memory in warp order.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/qf_b200.h"
#include "qf_fp8.cuh"
#include "qf_host.h"
#include "qf_ptx.cuh"

namespace qf {
namespace {

constexpr int kRowWarps = 8;

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

// 16 bytes of an operand row from column k; bytes past K read as zero and are not touched.
__device__ __forceinline__ uint4 load_chunk(const uint8_t* row, int k, int K) {
  if (k + 16 <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) w[i / 4] |= static_cast<uint32_t>(__ldg(row + k + i)) << (8 * (i % 4));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int NT>
__global__ void __launch_bounds__(kRowWarps * 32) fp8_rows_kernel(const Fp8Params p) {
  __shared__ float red[kRowWarps][NT][32][4];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (8 * NT);
  // rows past the end repeat the last one: their products are computed and not stored
  const uint8_t* w_lo = p.w + static_cast<int64_t>(min(n0 + gid, p.N - 1)) * p.ldw;
  const uint8_t* w_hi = p.w + static_cast<int64_t>(min(n0 + gid + 8, p.N - 1)) * p.ldw;
  const uint8_t* a_row[NT];
  const float* sa_row[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    a_row[j] = p.a + static_cast<int64_t>(min(m0 + 8 * j + gid, p.M - 1)) * p.lda;
#pragma unroll
    for (int i = 0; i < 2; ++i) sa_row[j][i] = p.sa + static_cast<int64_t>(min(m0 + 8 * j + 2 * t + i, p.M - 1)) * p.sa_m;
  }
  const float* sw_row = p.sw + static_cast<int64_t>(n0 / kFp8Block) * p.sw_n;
  float acc[NT][4] = {};
  for (int g = warp; g < p.kb; g += kRowWarps) {
    const int k = g * kFp8Block + 16 * t;
    uint4 lo[2], hi[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      lo[c] = load_chunk(w_lo, k + 64 * c, p.K);
      hi[c] = load_chunk(w_hi, k + 64 * c, p.K);
    }
    const float sw = __ldg(sw_row + g * p.sw_g);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float d[4] = {};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint4 b = load_chunk(a_row[j], k + 64 * c, p.K);
        // the thread's 16 bytes stand for the instruction's k slots of two steps, the same ones in both operands
        mma_e4m3_m16n8k32(d, lo[c].x, hi[c].x, lo[c].y, hi[c].y, b.x, b.y);
        mma_e4m3_m16n8k32(d, lo[c].z, hi[c].z, lo[c].w, hi[c].w, b.z, b.w);
      }
      const float s0 = sw * __ldg(sa_row[j][0] + g * p.sa_g), s1 = sw * __ldg(sa_row[j][1] + g * p.sa_g);
      acc[j][0] = fmaf(d[0], s0, acc[j][0]);
      acc[j][1] = fmaf(d[1], s1, acc[j][1]);
      acc[j][2] = fmaf(d[2], s0, acc[j][2]);
      acc[j][3] = fmaf(d[3], s1, acc[j][3]);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[warp][j][lane][i] = acc[j][i];
  __syncthreads();
  for (int e = threadIdx.x; e < NT * 128; e += kRowWarps * 32) {
    const int r = e % 16, tok = e / 16;
    const int src = (r % 8) * 4 + (tok % 8) / 2, reg = (r / 8) * 2 + (tok & 1);
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) s += red[w][tok / 8][src][reg];
    const int n = n0 + r, m = m0 + tok;
    if (n < p.N && m < p.M) {
      if (p.bias) s += __bfloat162float(p.bias[n]);
      const int64_t at = static_cast<int64_t>(m) * p.ldy + n;
      if (p.y_f32)
        static_cast<float*>(p.y)[at] = s;
      else
        static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(s);
    }
  }
}

std::mutex g_dev_mu;
int g_dev_sms[64] = {};

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
  if (K > QF_FP8_MAX_K || N > QF_MAX_N || M > QF_MAX_N) return fail(QF_ERR_SHAPE, "M, N or K too large");
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
  const int rc = require_b200(nullptr, nullptr);
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
  const int nt = M <= 8 ? 1 : 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((N + 15) / 16), static_cast<unsigned>((M + 8 * nt - 1) / (8 * nt)));
  cfg.blockDim = dim3(kRowWarps * 32);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = (flags & QF_FLAG_PDL) ? 1 : 0;
  const cudaError_t e = nt == 1 ? cudaLaunchKernelEx(&cfg, fp8_rows_kernel<1>, p)
                                : cudaLaunchKernelEx(&cfg, fp8_rows_kernel<2>, p);
  return e == cudaSuccess ? QF_OK : fail(QF_ERR_LAUNCH, std::string("launch: ") + cudaGetErrorString(e));
}
