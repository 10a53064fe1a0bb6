// qf_torch_ops.cpp -- the thin PyTorch operator over the C ABI of libqf_b200 (include/qf_b200.h).
//
// torch.ops.qf_b200.int8_linear(x, w_q, w_s, bias) is the body of the reference plugin's qf_int8_linear custom op
// (plugin/qwen_fastpath/patches.py:84-101) for bf16 activations on a K-major int8 weight: leading dimensions
// flattened to rows, M <= 16 rows on the small-M W8A16 kernel (bias fused with the reference's two roundings), more
// rows on the tcgen05 W8A8 prefill kernel (the reference's vLLM fallback arithmetic), output in x's shape with N
// columns.  It exists so that an eager call costs one dispatcher hop and the argument checks of the C ABI, instead
// of Python-level checks and a ctypes call.  Workspaces come from the PyTorch caching allocator, one per
// (device, stream) and kind, zero-filled when allocated (the kernels leave their counters at zero).  The caller
// decides eligibility (bf16 activations, a weight the tensor maps can take); anything else raises.
//
// torch.ops.qf_b200.fp8_quantize / fp8_block_mm / fp8_block_linear / residual_norm are the operators of block-scaled fp8
// layers (fp8.py and norms.py document them).  They need no workspace: what they make comes from the caching allocator,
// so calls on several streams, and captured graphs, share nothing.  They refuse a call with a ValueError before anything
// is launched, and tensors that require a gradient or carry a tangent too: none of them has a derivative.
#include <map>
#include <mutex>
#include <tuple>

#include "qf_torch.h"

using namespace qf_torch;

namespace {

std::mutex g_ws_mu;
std::map<std::tuple<int, uintptr_t, int>, at::Tensor> g_ws;  // (device, stream, kind) -> workspace

at::Tensor workspace(const at::Device& dev, cudaStream_t stream, int kind, size_t nbytes) {
  std::lock_guard<std::mutex> lk(g_ws_mu);
  auto key = std::make_tuple(static_cast<int>(dev.index()), reinterpret_cast<uintptr_t>(stream), kind);
  auto it = g_ws.find(key);
  if (it == g_ws.end() || static_cast<size_t>(it->second.numel()) < nbytes) {
    const int64_t n = static_cast<int64_t>(nbytes < (8u << 20) ? (8u << 20) : nbytes);
    at::Tensor t = at::zeros({n}, at::TensorOptions().dtype(at::kByte).device(dev));
    g_ws[key] = t;
    return t;
  }
  return it->second;
}

at::Tensor int8_linear(const at::Tensor& x, const at::Tensor& w_q, const at::Tensor& w_s,
                       const c10::optional<at::Tensor>& bias) {
  TORCH_CHECK(x.is_cuda() && w_q.is_cuda() && w_s.is_cuda(), "qf_b200.int8_linear needs CUDA tensors");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, "activations must be bf16");
  TORCH_CHECK(w_q.scalar_type() == at::kChar && w_q.dim() == 2 && w_q.stride(0) == 1,
              "w_q must be int8 [K, N] with stride (1, ldw)");
  TORCH_CHECK(w_s.scalar_type() == at::kFloat, "w_s must be fp32");
  const int64_t K = x.size(-1);
  const int64_t N = w_q.size(1);
  TORCH_CHECK(w_q.size(0) == K, "w_q rows must match the activations' last dimension");
  TORCH_CHECK(w_s.numel() == N, "w_s must hold N per-channel scales");
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor x2 = x.reshape({-1, K});
  const int64_t M = x2.size(0);
  std::vector<int64_t> out_shape(x.sizes().begin(), x.sizes().end());
  out_shape.back() = N;
  at::Tensor y = at::empty({M, N}, x.options());
  if (M == 0 || N == 0) return y.view(out_shape);
  if (x2.stride(-1) != 1) x2 = x2.contiguous();
  const at::Tensor scale = w_s.reshape({-1}).contiguous();
  at::Tensor b;
  if (bias.has_value() && bias->defined()) {
    TORCH_CHECK(bias->scalar_type() == at::kBFloat16 && bias->numel() == N, "bias must be bf16 [N]");
    b = bias->reshape({-1}).contiguous();
  }
  const int64_t ldw = N > 1 ? w_q.stride(1) : (K + 15) / 16 * 16;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  int rc;
  if (M <= QF_MAX_M) {
    if (reinterpret_cast<uintptr_t>(x2.data_ptr()) % 16 || (M > 1 && x2.stride(0) % 8))
      x2 = x2.clone(at::MemoryFormat::Contiguous);
    at::Tensor ws = workspace(x.device(), stream, 0,
                              qf_w8a16_workspace_bytes(static_cast<int>(M), static_cast<int>(N), static_cast<int>(K)));
    rc = qf_w8a16_gemm(x2.data_ptr(), x2.stride(0), static_cast<const int8_t*>(w_q.data_ptr()), ldw,
                       scale.data_ptr<float>(), b.defined() ? b.data_ptr() : nullptr, y.data_ptr(), N, QF_DTYPE_BF16,
                       static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), ws.data_ptr(),
                       static_cast<size_t>(ws.numel()), QF_FLAG_PDL, stream);
    check(rc, "qf_w8a16_gemm");
  } else {
    at::Tensor ws = workspace(x.device(), stream, 1, qf_w8a8_workspace_bytes(static_cast<int>(M), static_cast<int>(K)));
    rc = qf_w8a8_gemm(x2.data_ptr(), x2.stride(0), static_cast<const int8_t*>(w_q.data_ptr()), ldw,
                      scale.data_ptr<float>(), b.defined() ? b.data_ptr() : nullptr, y.data_ptr(), N,
                      static_cast<int>(M), static_cast<int>(N), static_cast<int>(K), ws.data_ptr(),
                      static_cast<size_t>(ws.numel()), QF_FLAG_PDL, stream);
    check(rc, "qf_w8a8_gemm");
  }
  return y.view(out_shape);
}

at::Tensor int8_linear_meta(const at::Tensor& x, const at::Tensor& w_q, const at::Tensor& w_s,
                            const c10::optional<at::Tensor>& bias) {
  std::vector<c10::SymInt> out_shape = x.sym_sizes().vec();
  out_shape.back() = w_q.sym_size(1);
  return at::empty_symint(out_shape, x.options());
}

// ---------------------------------------------------------------------------------------- block-scaled fp8 layers
constexpr int64_t kBlock = 128;
int64_t blocks(int64_t v) { return (v + kBlock - 1) / kBlock; }
c10::SymInt blocks(const c10::SymInt& v) { return (v + (kBlock - 1)) / kBlock; }

// ---- types and shapes, of real calls and of traced ones (whose sizes may be symbolic) ----
void check_quantize_shapes(const at::Tensor& x, bool silu_mul) {
  const char* op = "fp8_quantize";
  QF_REFUSE_UNLESS(x.dim() >= 1, op, ": x must have at least one dimension");
  check_type(op, "x", x, at::kBFloat16);
  if (silu_mul)
    QF_REFUSE_UNLESS_EQ(x.sym_size(-1) % 2, 0, op, ": silu_mul needs gate and up halves of one width");
}

void check_weight_shapes(const char* op, const at::Tensor& w_t, const at::Tensor& w_scale, const OptTensor& bias,
                         const c10::SymInt& K) {
  check_type(op, "w_t", w_t, at::kFloat8_e4m3fn);
  QF_REFUSE_UNLESS(w_t.dim() == 2, op, ": w_t must be [K, N], got ", w_t.sym_sizes());
  QF_REFUSE_UNLESS_EQ(w_t.sym_size(0), K, op, ": w_t must be [K, N] with K = ", K, ", got ", w_t.sym_sizes());
  const c10::SymInt N = w_t.sym_size(1);
  check_type(op, "w_scale", w_scale, at::kFloat);
  QF_REFUSE_UNLESS(w_scale.dim() == 2, op, ": w_scale must have two dimensions");
  for (int i = 0; i < 2; ++i)
    QF_REFUSE_UNLESS_EQ(w_scale.sym_size(i), blocks(i ? K : N), op, ": w_scale must be [", blocks(N), ", ", blocks(K),
                        "], got ", w_scale.sym_sizes());
  if (given(bias)) {
    check_type(op, "bias", *bias, at::kBFloat16);
    QF_REFUSE_UNLESS_EQ(bias->sym_numel(), N, op, ": bias must hold ", N, " values");
  }
}

void check_mm_shapes(const char* op, const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& w_t,
                     const at::Tensor& w_scale, const OptTensor& bias) {
  QF_REFUSE_UNLESS(a.dim() == 2, op, ": a must be [M, K]");
  check_type(op, "a", a, at::kFloat8_e4m3fn);
  const c10::SymInt M = a.sym_size(0), K = a.sym_size(1);
  check_weight_shapes(op, w_t, w_scale, bias, K);
  check_type(op, "a_scale", a_scale, at::kFloat);
  QF_REFUSE_UNLESS(a_scale.dim() == 2, op, ": a_scale must have two dimensions");
  for (int i = 0; i < 2; ++i)
    QF_REFUSE_UNLESS_EQ(a_scale.sym_size(i), i ? blocks(K) : M, op, ": a_scale must be [", M, ", ", blocks(K), "], got ",
                        a_scale.sym_sizes());
}

void check_out_shapes(const char* op, const at::Tensor& out, const at::Tensor& a, const at::Tensor& w_t) {
  const c10::SymInt M = a.sym_size(0), N = w_t.sym_size(1);
  QF_REFUSE_UNLESS(out.dim() == 2 && (out.scalar_type() == at::kFloat || out.scalar_type() == at::kBFloat16), op,
                   ": out must be bf16 or fp32 [", M, ", ", N, "]");
  for (int i = 0; i < 2; ++i)
    QF_REFUSE_UNLESS_EQ(out.sym_size(i), i ? N : M, op, ": out must be bf16 or fp32 [", M, ", ", N, "], got ",
                        out.sym_sizes());
}

void check_linear_shapes(const char* op, const at::Tensor& x, const at::Tensor& w_t, const at::Tensor& w_scale,
                         const OptTensor& bias) {
  QF_REFUSE_UNLESS(x.dim() >= 1, op, ": x must have at least one dimension");
  check_type(op, "x", x, at::kBFloat16);
  check_weight_shapes(op, w_t, w_scale, bias, x.sym_size(-1));
}

void check_same_sizes(const char* op, const char* name, const at::Tensor& t, const at::Tensor& x) {
  QF_REFUSE_UNLESS(t.dim() == x.dim(), op, ": ", name, " must have x's shape ", x.sym_sizes(), ", got ", t.sym_sizes());
  // (an equality at a time, so that a symbolic one is taken as a fact)
  for (int64_t i = 0; i < x.dim(); ++i)
    QF_REFUSE_UNLESS_EQ(t.sym_size(i), x.sym_size(i), op, ": ", name, " must have x's shape ", x.sym_sizes(), ", got ",
                        t.sym_sizes());
}

void check_norm_shapes(const at::Tensor& x, const OptTensor& residual, const OptTensor& pre_weight,
                       const OptTensor& post_weight, const OptTensor& gate, int64_t gate_act, double eps, bool quantize) {
  const char* op = "residual_norm";
  QF_REFUSE_UNLESS(x.dim() >= 1, op, ": x must have at least one dimension");
  check_type(op, "x", x, at::kBFloat16);
  if (given(residual)) {
    QF_REFUSE_UNLESS(residual->scalar_type() == at::kBFloat16 || residual->scalar_type() == at::kFloat, op,
                     ": residual must be bf16 or fp32");
    check_same_sizes(op, "residual", *residual, x);
  }
  for (const auto& [name, w] : {std::make_pair("pre_weight", &pre_weight), std::make_pair("post_weight", &post_weight)})
    if (given(*w)) {
      check_type(op, name, **w, at::kBFloat16);
      QF_REFUSE_UNLESS((*w)->dim() == 1, op, ": ", name, " must be [", x.sym_size(-1), "]");
      QF_REFUSE_UNLESS_EQ((*w)->sym_size(0), x.sym_size(-1), op, ": ", name, " must be [", x.sym_size(-1), "]");
    }
  QF_REFUSE_UNLESS(!quantize || given(pre_weight), op, ": quantize needs pre_weight");
  QF_REFUSE_UNLESS(gate_act >= QF_GATE_NONE && gate_act <= QF_GATE_SILU, op, ": unknown gate activation");
  if (given(gate)) {
    check_type(op, "gate", *gate, at::kBFloat16);
    QF_REFUSE_UNLESS(gate->dim() <= x.dim(), op, ": gate has more dimensions than x");
    for (int64_t i = 1; i <= gate->dim(); ++i) {
      const std::optional<int64_t> g = gate->sym_size(-i).maybe_as_int();
      if (!g || *g != 1)
        QF_REFUSE_UNLESS_EQ(gate->sym_size(-i), x.sym_size(-i), op, ": gate ", gate->sym_sizes(), " does not broadcast to ",
                            x.sym_sizes());
    }
  } else {
    QF_REFUSE_UNLESS(gate_act == QF_GATE_NONE, op, ": a gate activation without a gate");
  }
  QF_REFUSE_UNLESS(eps >= 0 && eps <= 3.4e38, op, ": eps must be finite and >= 0");
}

// Rows of [..., K], K >= 1.
int64_t rows_of(const at::Tensor& x) { return x.dim() == 2 ? x.size(0) : x.numel() / x.size(-1); }

void check_groups(const char* op, int64_t M, int64_t K) {
  QF_REFUSE_UNLESS(M <= INT32_MAX && M * blocks(K) <= INT32_MAX, op, ": ", M, " rows of ", blocks(K),
                   " groups are more than 2^31 - 1 groups");
}

// What the product takes (the last limit is the one on its tiles).
void check_rows(const char* op, int64_t M, int64_t N) {
  QF_REFUSE_UNLESS(M <= QF_FP8_MAX_M && (M + 127) / 128 * ((N + 63) / 64) < INT32_MAX - 4095, op, ": ", M, " rows of ", N,
                   " results are too many");
}

// [..., K] as rows of unit column stride, without a copy where the strides allow it.
at::Tensor as_rows(const at::Tensor& x) {
  at::Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if (r.size(1) > 1 && r.stride(1) != 1) r = r.contiguous();
  if (r.size(0) > 1 && r.stride(0) < r.size(1)) r = r.contiguous();  // broadcast or overlapping rows
  return r;
}

// The rows of a result with x's leading dimensions (a view).
at::Tensor with_leading(const at::Tensor& rows, const at::Tensor& x) {
  if (x.dim() == 2) return rows;
  return x.dim() == 1 ? rows.select(0, 0) : rows.unflatten(0, x.sizes().slice(0, x.dim() - 1));
}

// e4m3 rows of 16-byte stride, as the product's tensor maps take them.
at::Tensor empty_rows(int64_t M, int64_t K, const at::Tensor& like) {
  at::Tensor q = empty_on(like, {M, (K + 15) / 16 * 16}, at::kFloat8_e4m3fn);
  return K % 16 ? q.narrow(1, 0, K) : q;
}

std::tuple<at::Tensor, at::Tensor> quantize_rows(const at::Tensor& x2, bool silu_mul) {
  const int64_t M = x2.size(0), K = silu_mul ? x2.size(1) / 2 : x2.size(1);
  at::Tensor q = empty_rows(M, K, x2);
  at::Tensor s = empty_on(x2, {M, blocks(K)}, at::kFloat);
  if (M && K)
    check(qf_fp8_quantize(x2.data_ptr(), x2.stride(0), static_cast<int>(M), static_cast<int>(K), silu_mul, q.data_ptr(),
                          q.stride(0), s.data_ptr<float>(), s.stride(0), QF_FLAG_PDL, stream_of(x2)),
          "qf_fp8_quantize");
  return {q, s};
}

std::tuple<at::Tensor, at::Tensor> fp8_quantize(const at::Tensor& x, bool silu_mul) {
  check_quantize_shapes(x, silu_mul);
  const int64_t K = silu_mul ? x.size(-1) / 2 : x.size(-1);
  QF_REFUSE_UNLESS(K >= 1 && K <= QF_FP8_MAX_K, "fp8_quantize: 1 to ", QF_FP8_MAX_K, " values per row, got ", K);
  check_input("fp8_quantize", "x", x, x.device());
  check_groups("fp8_quantize", rows_of(x), K);
  c10::cuda::CUDAGuard guard(x.device());
  auto [q, s] = quantize_rows(as_rows(x), silu_mul);
  return {with_leading(q, x), with_leading(s, x)};
}

void check_weight(const char* op, const at::Tensor& w_t, const at::Tensor& w_scale, const OptTensor& bias,
                  const at::Device& dev) {
  check_input(op, "w_t", w_t, dev);
  const int64_t K = w_t.size(0), N = w_t.size(1);
  QF_REFUSE_UNLESS(K >= 1 && K <= QF_FP8_MAX_K && N <= QF_MAX_N, op, ": K must be 1 to ", QF_FP8_MAX_K,
                   " and N at most ", QF_MAX_N);
  QF_REFUSE_UNLESS((K == 1 || w_t.stride(0) == 1) && (N <= 1 || (w_t.stride(1) >= K && w_t.stride(1) % 16 == 0)) &&
                       reinterpret_cast<uintptr_t>(w_t.data_ptr()) % 16 == 0,
                   op, ": w_t must be the [K, N] view of 16-byte aligned rows of a weight (stride (1, ldw), ldw a multiple "
                   "of 16)");
  check_input(op, "w_scale", w_scale, dev);
  if (given(bias)) check_input(op, "bias", *bias, dev);
}

void run_mm(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& w_t,
            const at::Tensor& w_scale, const OptTensor& bias, at::Tensor& y) {
  const int64_t M = a.size(0), K = a.size(1), N = w_t.size(1);
  if (M == 0 || N == 0) return;
  at::Tensor b;
  if (given(bias)) b = bias->reshape({-1}).contiguous();
  check(qf_fp8_block_gemm(a.data_ptr(), a.stride(0), a_scale.data_ptr<float>(), a_scale.stride(0), a_scale.stride(1),
                          w_t.data_ptr(), N > 1 ? w_t.stride(1) : K, w_scale.data_ptr<float>(), w_scale.stride(0),
                          w_scale.stride(1), b.defined() ? b.data_ptr() : nullptr, y.data_ptr(), y.stride(0),
                          y.scalar_type() == at::kFloat ? QF_DTYPE_F32 : QF_DTYPE_BF16, static_cast<int>(M),
                          static_cast<int>(N), static_cast<int>(K), QF_FLAG_PDL, stream_of(a)),
        "qf_fp8_block_gemm");
}

void check_mm(const char* op, const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& w_t,
              const at::Tensor& w_scale, const OptTensor& bias) {
  check_mm_shapes(op, a, a_scale, w_t, w_scale, bias);
  check_input(op, "a", a, a.device());
  check_weight(op, w_t, w_scale, bias, a.device());
  check_input(op, "a_scale", a_scale, a.device());
  check_rows(op, a.size(0), w_t.size(1));
}

// a with rows that the product's tensor maps take, copied where they are not.
at::Tensor aligned_rows(const at::Tensor& a) {
  const int64_t M = a.size(0), K = a.size(1);
  const bool fits = (K == 1 || a.stride(1) == 1) && (M <= 1 || (a.stride(0) >= K && a.stride(0) % 16 == 0)) &&
                    reinterpret_cast<uintptr_t>(a.data_ptr()) % 16 == 0;
  if (fits || M == 0) return a;
  at::Tensor r = empty_rows(M, K, a);
  r.copy_(a);
  return r;
}

at::Tensor fp8_block_mm(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& w_t,
                        const at::Tensor& w_scale, const OptTensor& bias, bool out_f32) {
  c10::cuda::OptionalCUDAGuard guard(a.is_cuda() ? c10::optional<c10::Device>(a.device()) : c10::nullopt);
  check_mm("fp8_block_mm", a, a_scale, w_t, w_scale, bias);
  const at::Tensor r = aligned_rows(a);
  at::Tensor y = empty_on(a, {a.size(0), w_t.size(1)}, out_f32 ? at::kFloat : at::kBFloat16);
  run_mm(r, a_scale, w_t, w_scale, bias, y);
  return y;
}

void fp8_block_mm_out(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& w_t, const at::Tensor& w_scale,
                      const OptTensor& bias, at::Tensor out) {
  const char* op = "fp8_block_mm";
  c10::cuda::OptionalCUDAGuard guard(a.is_cuda() ? c10::optional<c10::Device>(a.device()) : c10::nullopt);
  check_mm(op, a, a_scale, w_t, w_scale, bias);
  check_out_shapes(op, out, a, w_t);
  const int64_t M = a.size(0), N = w_t.size(1);
  QF_REFUSE_UNLESS(out.device() == a.device() && (N == 1 || out.stride(1) == 1) && (M <= 1 || out.stride(0) >= N), op,
                   ": out must be on a's device with unit column stride and rows that do not overlap");
  check_no_overlap(op, "out", out, "a", a);
  check_no_overlap(op, "out", out, "a_scale", a_scale);
  check_no_overlap(op, "out", out, "w_t", w_t);
  check_no_overlap(op, "out", out, "w_scale", w_scale);
  if (given(bias)) check_no_overlap(op, "out", out, "bias", *bias);
  run_mm(aligned_rows(a), a_scale, w_t, w_scale, bias, out);
  written(out);
}

at::Tensor fp8_block_linear(const at::Tensor& x, const at::Tensor& w_t, const at::Tensor& w_scale, const OptTensor& bias) {
  const char* op = "fp8_block_linear";
  check_linear_shapes(op, x, w_t, w_scale, bias);
  check_input(op, "x", x, x.device());
  check_weight(op, w_t, w_scale, bias, x.device());
  check_groups(op, rows_of(x), x.size(-1));
  check_rows(op, rows_of(x), w_t.size(1));
  c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor x2 = as_rows(x);
  at::Tensor y = empty_on(x, {x2.size(0), w_t.size(1)}, at::kBFloat16);
  if (x2.size(0) && w_t.size(1)) {
    auto [q, s] = quantize_rows(x2, false);
    run_mm(q, s, w_t, w_scale, bias, y);
  }
  return with_leading(y, x);
}

// What residual_norm and residual_norm_out share; `r_out` is where the new residual goes.  Returns (h, scale), each
// undefined where it is not asked for.
std::tuple<at::Tensor, at::Tensor> run_norm(const at::Tensor& x, const OptTensor& residual, const OptTensor& pre_weight,
                                            const OptTensor& post_weight, const OptTensor& gate, int64_t gate_act,
                                            double residual_scale, double weight_offset, double eps, bool quantize,
                                            at::Tensor& r_out) {
  const int64_t H = x.size(-1);
  const at::Tensor x2 = as_rows(x);
  const int64_t M = x2.size(0);
  at::Tensor r2, g2, post, pre, h, s;
  if (given(residual)) r2 = as_rows(*residual);
  int64_t gm = 0, gh = 0;
  if (given(gate)) {
    // broadcast to the rows; the kernel takes a column stride of zero or one and any row stride
    g2 = gate->dim() == 2 && x.dim() == 2 ? gate->expand({M, H}) : gate->expand(x.sizes()).reshape({M, H});
    if (H > 1 && g2.stride(1) != 0 && g2.stride(1) != 1) g2 = g2.contiguous();
    gm = M > 1 ? g2.stride(0) : 0;
    gh = H > 1 ? g2.stride(1) : 0;
  }
  if (given(post_weight)) post = post_weight->contiguous();
  const bool want_h = given(pre_weight);
  if (want_h) {
    pre = pre_weight->contiguous();
    h = quantize ? empty_rows(M, H, x) : empty_on(x, {M, H}, at::kBFloat16);
    if (quantize) s = empty_on(x, {M, blocks(H)}, at::kFloat);
  }
  at::Tensor ro2 = r_out.dim() == 2 ? r_out : r_out.view({M, H});
  if (M) {
    auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    auto ld = [](const at::Tensor& t) { return t.defined() ? t.stride(0) : 0; };
    check(qf_residual_norm(ptr(x2), ld(x2), ptr(r2), ld(r2),
                           r_out.scalar_type() == at::kFloat ? QF_DTYPE_F32 : QF_DTYPE_BF16, ptr(g2), gm, gh,
                           static_cast<int>(gate_act), ptr(post), ptr(pre), static_cast<float>(weight_offset),
                           static_cast<float>(residual_scale), static_cast<float>(eps), ro2.data_ptr(), ro2.stride(0),
                           ptr(h), ld(h), s.defined() ? s.data_ptr<float>() : nullptr, ld(s), static_cast<int>(M),
                           static_cast<int>(H), QF_FLAG_PDL, stream_of(x)),
          "qf_residual_norm");
  }
  if (h.defined()) h = with_leading(h, x);
  if (s.defined()) s = with_leading(s, x);
  return {h, s};
}

void check_norm(const at::Tensor& x, const OptTensor& residual, const OptTensor& pre_weight, const OptTensor& post_weight,
                const OptTensor& gate, int64_t gate_act, double eps, bool quantize) {
  const char* op = "residual_norm";
  check_norm_shapes(x, residual, pre_weight, post_weight, gate, gate_act, eps, quantize);
  check_input(op, "x", x, x.device());
  const int64_t H = x.size(-1);
  QF_REFUSE_UNLESS(H >= 1 && H <= QF_NORM_MAX_H, op, ": rows of 1 to ", QF_NORM_MAX_H, " values, got ", H);
  QF_REFUSE_UNLESS(rows_of(x) <= INT32_MAX, op, ": ", rows_of(x), " rows are too many");
  if (given(residual)) check_input(op, "residual", *residual, x.device());
  if (given(pre_weight)) check_input(op, "pre_weight", *pre_weight, x.device());
  if (given(post_weight)) check_input(op, "post_weight", *post_weight, x.device());
  if (given(gate)) check_input(op, "gate", *gate, x.device());
}

std::tuple<OptTensor, OptTensor, at::Tensor> residual_norm(const at::Tensor& x, const OptTensor& residual,
                                                           const OptTensor& pre_weight, const OptTensor& post_weight,
                                                           const OptTensor& gate, int64_t gate_act, double residual_scale,
                                                           double weight_offset, double eps, bool quantize) {
  check_norm(x, residual, pre_weight, post_weight, gate, gate_act, eps, quantize);
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor r_out = empty_on(x, x.sizes(), given(residual) ? residual->scalar_type() : at::kBFloat16);
  auto [h, s] = run_norm(x, residual, pre_weight, post_weight, gate, gate_act, residual_scale, weight_offset, eps, quantize,
                         r_out);
  return {h.defined() ? OptTensor(h) : c10::nullopt, s.defined() ? OptTensor(s) : c10::nullopt, r_out};
}

std::tuple<OptTensor, OptTensor> residual_norm_out(const at::Tensor& x, const OptTensor& residual,
                                                   const OptTensor& pre_weight, const OptTensor& post_weight,
                                                   const OptTensor& gate, int64_t gate_act, double residual_scale,
                                                   double weight_offset, double eps, bool quantize,
                                                   at::Tensor residual_out) {
  const char* op = "residual_norm";
  check_norm(x, residual, pre_weight, post_weight, gate, gate_act, eps, quantize);
  const at::ScalarType type = given(residual) ? residual->scalar_type() : at::kBFloat16;
  check_type(op, "residual_out", residual_out, type);
  check_input(op, "residual_out", residual_out, x.device());
  check_same_sizes(op, "residual_out", residual_out, x);
  const int64_t H = x.size(-1);
  QF_REFUSE_UNLESS((H == 1 || residual_out.stride(-1) == 1) && (residual_out.dim() == 2 || residual_out.is_contiguous()) &&
                       (residual_out.dim() != 2 || residual_out.size(0) <= 1 || residual_out.stride(0) >= H),
                   op, ": residual_out must have unit column stride and rows that do not overlap (and be contiguous "
                   "unless it is 2-D)");
  // the residual itself is updated in place; any other overlap would be read after it is written
  if (given(residual) && !same_elements(*residual, residual_out))
    check_no_overlap(op, "residual_out", residual_out, "residual", *residual);
  check_no_overlap(op, "residual_out", residual_out, "x", x);
  if (given(pre_weight)) check_no_overlap(op, "residual_out", residual_out, "pre_weight", *pre_weight);
  if (given(post_weight)) check_no_overlap(op, "residual_out", residual_out, "post_weight", *post_weight);
  if (given(gate)) check_no_overlap(op, "residual_out", residual_out, "gate", *gate);
  c10::cuda::CUDAGuard guard(x.device());
  auto [h, s] = run_norm(x, residual, pre_weight, post_weight, gate, gate_act, residual_scale, weight_offset, eps, quantize,
                         residual_out);
  written(residual_out);
  return {h.defined() ? OptTensor(h) : c10::nullopt, s.defined() ? OptTensor(s) : c10::nullopt};
}

// Types and shapes only, for tracing: the same refusals of them, the same leading dimensions (which may be symbolic), e4m3
// rows of 16-byte stride.
at::Tensor meta_rows(const at::Tensor& x, const c10::SymInt& K) {
  std::vector<c10::SymInt> s = x.sym_sizes().vec();
  s.back() = (K + 15) / 16 * 16;
  at::Tensor q = at::empty_symint(s, x.options().dtype(at::kFloat8_e4m3fn));
  const std::optional<int64_t> k = K.maybe_as_int();
  return k && *k % 16 == 0 ? q : q.narrow_symint(-1, 0, K);
}
at::Tensor meta_like(const at::Tensor& x, const c10::SymInt& last, at::ScalarType type) {
  std::vector<c10::SymInt> s = x.sym_sizes().vec();
  s.back() = last;
  return at::empty_symint(s, x.options().dtype(type));
}
std::tuple<at::Tensor, at::Tensor> fp8_quantize_meta(const at::Tensor& x, bool silu_mul) {
  check_quantize_shapes(x, silu_mul);
  const c10::SymInt K = silu_mul ? x.sym_size(-1) / 2 : x.sym_size(-1);
  return {meta_rows(x, K), meta_like(x, blocks(K), at::kFloat)};
}
at::Tensor fp8_block_mm_meta(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& w_t,
                             const at::Tensor& w_scale, const OptTensor& bias, bool out_f32) {
  check_mm_shapes("fp8_block_mm", a, a_scale, w_t, w_scale, bias);
  return meta_like(a, w_t.sym_size(1), out_f32 ? at::kFloat : at::kBFloat16);
}
void fp8_block_mm_out_meta(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& w_t, const at::Tensor& w_scale,
                           const OptTensor& bias, at::Tensor out) {
  check_mm_shapes("fp8_block_mm", a, a_scale, w_t, w_scale, bias);
  check_out_shapes("fp8_block_mm", out, a, w_t);
  written(out);
}
at::Tensor fp8_block_linear_meta(const at::Tensor& x, const at::Tensor& w_t, const at::Tensor& w_scale,
                                 const OptTensor& bias) {
  check_linear_shapes("fp8_block_linear", x, w_t, w_scale, bias);
  return meta_like(x, w_t.sym_size(1), at::kBFloat16);
}
// (h, scale) of a call without refusals left.
std::tuple<OptTensor, OptTensor> meta_h(const at::Tensor& x, const OptTensor& pre_weight, bool quantize) {
  if (!given(pre_weight)) return {c10::nullopt, c10::nullopt};
  if (!quantize) return {meta_like(x, x.sym_size(-1), at::kBFloat16), c10::nullopt};
  return {meta_rows(x, x.sym_size(-1)), meta_like(x, blocks(x.sym_size(-1)), at::kFloat)};
}
std::tuple<OptTensor, OptTensor> residual_norm_out_meta(const at::Tensor& x, const OptTensor& residual,
                                                        const OptTensor& pre_weight, const OptTensor& post_weight,
                                                        const OptTensor& gate, int64_t gate_act, double, double, double eps,
                                                        bool quantize, at::Tensor residual_out) {
  check_norm_shapes(x, residual, pre_weight, post_weight, gate, gate_act, eps, quantize);
  check_type("residual_norm", "residual_out", residual_out, given(residual) ? residual->scalar_type() : at::kBFloat16);
  check_same_sizes("residual_norm", "residual_out", residual_out, x);
  written(residual_out);
  return meta_h(x, pre_weight, quantize);
}
std::tuple<OptTensor, OptTensor, at::Tensor> residual_norm_meta(const at::Tensor& x, const OptTensor& residual,
                                                                const OptTensor& pre_weight, const OptTensor& post_weight,
                                                                const OptTensor& gate, int64_t gate_act, double, double,
                                                                double eps, bool quantize) {
  check_norm_shapes(x, residual, pre_weight, post_weight, gate, gate_act, eps, quantize);
  auto [h, s] = meta_h(x, pre_weight, quantize);
  return {h, s, meta_like(x, x.sym_size(-1), given(residual) ? residual->scalar_type() : at::kBFloat16)};
}

}  // namespace

TORCH_LIBRARY(qf_b200, m) {
  m.def("int8_linear(Tensor x, Tensor w_q, Tensor w_s, Tensor? bias) -> Tensor");
  m.def("fp8_quantize(Tensor x, bool silu_mul) -> (Tensor, Tensor)");
  m.def("fp8_block_mm(Tensor a, Tensor a_scale, Tensor w_t, Tensor w_scale, Tensor? bias, bool out_f32) -> Tensor");
  m.def("fp8_block_mm_out(Tensor a, Tensor a_scale, Tensor w_t, Tensor w_scale, Tensor? bias, Tensor(a!) out) -> ()");
  m.def("fp8_block_linear(Tensor x, Tensor w_t, Tensor w_scale, Tensor? bias) -> Tensor");
  m.def("residual_norm(Tensor x, Tensor? residual, Tensor? pre_weight, Tensor? post_weight, Tensor? gate, int gate_act, "
        "float residual_scale, float weight_offset, float eps, bool quantize) -> (Tensor?, Tensor?, Tensor)");
  m.def("residual_norm_out(Tensor x, Tensor? residual, Tensor? pre_weight, Tensor? post_weight, Tensor? gate, int gate_act, "
        "float residual_scale, float weight_offset, float eps, bool quantize, Tensor(a!) residual_out) -> "
        "(Tensor?, Tensor?)");
}
// CompositeExplicitAutograd: CPU tensors reach the operators' own refusals instead of the dispatcher's.
TORCH_LIBRARY_IMPL(qf_b200, CompositeExplicitAutograd, m) {
  m.impl("fp8_quantize", fp8_quantize);
  m.impl("fp8_block_mm", fp8_block_mm);
  m.impl("fp8_block_mm_out", fp8_block_mm_out);
  m.impl("fp8_block_linear", fp8_block_linear);
  m.impl("residual_norm", residual_norm);
  m.impl("residual_norm_out", residual_norm_out);
}
TORCH_LIBRARY_IMPL(qf_b200, Autograd, m) {
  for (const char* op : {"fp8_quantize", "fp8_block_mm", "fp8_block_mm_out", "fp8_block_linear", "residual_norm",
                         "residual_norm_out"})
    m.impl(op, torch::CppFunction::makeFromBoxedFunction<&refuse_derivatives>());
}
TORCH_LIBRARY_IMPL(qf_b200, CUDA, m) { m.impl("int8_linear", int8_linear); }
TORCH_LIBRARY_IMPL(qf_b200, Meta, m) {
  m.impl("int8_linear", int8_linear_meta);
  m.impl("fp8_quantize", fp8_quantize_meta);
  m.impl("fp8_block_mm", fp8_block_mm_meta);
  m.impl("fp8_block_mm_out", fp8_block_mm_out_meta);
  m.impl("fp8_block_linear", fp8_block_linear_meta);
  m.impl("residual_norm", residual_norm_meta);
  m.impl("residual_norm_out", residual_norm_out_meta);
}
