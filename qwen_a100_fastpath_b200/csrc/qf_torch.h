// qf_torch.h -- what the PyTorch operators over the C ABI share: refusals, overlap checks, allocation.  Included once by each
// of the operator layer's sources.
#pragma once
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <cstdint>

#include "../../include/qf_b200.h"

namespace qf_torch {

inline void check(int rc, const char* fn) {
  TORCH_CHECK(rc == QF_OK, fn, ": ", qf_strerror(rc), " (", rc, "): ", qf_last_error_detail());
}

#define QF_REFUSE_UNLESS(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)
// Equality of sizes that may be symbolic: tracing goes on with it as a fact and fixes neither side.
inline bool same_size(const c10::SymInt& a, const c10::SymInt& b) {
  if (C10_LIKELY(!a.is_heap_allocated() && !b.is_heap_allocated())) return a.as_int_unchecked() == b.as_int_unchecked();
  return a.sym_eq(b).expect_true(__FILE__, __LINE__);
}
#define QF_REFUSE_UNLESS_EQ(a, b, ...) TORCH_CHECK_VALUE(same_size(a, b), __VA_ARGS__)

using OptTensor = c10::optional<at::Tensor>;

inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

inline void check_type(const char* op, const char* name, const at::Tensor& t, at::ScalarType type) {
  QF_REFUSE_UNLESS(t.scalar_type() == type, op, ": ", name, " must be ", type, ", got ", t.scalar_type());
}

inline void check_input(const char* op, const char* name, const at::Tensor& t, const at::Device& dev) {
  QF_REFUSE_UNLESS(t.is_cuda(), op, ": ", name, " must be a CUDA tensor (there is no CPU path)");
  QF_REFUSE_UNLESS(t.device() == dev, op, ": ", name, " is on ", t.device(), ", the first input on ", dev);
}

// In the place of torch's fallback for operators without a backward: refuses tensors that want a derivative, outputs among
// them, and goes on to the operator.  Here the derivatives of torch.func's transformations can be seen too.
inline void refuse_derivatives(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const bool backward = at::GradMode::is_enabled();
  const bool forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  const size_t n = op.schema().arguments().size();
  for (size_t i = 0; i < n; ++i) {
    const c10::IValue& v = (*stack)[stack->size() - n + i];
    if (!v.isTensor()) continue;
    const at::Tensor& t = v.toTensor();
    if (!t.defined()) continue;
    QF_REFUSE_UNLESS(!(backward && t.requires_grad()), op.schema().name(), ": ", op.schema().arguments()[i].name(),
                     " requires a gradient and the operator has no backward (call it under torch.no_grad())");
    QF_REFUSE_UNLESS(!(forward && t._fw_grad(0).defined()), op.schema().name(), ": ", op.schema().arguments()[i].name(),
                     " has a forward-mode tangent and the operator has no derivative");
  }
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

// A tensor was written: autograd tells by its version where a value it kept is no longer there.
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

inline cudaStream_t stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The bytes of a tensor as `rows` intervals of `width` bytes, `step` bytes apart.  Exact for rows of adjacent elements; what
// lies between the elements of other tensors counts as theirs (`overlap` looks closer where these intervals meet).
struct Intervals {
  int64_t begin, width, step, rows;
  int64_t end() const { return begin + (rows - 1) * step + width; }
};

inline Intervals intervals_of(const at::Tensor& t) {
  // the dimension of the largest stride gives the rows, the others' span their width
  int64_t rows = 1, step = 0, span = 1;
  int outer = -1;
  for (int i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) > step) step = t.stride(i), rows = t.size(i), outer = i;
  for (int i = 0; i < t.dim(); ++i)
    if (i != outer && t.size(i) > 1) span += (t.size(i) - 1) * t.stride(i);
  const int64_t es = static_cast<int64_t>(t.element_size());
  Intervals v = {static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.data_ptr())), span * es, step * es, rows};
  if (v.width >= v.step) v = {v.begin, (v.rows - 1) * v.step + v.width, 0, 1};  // adjacent or overlapping rows: one interval
  return v;
}

inline bool spans_overlap(const at::Tensor& ta, const at::Tensor& tb) {
  if (ta.numel() == 0 || tb.numel() == 0) return false;
  Intervals a = intervals_of(ta), b = intervals_of(tb);
  if (a.end() <= b.begin || b.end() <= a.begin) return false;
  if (a.rows > 1 && b.rows > 1 && a.step == b.step) {
    // columns of one larger tensor: the rows' places within a step decide
    const int64_t at = ((b.begin - a.begin) % a.step + a.step) % a.step;
    if (at >= a.width && at + b.width <= a.step) return false;
  }
  // walk both upwards, always on with the row that ends first
  int64_t i = 0, j = 0;
  // rows that end before the other begins
  if (a.step && b.begin > a.begin + a.width) i = (b.begin - a.begin - a.width) / a.step;
  if (b.step && a.begin > b.begin + b.width) j = (a.begin - b.begin - b.width) / b.step;
  while (i < a.rows && j < b.rows) {
    const int64_t pa = a.begin + i * a.step, pb = b.begin + j * b.step;
    if (pa < pb + b.width && pb < pa + a.width) return true;
    if (pa + a.width <= pb) ++i; else ++j;
  }
  return false;
}

// The bytes of a tensor as runs of span[n] adjacent bytes, repeated at nested strides, the largest first; level l and those
// inside it reach over span[l] bytes.  For up to kLevels strides.
struct Runs {
  static constexpr int kLevels = 8;
  int64_t begin = 0, stride[kLevels], size[kLevels], span[kLevels + 1];
  int n = 0;
  bool fits = true;
  explicit Runs(const at::Tensor& t) : begin(static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.data_ptr()))) {
    const int64_t es = static_cast<int64_t>(t.element_size());
    for (int i = 0; i < t.dim(); ++i) {
      if (t.size(i) == 1 || t.stride(i) == 0) continue;
      if (n == kLevels) {
        fits = false;
        return;
      }
      int at = n++;
      for (; at > 0 && stride[at - 1] < t.stride(i) * es; --at) stride[at] = stride[at - 1], size[at] = size[at - 1];
      stride[at] = t.stride(i) * es, size[at] = t.size(i);
    }
    int64_t run = es;
    while (n > 0 && stride[n - 1] == run) run *= size[--n];
    for (int i = n - 1; i > 0; --i)
      if (stride[i - 1] == stride[i] * size[i]) {  // rows of rows without a gap between: one level
        stride[i - 1] = stride[i], size[i - 1] *= size[i];
        for (int j = i; j + 1 < n; ++j) stride[j] = stride[j + 1], size[j] = size[j + 1];
        --n;
      }
    span[n] = run;
    for (int i = n - 1; i >= 0; --i) span[i] = (size[i] - 1) * stride[i] + span[i + 1];
  }
};

inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }

// Whether bytes of a's levels from la on and of b's from lb on, d bytes further, are the same; exact within `budget` steps,
// true beyond it.  Levels of one stride are taken together: only rows whose distance brings them within reach of one another
// are looked at, two or three of any number.
inline bool runs_meet(const Runs& a, int la, const Runs& b, int lb, int64_t d, int* budget) {
  if (d >= a.span[la] || -d >= b.span[lb]) return false;
  if (la == a.n && lb == b.n) return true;
  if (--*budget < 0) return true;
  const int64_t sa = la < a.n ? a.stride[la] : 0, sb = lb < b.n ? b.stride[lb] : 0;
  const int ia = la + (sa >= sb), ib = lb + (sb >= sa);
  // rows i of a and j of b lie d + m s apart, m = j - i (of the one that steps, where only one does)
  const int64_t s = sa > sb ? sa : sb, ra = sa >= sb ? a.size[la] - 1 : 0, rb = sb >= sa ? b.size[lb] - 1 : 0;
  const int64_t lo = floor_div(-b.span[ib] - d, s) + 1, hi = floor_div(a.span[ia] - d - 1, s);
  for (int64_t m = lo > -ra ? lo : -ra; m <= (hi < rb ? hi : rb); ++m)
    if (runs_meet(a, ia, b, ib, d + m * s, budget)) return true;
  return false;
}

inline bool overlap(const at::Tensor& ta, const at::Tensor& tb) {
  if (!spans_overlap(ta, tb)) return false;
  // views side by side within a row (keys and values of a slot, for instance)
  const Runs a(ta), b(tb);
  int budget = 4096;
  return !a.fits || !b.fits || runs_meet(a, 0, b, 0, b.begin - a.begin, &budget);
}

// Whether two tensors of one shape and type hold the same elements at the same places.
inline bool same_elements(const at::Tensor& a, const at::Tensor& b) {
  if (a.data_ptr() != b.data_ptr()) return false;
  for (int i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

// The bytes from a tensor's first element to the end of its last: where two tensors' do not meet, neither do they.
struct Extent {
  uintptr_t begin, end;
};
inline Extent extent_of(const at::Tensor& t) {
  if (t.numel() == 0) return {0, 0};
  int64_t last = 0;
  const auto sizes = t.sizes(), strides = t.strides();
  for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
  const uintptr_t begin = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {begin, begin + (last + 1) * t.element_size()};
}
inline bool meet(const Extent& a, const Extent& b) { return a.begin < b.end && b.begin < a.end; }

// "single memory location" is what torch's own operators say of such a call.
inline void check_no_overlap(const char* op, const char* out_name, const at::Tensor& out, const char* name, const at::Tensor& t) {
  QF_REFUSE_UNLESS(!overlap(out, t), op, ": ", out_name, " shares memory with ", name,
                   ": elements of the two refer to a single memory location");
}

// A new tensor of the caching allocator, without the dispatcher's share of a small call's time.
inline at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}

}  // namespace qf_torch
