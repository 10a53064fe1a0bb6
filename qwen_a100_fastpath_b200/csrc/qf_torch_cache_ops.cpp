// qf_torch_cache_ops.cpp -- the PyTorch operators of a step on the 4-bit paged cache, over the C ABI of libqf_b200
// (include/qf_b200.h): torch.ops.qf_b200.step_maps / step_maps_grow (paged.py documents them), qk_norm_rope /
// qk_norm_rope_kv4 (norms.py), kv4_write / kv4_read / kv4_attention / kv4_attention_out (kv4.py).
//
// As the operators of qf_torch_ops.cpp: what they make, the attention's partial sums among it, comes from the caching
// allocator, so that calls on several streams, and captured graphs, share nothing.  A call that cannot be taken raises a
// ValueError before anything is launched, tensors that require a gradient or carry a tangent too.
#include <array>
#include <tuple>
#include <vector>

#include "qf_torch.h"

using namespace qf_torch;

namespace {

// ---- types and shapes, of real calls and of traced ones (whose sizes may be symbolic) ----
void check_dims(const char* op, const char* name, const at::Tensor& t, at::ScalarType type, int64_t dims) {
  check_type(op, name, t, type);
  QF_REFUSE_UNLESS(t.dim() == dims, op, ": ", name, " must have ", dims, " dimension", dims > 1 ? "s" : "", ", got ",
                   t.sym_sizes());
}

struct CacheArgs {
  const at::Tensor &k, &v, &k_scale, &v_scale;
  const at::Tensor& operator[](int i) const { return i == 0 ? k : i == 1 ? v : i == 2 ? k_scale : v_scale; }
  c10::SymInt heads() const { return k.sym_size(1); }
  c10::SymInt head_size() const { return k.sym_size(3) * 2; }
};

void check_cache_shapes(const char* op, const CacheArgs& c) {
  check_dims(op, "cache.k", c.k, at::kByte, 4);
  check_dims(op, "cache.v", c.v, at::kByte, 4);
  check_dims(op, "cache.k_scale", c.k_scale, at::kBFloat16, 5);
  check_dims(op, "cache.v_scale", c.v_scale, at::kBFloat16, 5);
  const std::optional<int64_t> half = c.k.sym_size(3).maybe_as_int();
  QF_REFUSE_UNLESS(half && (*half == 32 || *half == 64 || *half == 128), op,
                   ": the cache's heads must have 64, 128 or 256 values, cache.k has ", c.k.sym_sizes());
  for (int i = 0; i < 4; ++i)
    QF_REFUSE_UNLESS_EQ(c.v.sym_size(i), c.k.sym_size(i), op, ": cache.v must have cache.k's shape ", c.k.sym_sizes(),
                        ", got ", c.v.sym_sizes());
  for (const auto& [name, s] : {std::make_pair("cache.k_scale", &c.k_scale), std::make_pair("cache.v_scale", &c.v_scale)}) {
    for (int i = 0; i < 3; ++i)
      QF_REFUSE_UNLESS_EQ(s->sym_size(i), c.k.sym_size(i), op, ": ", name, " must be [pages, heads, slots, ",
                          *half * 2 / QF_KV4_GROUP, ", 2] like cache.k ", c.k.sym_sizes(), ", got ", s->sym_sizes());
    QF_REFUSE_UNLESS_EQ(s->sym_size(3), *half * 2 / QF_KV4_GROUP, op, ": ", name, " must have ",
                        *half * 2 / QF_KV4_GROUP, " groups, got ", s->sym_sizes());
    QF_REFUSE_UNLESS_EQ(s->sym_size(4), 2, op, ": ", name, " must hold a step and an offset for each group, got ",
                        s->sym_sizes());
  }
}

void check_kv_shapes(const char* op, const char* name, const at::Tensor& x, const CacheArgs& c) {
  check_dims(op, name, x, at::kBFloat16, 3);
  QF_REFUSE_UNLESS_EQ(x.sym_size(1), c.heads(), op, ": ", name, " must be [tokens, ", c.heads(), ", ", c.head_size(),
                      "] like the cache, got ", x.sym_sizes());
  QF_REFUSE_UNLESS_EQ(x.sym_size(2), c.head_size(), op, ": ", name, " must be [tokens, ", c.heads(), ", ", c.head_size(),
                      "] like the cache, got ", x.sym_sizes());
}

void check_per_token(const char* op, const char* name, const at::Tensor& t, const c10::SymInt& tokens) {
  check_dims(op, name, t, at::kLong, 1);
  QF_REFUSE_UNLESS_EQ(t.sym_size(0), tokens, op, ": ", name, " must hold ", tokens, " values, got ", t.sym_sizes());
}

void check_write_shapes(const char* op, const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots,
                        const CacheArgs& c) {
  check_cache_shapes(op, c);
  check_kv_shapes(op, "k", k, c);
  check_kv_shapes(op, "v", v, c);
  QF_REFUSE_UNLESS_EQ(v.sym_size(0), k.sym_size(0), op, ": k and v must have the same tokens, got ", k.sym_sizes(), " and ",
                      v.sym_sizes());
  check_per_token(op, "slots", slots, k.sym_size(0));
}

void check_rope_shapes(const char* op, const at::Tensor& q, const at::Tensor& k, const OptTensor& q_weight,
                       const OptTensor& k_weight, const OptTensor& positions, const OptTensor& cos_sin, double eps) {
  check_dims(op, "q", q, at::kBFloat16, 3);
  check_dims(op, "k", k, at::kBFloat16, 3);
  const c10::SymInt T = q.sym_size(0), D = q.sym_size(2);
  QF_REFUSE_UNLESS_EQ(k.sym_size(0), T, op, ": q and k must have the same tokens, got ", q.sym_sizes(), " and ",
                      k.sym_sizes());
  QF_REFUSE_UNLESS_EQ(k.sym_size(2), D, op, ": q and k must have heads of one size, got ", q.sym_sizes(), " and ",
                      k.sym_sizes());
  for (const auto& [name, w] : {std::make_pair("q_weight", &q_weight), std::make_pair("k_weight", &k_weight)})
    if (given(*w)) {
      check_dims(op, name, **w, at::kBFloat16, 1);
      QF_REFUSE_UNLESS_EQ((*w)->sym_size(0), D, op, ": ", name, " must be [", D, "], got ", (*w)->sym_sizes());
    }
  if (given(cos_sin)) {
    QF_REFUSE_UNLESS(given(positions), op, ": a table of angles needs positions");
    check_per_token(op, "positions", *positions, T);
    QF_REFUSE_UNLESS(cos_sin->scalar_type() == at::kFloat || cos_sin->scalar_type() == at::kBFloat16, op,
                     ": cos_sin must be bf16 or fp32, got ", cos_sin->scalar_type());
    QF_REFUSE_UNLESS(cos_sin->dim() == 2, op, ": cos_sin must be [positions, rotated], got ", cos_sin->sym_sizes());
    const std::optional<int64_t> rot = cos_sin->sym_size(1).maybe_as_int(), d = D.maybe_as_int();
    if (rot) QF_REFUSE_UNLESS(*rot % 2 == 0 && (!d || *rot <= *d), op, ": the rotated part of a head must be even and at most ",
                              D, ", got ", *rot);
  }
  QF_REFUSE_UNLESS(eps >= 0 && eps <= 3.4e38, op, ": eps must be finite and >= 0");
}

void check_attention_shapes(const char* op, const at::Tensor& query, const CacheArgs& c, const at::Tensor& seq_lens,
                            const at::Tensor& block_table, int64_t q_len, double scale) {
  check_cache_shapes(op, c);
  check_dims(op, "query", query, at::kBFloat16, 3);
  QF_REFUSE_UNLESS_EQ(query.sym_size(2), c.head_size(), op, ": the query's heads must have ", c.head_size(),
                      " values, got ", query.sym_sizes());
  check_dims(op, "seq_lens", seq_lens, at::kInt, 1);
  check_dims(op, "block_table", block_table, at::kInt, 2);
  QF_REFUSE_UNLESS(q_len >= 1, op, ": q_len must be at least 1, got ", q_len);
  QF_REFUSE_UNLESS(scale > -3.4e38 && scale < 3.4e38, op, ": scale must be finite");
  const std::optional<int64_t> h = query.sym_size(1).maybe_as_int(), hkv = c.heads().maybe_as_int();
  if (h && hkv) {
    QF_REFUSE_UNLESS(*hkv >= 1 && *h % *hkv == 0, op, ": ", *h, " query heads are no multiple of the cache's ", *hkv);
    QF_REFUSE_UNLESS(q_len <= 64 && q_len * (*h / *hkv) <= 64, op, ": ", q_len, " query tokens of ", *h / *hkv,
                     " heads are more than 64 rows for a key head");
  }
  const std::optional<int64_t> n = query.sym_size(0).maybe_as_int(), b = seq_lens.sym_size(0).maybe_as_int(),
                               rows = block_table.sym_size(0).maybe_as_int();
  if (n && b)
    QF_REFUSE_UNLESS(*n / q_len >= *b, op, ": query has ", *n, " tokens, ", *b, " requests of ", q_len, " need more");
  if (rows && b) QF_REFUSE_UNLESS(*rows >= *b, op, ": block_table has ", *rows, " rows for ", *b, " requests");
}

void check_maps_shapes(const char* op, const at::Tensor& query_lens, const at::Tensor& past_lens,
                       const at::Tensor& block_table, int64_t page_size, int64_t num_tokens) {
  check_dims(op, "query_lens", query_lens, at::kInt, 1);
  check_dims(op, "past_lens", past_lens, at::kInt, 1);
  check_dims(op, "block_table", block_table, at::kInt, 2);
  QF_REFUSE_UNLESS_EQ(past_lens.sym_size(0), query_lens.sym_size(0), op, ": past_lens must be like query_lens ",
                      query_lens.sym_sizes(), ", got ", past_lens.sym_sizes());
  QF_REFUSE_UNLESS_EQ(block_table.sym_size(0), query_lens.sym_size(0), op, ": block_table must have a row for each of ",
                      query_lens.sym_size(0), " requests, got ", block_table.sym_sizes());
  QF_REFUSE_UNLESS(page_size >= 1 && page_size <= INT32_MAX, op, ": page_size must be 1 to 2^31 - 1, got ", page_size);
  QF_REFUSE_UNLESS(num_tokens >= 0 && num_tokens <= INT32_MAX, op, ": num_tokens must be 0 to 2^31 - 1, got ", num_tokens);
}

void check_free_shapes(const char* op, const at::Tensor& free_pages, const at::Tensor& free_head) {
  check_dims(op, "free_pages", free_pages, at::kInt, 1);
  check_dims(op, "free_head", free_head, at::kInt, 1);
  QF_REFUSE_UNLESS_EQ(free_head.sym_size(0), 1, op, ": free_head must hold one value, got ", free_head.sym_sizes());
}

// ---- devices, strides and memory of real calls ----
int64_t stride_of(const at::Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; }

bool at16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// No two elements of a tensor that is written at one place (up to eight dimensions: taken from the smallest stride on, each
// steps over what the ones before span).
bool distinct(const at::Tensor& t) {
  const auto sizes = t.sizes(), strides = t.strides();
  bool done[8] = {};
  int64_t extent = 1;
  for (;;) {
    int next = -1;
    for (int i = 0; i < static_cast<int>(sizes.size()); ++i)
      if (!done[i] && sizes[i] > 1 && (next < 0 || strides[i] < strides[next])) next = i;
    if (next < 0) return true;
    if (strides[next] < extent) return false;
    extent += strides[next] * (sizes[next] - 1);
    done[next] = true;
  }
}

// [tokens, heads, D] as the kernels read it (unit innermost stride; with `wide` 16-byte aligned heads), copied where it is not.
at::Tensor as_heads(const at::Tensor& t, bool wide) {
  if (t.numel() == 0) return t;
  const bool fits = (t.size(2) == 1 || t.stride(2) == 1) &&
                    (!wide || (at16(t) && stride_of(t, 0) % 8 == 0 && stride_of(t, 1) % 8 == 0));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);  // (contiguous() returns contiguous heads at an odd address as they are)
}

qf_kv4_cache check_cache(const char* op, const CacheArgs& c, const at::Device& dev, bool written_to) {
  const std::array<std::pair<const char*, const at::Tensor*>, 4> all = {{{"cache.k", &c.k}, {"cache.v", &c.v},
                                                                         {"cache.k_scale", &c.k_scale},
                                                                         {"cache.v_scale", &c.v_scale}}};
  for (const auto& [name, t] : all) check_input(op, name, *t, dev);
  const int64_t G = c.k.size(3) * 2 / QF_KV4_GROUP;
  QF_REFUSE_UNLESS(c.k.size(1) >= 1 && c.k.size(2) >= 1, op, ": the cache needs a head and a slot, cache.k is ", c.k.sizes());
  for (int i = 0; i < 4; ++i)
    QF_REFUSE_UNLESS(c.k.size(i) <= INT32_MAX, op, ": cache.k is too large: ", c.k.sizes());
  for (int i = 0; i < 3; ++i) {
    QF_REFUSE_UNLESS(stride_of(c.k, i) == stride_of(c.v, i) && stride_of(c.k_scale, i) == stride_of(c.v_scale, i), op,
                     ": cache.k and cache.v, and their scales, must have the same strides");
    QF_REFUSE_UNLESS(stride_of(c.k, i) % 16 == 0 && stride_of(c.k_scale, i) % (2 * G) == 0, op,
                     ": a cache's strides must be multiples of 16 bytes, its scales' of ", 2 * G, " elements");
  }
  for (int i : {0, 2})
    QF_REFUSE_UNLESS(stride_of(c.k, i) <= UINT32_MAX && stride_of(c.k_scale, i) <= UINT32_MAX / 2, op,
                     ": a cache's pages and slots must lie less than 2^32 bytes apart");
  for (const auto& [name, t] : all) {
    const bool scale = t->dim() == 5;
    QF_REFUSE_UNLESS(t->numel() == 0 || (scale ? t->stride(4) == 1 && (G == 1 || t->stride(3) == 2) : t->stride(3) == 1), op,
                     ": ", name, " must have its last dimension", scale ? "s" : "", " adjacent");
    QF_REFUSE_UNLESS(reinterpret_cast<uintptr_t>(t->data_ptr()) % (scale ? 4 * G : 16) == 0, op, ": ", name,
                     " must be aligned to ", scale ? 4 * G : 16, " bytes");
    if (written_to) QF_REFUSE_UNLESS(distinct(*t), op, ": elements of ", name, " refer to a single memory location");
  }
  if (written_to)
    for (size_t i = 0; i < all.size(); ++i)
      for (size_t j = 0; j < i; ++j)
        if (meet(extent_of(*all[i].second), extent_of(*all[j].second)))
          check_no_overlap(op, all[i].first, *all[i].second, all[j].first, *all[j].second);
  qf_kv4_cache r = {};
  r.k = c.k.data_ptr(), r.v = c.v.data_ptr();
  r.k_scale = c.k_scale.data_ptr(), r.v_scale = c.v_scale.data_ptr();
  r.page_stride = stride_of(c.k, 0), r.head_stride = stride_of(c.k, 1), r.slot_stride = stride_of(c.k, 2);
  r.scale_page_stride = stride_of(c.k_scale, 0), r.scale_head_stride = stride_of(c.k_scale, 1);
  r.scale_slot_stride = stride_of(c.k_scale, 2);
  r.num_pages = static_cast<int>(c.k.size(0)), r.num_heads = static_cast<int>(c.k.size(1));
  r.page_size = static_cast<int>(c.k.size(2)), r.head_size = static_cast<int>(c.k.size(3) * 2);
  return r;
}

// Nothing that a call reads lies in a cache that it writes, nor the other way round.
struct CacheExtents {
  const CacheArgs& c;
  Extent e[4];
  explicit CacheExtents(const CacheArgs& args) : c(args), e{extent_of(c.k), extent_of(c.v), extent_of(c.k_scale),
                                                             extent_of(c.v_scale)} {}
  void apart(const char* op, const char* name, const at::Tensor& t) const {
    static const char* const names[] = {"cache.k", "cache.v", "cache.k_scale", "cache.v_scale"};
    const Extent x = extent_of(t);
    for (int i = 0; i < 4; ++i)
      if (C10_UNLIKELY(meet(e[i], x))) check_no_overlap(op, names[i], c[i], name, t);
  }
};

void cache_written(const CacheArgs& c) {
  for (const at::Tensor* t : {&c.k, &c.v, &c.k_scale, &c.v_scale}) written(*t);
}

void check_pieces(const char* op, int64_t tokens, int64_t heads, int64_t d) {
  QF_REFUSE_UNLESS(tokens <= INT32_MAX && tokens * heads <= INT32_MAX / (d / 4), op, ": ", tokens, " tokens of ", heads,
                   " heads are too many for one call");
}

// ---- the cache's writer and reader ----
void kv4_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots, at::Tensor ck, at::Tensor cv,
               at::Tensor cks, at::Tensor cvs) {
  const char* op = "kv4_write";
  const CacheArgs c = {ck, cv, cks, cvs};
  check_write_shapes(op, k, v, slots, c);
  check_input(op, "k", k, k.device());
  check_input(op, "v", v, k.device());
  check_input(op, "slots", slots, k.device());
  const qf_kv4_cache cache = check_cache(op, c, k.device(), true);
  check_pieces(op, k.size(0), k.size(1), k.size(2));
  const CacheExtents extents(c);
  extents.apart(op, "k", k);
  extents.apart(op, "v", v);
  extents.apart(op, "slots", slots);
  if (k.size(0) == 0) return;
  c10::cuda::CUDAGuard guard(k.device());
  const at::Tensor k3 = as_heads(k, true), v3 = as_heads(v, true), s = slots.contiguous();
  check(qf_kv4_write(k3.data_ptr(), stride_of(k3, 0), stride_of(k3, 1), v3.data_ptr(), stride_of(v3, 0), stride_of(v3, 1),
                     s.data_ptr<int64_t>(), static_cast<int>(k.size(0)), &cache, QF_FLAG_PDL, stream_of(k)),
        "qf_kv4_write");
  cache_written(c);
}

std::tuple<at::Tensor, at::Tensor> kv4_read(const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& cks,
                                            const at::Tensor& cvs, const at::Tensor& slots) {
  const char* op = "kv4_read";
  const CacheArgs c = {ck, cv, cks, cvs};
  check_cache_shapes(op, c);
  check_dims(op, "slots", slots, at::kLong, 1);
  check_input(op, "slots", slots, slots.device());
  const qf_kv4_cache cache = check_cache(op, c, slots.device(), false);
  const int64_t T = slots.size(0), H = ck.size(1), D = cache.head_size;
  check_pieces(op, T, H, D);
  c10::cuda::CUDAGuard guard(slots.device());
  at::Tensor k = empty_on(slots, {T, H, D}, at::kBFloat16), v = empty_on(slots, {T, H, D}, at::kBFloat16);
  if (T) {
    const at::Tensor s = slots.contiguous();
    check(qf_kv4_read(k.data_ptr(), H * D, D, v.data_ptr(), H * D, D, s.data_ptr<int64_t>(), static_cast<int>(T), &cache,
                      QF_FLAG_PDL, stream_of(slots)),
          "qf_kv4_read");
  }
  return {k, v};
}

// ---- attention ----
void run_attention(const char* op, const at::Tensor& query, const CacheArgs& c, const qf_kv4_cache& cache,
                   const at::Tensor& seq_lens, const at::Tensor& block_table, int64_t q_len, double scale, at::Tensor& out) {
  const int64_t B = seq_lens.size(0), H = query.size(1);
  if (B == 0 || H == 0) return;
  const at::Tensor q = as_heads(query, true), lens = seq_lens.contiguous();
  const at::Tensor table = block_table.size(1) > 1 && block_table.stride(1) != 1 ? block_table.contiguous() : block_table;
  const size_t bytes = qf_kv4_attn_workspace_bytes(static_cast<int>(B), static_cast<int>(q_len), static_cast<int>(H),
                                                   cache.num_heads, cache.head_size);
  const at::Tensor ws = empty_on(query, {static_cast<int64_t>(bytes)}, at::kByte);
  check(qf_kv4_attn(q.data_ptr(), stride_of(q, 0), stride_of(q, 1), &cache, table.data_ptr<int32_t>(), stride_of(table, 0),
                    static_cast<int>(table.size(1)), lens.data_ptr<int32_t>(), out.data_ptr(), stride_of(out, 0),
                    stride_of(out, 1), static_cast<int>(B), static_cast<int>(q_len), static_cast<int>(H),
                    static_cast<float>(scale), ws.data_ptr(), bytes, QF_FLAG_PDL, stream_of(query)),
        "qf_kv4_attn");
}

qf_kv4_cache check_attention(const char* op, const at::Tensor& query, const CacheArgs& c, const at::Tensor& seq_lens,
                             const at::Tensor& block_table, int64_t q_len, double scale) {
  check_attention_shapes(op, query, c, seq_lens, block_table, q_len, scale);
  check_input(op, "query", query, query.device());
  check_input(op, "seq_lens", seq_lens, query.device());
  check_input(op, "block_table", block_table, query.device());
  QF_REFUSE_UNLESS(query.size(0) <= INT32_MAX / 64 && query.size(1) <= 65535 && block_table.size(1) <= INT32_MAX, op,
                   ": too many query rows or pages for one call");
  const qf_kv4_cache cache = check_cache(op, c, query.device(), false);
  const int64_t tiles = block_table.size(1) * cache.page_size / 64 + 4;  // of a request and head
  QF_REFUSE_UNLESS(tiles <= INT32_MAX && seq_lens.size(0) * cache.num_heads <= INT32_MAX / tiles, op, ": ",
                   seq_lens.size(0), " requests of up to ", block_table.size(1) * cache.page_size, " keys in ",
                   cache.num_heads, " heads are too many for one call");
  return cache;
}

at::Tensor kv4_attention(const at::Tensor& query, const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& cks,
                         const at::Tensor& cvs, const at::Tensor& seq_lens, const at::Tensor& block_table, int64_t q_len,
                         double scale) {
  const CacheArgs c = {ck, cv, cks, cvs};
  const qf_kv4_cache cache = check_attention("kv4_attention", query, c, seq_lens, block_table, q_len, scale);
  c10::cuda::CUDAGuard guard(query.device());
  at::Tensor out = empty_on(query, {seq_lens.size(0) * q_len, query.size(1), query.size(2)}, at::kBFloat16);
  run_attention("kv4_attention", query, c, cache, seq_lens, block_table, q_len, scale, out);
  return out;
}

void check_out_shape(const char* op, const at::Tensor& out, const at::Tensor& query) {
  check_dims(op, "out", out, at::kBFloat16, 3);
  for (int i = 0; i < 3; ++i)
    QF_REFUSE_UNLESS_EQ(out.sym_size(i), query.sym_size(i), op, ": out must have the query's shape ", query.sym_sizes(),
                        ", got ", out.sym_sizes());
}

void kv4_attention_out(const at::Tensor& query, const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& cks,
                       const at::Tensor& cvs, const at::Tensor& seq_lens, const at::Tensor& block_table, int64_t q_len,
                       double scale, at::Tensor out) {
  const char* op = "kv4_attention";
  const CacheArgs c = {ck, cv, cks, cvs};
  const qf_kv4_cache cache = check_attention(op, query, c, seq_lens, block_table, q_len, scale);
  check_out_shape(op, out, query);
  check_input(op, "out", out, query.device());
  QF_REFUSE_UNLESS(out.numel() == 0 || (out.stride(2) == 1 && at16(out) && stride_of(out, 0) % 8 == 0 &&
                                        stride_of(out, 1) % 8 == 0 && distinct(out)),
                   op, ": out must have unit stride within a head, 16-byte aligned heads and no two elements at one place");
  check_no_overlap(op, "out", out, "query", query);
  CacheExtents(c).apart(op, "out", out);
  check_no_overlap(op, "out", out, "seq_lens", seq_lens);
  check_no_overlap(op, "out", out, "block_table", block_table);
  c10::cuda::CUDAGuard guard(query.device());
  run_attention(op, query, c, cache, seq_lens, block_table, q_len, scale, out);
  written(out);
}

// ---- norms of queries and keys with the rotation ----
struct RopeRun {
  const at::Tensor &q, &k;
  const OptTensor &q_weight, &k_weight, &positions, &cos_sin;
  double offset, eps;
  bool interleaved;
};

void check_rope(const char* op, const RopeRun& r) {
  check_rope_shapes(op, r.q, r.k, r.q_weight, r.k_weight, r.positions, r.cos_sin, r.eps);
  const at::Device dev = r.q.device();
  check_input(op, "q", r.q, dev);
  check_input(op, "k", r.k, dev);
  for (const auto& [name, t] : {std::make_pair("q_weight", &r.q_weight), std::make_pair("k_weight", &r.k_weight),
                                std::make_pair("positions", &r.positions), std::make_pair("cos_sin", &r.cos_sin)})
    if (given(*t)) check_input(op, name, **t, dev);
  QF_REFUSE_UNLESS(r.q.size(2) >= 1 && r.q.size(2) <= QF_ROPE_MAX_D, op, ": heads of 1 to ", QF_ROPE_MAX_D, " values, got ",
                   r.q.size(2));
  QF_REFUSE_UNLESS(r.q.size(0) <= INT32_MAX && r.q.size(1) <= INT32_MAX / 4 && r.k.size(1) <= INT32_MAX / 4 &&
                       (r.q.size(1) + 2 * r.k.size(1)) * r.q.size(0) <= INT32_MAX,
                   op, ": too many rows for one call");
}

void run_rope(const RopeRun& r, at::Tensor& q_out, at::Tensor* k_out, const at::Tensor* v, const at::Tensor* slots,
              const qf_kv4_cache* cache) {
  const int64_t T = r.q.size(0), H = r.q.size(1), HKV = r.k.size(1), D = r.q.size(2);
  if (T == 0 || H + HKV == 0) return;
  const at::Tensor q = as_heads(r.q, false), k = as_heads(r.k, false);
  at::Tensor qw, kw, pos, table, v3, s;
  if (given(r.q_weight)) qw = r.q_weight->contiguous();
  if (given(r.k_weight)) kw = r.k_weight->contiguous();
  int64_t rot = 0, max_pos = 0, row = 0;
  int type = QF_DTYPE_F32;
  if (given(r.cos_sin)) {
    pos = r.positions->contiguous();
    rot = r.cos_sin->size(1), max_pos = r.cos_sin->size(0);
    table = rot > 1 && r.cos_sin->stride(1) != 1 ? r.cos_sin->contiguous() : *r.cos_sin;
    row = max_pos > 1 ? table.stride(0) : 0;
    type = table.scalar_type() == at::kFloat ? QF_DTYPE_F32 : QF_DTYPE_BF16;
  }
  if (v) v3 = as_heads(*v, false), s = slots->contiguous();
  auto ptr = [](const at::Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; };
  check(qf_qk_norm_rope(ptr(q), stride_of(q, 0), stride_of(q, 1), ptr(k), stride_of(k, 0), stride_of(k, 1), ptr(qw), ptr(kw),
                        static_cast<float>(r.offset), static_cast<float>(r.eps), static_cast<const int64_t*>(ptr(pos)),
                        ptr(table), row, type, max_pos, static_cast<int>(rot), r.interleaved, ptr(q_out), H * D, D,
                        k_out ? ptr(*k_out) : nullptr, HKV * D, D, ptr(v3), v ? stride_of(v3, 0) : 0,
                        v ? stride_of(v3, 1) : 0, static_cast<const int64_t*>(ptr(s)), cache, static_cast<int>(T),
                        static_cast<int>(H), static_cast<int>(HKV), static_cast<int>(D), QF_FLAG_PDL, stream_of(q)),
        "qf_qk_norm_rope");
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& q, const at::Tensor& k, const OptTensor& q_weight,
                                                const OptTensor& k_weight, const OptTensor& positions,
                                                const OptTensor& cos_sin, double weight_offset, double eps,
                                                bool interleaved) {
  const RopeRun r = {q, k, q_weight, k_weight, positions, cos_sin, weight_offset, eps, interleaved};
  check_rope("qk_norm_rope", r);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor q_out = empty_on(q, q.sizes(), at::kBFloat16), k_out = empty_on(k, k.sizes(), at::kBFloat16);
  run_rope(r, q_out, &k_out, nullptr, nullptr, nullptr);
  return {q_out, k_out};
}

at::Tensor qk_norm_rope_kv4(const at::Tensor& q, const at::Tensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                            const OptTensor& positions, const OptTensor& cos_sin, double weight_offset, double eps,
                            bool interleaved, const at::Tensor& v, const at::Tensor& slots, at::Tensor ck, at::Tensor cv,
                            at::Tensor cks, at::Tensor cvs) {
  const char* op = "qk_norm_rope";
  const CacheArgs c = {ck, cv, cks, cvs};
  const RopeRun r = {q, k, q_weight, k_weight, positions, cos_sin, weight_offset, eps, interleaved};
  check_write_shapes(op, k, v, slots, c);
  check_rope(op, r);
  check_input(op, "v", v, q.device());
  check_input(op, "slots", slots, q.device());
  const qf_kv4_cache cache = check_cache(op, c, q.device(), true);
  const CacheExtents extents(c);
  for (const auto& [name, t] : {std::make_pair("q", &q), std::make_pair("k", &k), std::make_pair("v", &v),
                                std::make_pair("slots", &slots)})
    extents.apart(op, name, *t);
  for (const auto& [name, t] : {std::make_pair("q_weight", &q_weight), std::make_pair("k_weight", &k_weight),
                                std::make_pair("positions", &positions), std::make_pair("cos_sin", &cos_sin)})
    if (given(*t)) extents.apart(op, name, **t);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor q_out = empty_on(q, q.sizes(), at::kBFloat16);
  run_rope(r, q_out, nullptr, &v, &slots, &cache);
  cache_written(c);
  return q_out;
}

// ---- the maps of a step ----
// `n` elements of a buffer as a tensor of their own.  (Results that share a buffer share none of its elements.)
at::Tensor piece_of(const at::Tensor& buffer, int64_t offset, int64_t n) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), buffer.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

using Maps = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

void check_maps(const char* op, const at::Tensor& query_lens, const at::Tensor& past_lens, const at::Tensor& block_table,
                int64_t page_size, int64_t num_tokens) {
  check_maps_shapes(op, query_lens, past_lens, block_table, page_size, num_tokens);
  check_input(op, "query_lens", query_lens, query_lens.device());
  check_input(op, "past_lens", past_lens, query_lens.device());
  check_input(op, "block_table", block_table, query_lens.device());
  QF_REFUSE_UNLESS(query_lens.size(0) <= QF_MAPS_MAX_REQS, op, ": at most ", QF_MAPS_MAX_REQS, " requests, got ",
                   query_lens.size(0));
  QF_REFUSE_UNLESS(block_table.size(1) <= INT32_MAX, op, ": block_table is too wide: ", block_table.sizes());
}

Maps run_maps(const at::Tensor& query_lens, const at::Tensor& past_lens, const at::Tensor& table, int64_t page_size,
              int64_t num_tokens, const at::Tensor* free_pages, const at::Tensor* free_head, at::Tensor* head_out) {
  const int64_t B = query_lens.size(0);
  c10::cuda::CUDAGuard guard(query_lens.device());
  const at::Tensor q = query_lens.contiguous(), past = past_lens.contiguous();
  // an allocation for each type (64 32-bit numbers are 256 bytes: every result is aligned as one of its own)
  const int64_t row = (B + 1 + 63) / 64 * 64, col = (num_tokens + 31) / 32 * 32;
  const at::Tensor ints = empty_on(q, {2 * row + 1}, at::kInt), longs = empty_on(q, {2 * col}, at::kLong);
  at::Tensor start = piece_of(ints, 0, B + 1), seq = piece_of(ints, row, B);
  at::Tensor pos = piece_of(longs, 0, num_tokens), slots = piece_of(longs, col, num_tokens);
  at::Tensor free;
  if (free_pages) {
    free = free_pages->contiguous();
    *head_out = piece_of(ints, 2 * row, 1);
  }
  check(qf_step_maps(q.data_ptr<int32_t>(), past.data_ptr<int32_t>(), static_cast<int>(B), table.data_ptr<int32_t>(),
                     B > 1 ? table.stride(0) : table.size(1), static_cast<int>(table.size(1)), static_cast<int>(page_size),
                     free.defined() && free.numel() ? free.data_ptr<int32_t>() : nullptr,
                     free.defined() ? static_cast<int>(free.numel()) : 0,
                     free_head ? free_head->data_ptr<int32_t>() : nullptr, start.data_ptr<int32_t>(),
                     seq.data_ptr<int32_t>(), pos.data_ptr<int64_t>(), slots.data_ptr<int64_t>(),
                     static_cast<int>(num_tokens), head_out ? head_out->data_ptr<int32_t>() : nullptr, QF_FLAG_PDL,
                     stream_of(q)),
        "qf_step_maps");
  return {start, seq, pos, slots};
}

Maps step_maps(const at::Tensor& query_lens, const at::Tensor& past_lens, const at::Tensor& block_table, int64_t page_size,
               int64_t num_tokens) {
  check_maps("step_maps", query_lens, past_lens, block_table, page_size, num_tokens);
  const int64_t B = block_table.size(0), W = block_table.size(1);
  const bool rows = (W <= 1 || block_table.stride(1) == 1) && (B <= 1 || block_table.stride(0) >= W);
  return run_maps(query_lens, past_lens, rows ? block_table : block_table.contiguous(), page_size, num_tokens, nullptr,
                  nullptr, nullptr);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> step_maps_grow(
    const at::Tensor& query_lens, const at::Tensor& past_lens, at::Tensor block_table, int64_t page_size, int64_t num_tokens,
    const at::Tensor& free_pages, const at::Tensor& free_head) {
  const char* op = "step_maps";
  check_maps(op, query_lens, past_lens, block_table, page_size, num_tokens);
  check_free_shapes(op, free_pages, free_head);
  check_input(op, "free_pages", free_pages, query_lens.device());
  check_input(op, "free_head", free_head, query_lens.device());
  const int64_t B = block_table.size(0), W = block_table.size(1);
  QF_REFUSE_UNLESS((W <= 1 || block_table.stride(1) == 1) && (B <= 1 || block_table.stride(0) >= W), op,
                   ": a block_table that grows must have rows of adjacent entries that do not overlap");
  QF_REFUSE_UNLESS(free_pages.size(0) <= INT32_MAX, op, ": too many free pages");
  const Extent table = extent_of(block_table);
  for (const auto& [name, t] : {std::make_pair("query_lens", &query_lens), std::make_pair("past_lens", &past_lens),
                                std::make_pair("free_pages", &free_pages), std::make_pair("free_head", &free_head)})
    if (C10_UNLIKELY(meet(table, extent_of(*t)))) check_no_overlap(op, "block_table", block_table, name, *t);
  at::Tensor head;
  auto [start, seq, pos, slots] =
      run_maps(query_lens, past_lens, block_table, page_size, num_tokens, &free_pages, &free_head, &head);
  written(block_table);
  return {start, seq, pos, slots, head};
}

// ---- types and shapes only, for tracing ----
at::Tensor meta(const at::Tensor& like, std::vector<c10::SymInt> sizes, at::ScalarType type) {
  return at::empty_symint(sizes, like.options().dtype(type));
}
void kv4_write_meta(const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots, at::Tensor ck, at::Tensor cv,
                    at::Tensor cks, at::Tensor cvs) {
  const CacheArgs c = {ck, cv, cks, cvs};
  check_write_shapes("kv4_write", k, v, slots, c);
  cache_written(c);
}
std::tuple<at::Tensor, at::Tensor> kv4_read_meta(const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& cks,
                                                 const at::Tensor& cvs, const at::Tensor& slots) {
  const CacheArgs c = {ck, cv, cks, cvs};
  check_cache_shapes("kv4_read", c);
  check_dims("kv4_read", "slots", slots, at::kLong, 1);
  const std::vector<c10::SymInt> s = {slots.sym_size(0), c.heads(), c.head_size()};
  return {meta(slots, s, at::kBFloat16), meta(slots, s, at::kBFloat16)};
}
at::Tensor kv4_attention_meta(const at::Tensor& query, const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& cks,
                              const at::Tensor& cvs, const at::Tensor& seq_lens, const at::Tensor& block_table,
                              int64_t q_len, double scale) {
  check_attention_shapes("kv4_attention", query, {ck, cv, cks, cvs}, seq_lens, block_table, q_len, scale);
  return meta(query, {seq_lens.sym_size(0) * q_len, query.sym_size(1), query.sym_size(2)}, at::kBFloat16);
}
void kv4_attention_out_meta(const at::Tensor& query, const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& cks,
                            const at::Tensor& cvs, const at::Tensor& seq_lens, const at::Tensor& block_table, int64_t q_len,
                            double scale, at::Tensor out) {
  check_attention_shapes("kv4_attention", query, {ck, cv, cks, cvs}, seq_lens, block_table, q_len, scale);
  check_out_shape("kv4_attention", out, query);
  written(out);
}
std::tuple<at::Tensor, at::Tensor> qk_norm_rope_meta(const at::Tensor& q, const at::Tensor& k, const OptTensor& q_weight,
                                                     const OptTensor& k_weight, const OptTensor& positions,
                                                     const OptTensor& cos_sin, double, double eps, bool) {
  check_rope_shapes("qk_norm_rope", q, k, q_weight, k_weight, positions, cos_sin, eps);
  return {meta(q, q.sym_sizes().vec(), at::kBFloat16), meta(k, k.sym_sizes().vec(), at::kBFloat16)};
}
at::Tensor qk_norm_rope_kv4_meta(const at::Tensor& q, const at::Tensor& k, const OptTensor& q_weight,
                                 const OptTensor& k_weight, const OptTensor& positions, const OptTensor& cos_sin, double,
                                 double eps, bool, const at::Tensor& v, const at::Tensor& slots, at::Tensor ck, at::Tensor cv,
                                 at::Tensor cks, at::Tensor cvs) {
  const CacheArgs c = {ck, cv, cks, cvs};
  check_write_shapes("qk_norm_rope", k, v, slots, c);
  check_rope_shapes("qk_norm_rope", q, k, q_weight, k_weight, positions, cos_sin, eps);
  cache_written(c);
  return meta(q, q.sym_sizes().vec(), at::kBFloat16);
}
Maps step_maps_meta(const at::Tensor& query_lens, const at::Tensor& past_lens, const at::Tensor& block_table,
                    int64_t page_size, int64_t num_tokens) {
  check_maps_shapes("step_maps", query_lens, past_lens, block_table, page_size, num_tokens);
  const c10::SymInt B = query_lens.sym_size(0);
  return {meta(query_lens, {B + 1}, at::kInt), meta(query_lens, {B}, at::kInt), meta(query_lens, {num_tokens}, at::kLong),
          meta(query_lens, {num_tokens}, at::kLong)};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> step_maps_grow_meta(
    const at::Tensor& query_lens, const at::Tensor& past_lens, at::Tensor block_table, int64_t page_size, int64_t num_tokens,
    const at::Tensor& free_pages, const at::Tensor& free_head) {
  auto [start, seq, pos, slots] = step_maps_meta(query_lens, past_lens, block_table, page_size, num_tokens);
  check_free_shapes("step_maps", free_pages, free_head);
  written(block_table);
  return {start, seq, pos, slots, meta(query_lens, {1}, at::kInt)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(qf_b200, m) {
  m.def("step_maps(Tensor query_lens, Tensor past_lens, Tensor block_table, int page_size, int num_tokens) -> "
        "(Tensor, Tensor, Tensor, Tensor)");
  m.def("step_maps_grow(Tensor query_lens, Tensor past_lens, Tensor(a!) block_table, int page_size, int num_tokens, "
        "Tensor free_pages, Tensor free_head) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? positions, Tensor? cos_sin, "
        "float weight_offset, float eps, bool interleaved) -> (Tensor, Tensor)");
  m.def("qk_norm_rope_kv4(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? positions, Tensor? cos_sin, "
        "float weight_offset, float eps, bool interleaved, Tensor v, Tensor slots, Tensor(a!) cache_k, Tensor(b!) cache_v, "
        "Tensor(c!) cache_k_scale, Tensor(d!) cache_v_scale) -> Tensor");
  m.def("kv4_write(Tensor k, Tensor v, Tensor slots, Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor(c!) cache_k_scale, "
        "Tensor(d!) cache_v_scale) -> ()");
  m.def("kv4_read(Tensor cache_k, Tensor cache_v, Tensor cache_k_scale, Tensor cache_v_scale, Tensor slots) -> "
        "(Tensor, Tensor)");
  m.def("kv4_attention(Tensor query, Tensor cache_k, Tensor cache_v, Tensor cache_k_scale, Tensor cache_v_scale, "
        "Tensor seq_lens, Tensor block_table, int q_len, float scale) -> Tensor");
  m.def("kv4_attention_out(Tensor query, Tensor cache_k, Tensor cache_v, Tensor cache_k_scale, Tensor cache_v_scale, "
        "Tensor seq_lens, Tensor block_table, int q_len, float scale, Tensor(a!) out) -> ()");
}
// CompositeExplicitAutograd: CPU tensors reach the operators' own refusals instead of the dispatcher's.
TORCH_LIBRARY_IMPL(qf_b200, CompositeExplicitAutograd, m) {
  m.impl("step_maps", step_maps);
  m.impl("step_maps_grow", step_maps_grow);
  m.impl("qk_norm_rope", qk_norm_rope);
  m.impl("qk_norm_rope_kv4", qk_norm_rope_kv4);
  m.impl("kv4_write", kv4_write);
  m.impl("kv4_read", kv4_read);
  m.impl("kv4_attention", kv4_attention);
  m.impl("kv4_attention_out", kv4_attention_out);
}
TORCH_LIBRARY_IMPL(qf_b200, Autograd, m) {
  for (const char* op : {"step_maps", "step_maps_grow", "qk_norm_rope", "qk_norm_rope_kv4", "kv4_write", "kv4_read",
                         "kv4_attention", "kv4_attention_out"})
    m.impl(op, torch::CppFunction::makeFromBoxedFunction<&refuse_derivatives>());
}
TORCH_LIBRARY_IMPL(qf_b200, Meta, m) {
  m.impl("step_maps", step_maps_meta);
  m.impl("step_maps_grow", step_maps_grow_meta);
  m.impl("qk_norm_rope", qk_norm_rope_meta);
  m.impl("qk_norm_rope_kv4", qk_norm_rope_kv4_meta);
  m.impl("kv4_write", kv4_write_meta);
  m.impl("kv4_read", kv4_read_meta);
  m.impl("kv4_attention", kv4_attention_meta);
  m.impl("kv4_attention_out", kv4_attention_out_meta);
}
