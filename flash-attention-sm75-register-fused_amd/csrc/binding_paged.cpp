// PyTorch binding of the paged key/value cache (no reference counterpart):
// paged_cache_write, paged_cache_read, paged_cache_evict, flash_attention_paged,
// flash_attention_paged_prefix and paged_attention_weights.
//
// All checks run before any device work; the kernels are enqueued on the
// current HIP stream of the cache's device and the host is not blocked.
#include <torch/extension.h>

#include <ATen/DeviceGuard.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>

#include <initializer_list>
#include <tuple>
#include <utility>

#include "flash_attn_sm75.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

bool is_half_type(const Tensor& t) {
  return t.scalar_type() == torch::kFloat16 || t.scalar_type() == torch::kBFloat16;
}

int dtype_code(torch::ScalarType t) {
  return t == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_FP16;
}

// Stride of dimension i, or `fallback` where the dimension holds one entry (its
// stride then says nothing).
int64_t eff_stride(const Tensor& t, int i, int64_t fallback) {
  return t.size(i) == 1 ? fallback : t.stride(i);
}

void check_index(const Tensor& t, const char* name, int64_t dim, const Tensor& k_cache) {
  TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be int32");
  TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimension(s)");
  TORCH_CHECK(t.device() == k_cache.device(), name, " must be on the cache's device");
}

// The cache's description, checked.  `written`: rows are going to be written,
// which no two of them may share.
fa_paged_cache make_cache(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens,
                          const OptTensor& ks, const OptTensor& vs, bool written) {
  TORCH_CHECK(k.is_cuda() && v.is_cuda(), "the cache must be CUDA tensors");
  TORCH_CHECK(k.device() == v.device(), "k_cache and v_cache must be on the same device");
  TORCH_CHECK(k.dim() == 4 && v.dim() == 4, "k_cache and v_cache must be [pages, H_kv, page_size, D]");
  TORCH_CHECK(k.sizes() == v.sizes(), "k_cache and v_cache must have identical shapes");
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), "k_cache and v_cache must have the same dtype");
  const bool q8 = k.scalar_type() == torch::kFloat8_e4m3fn;
  TORCH_CHECK(q8 || is_half_type(k), "the cache must be FP16, BF16 or float8_e4m3fn");
  TORCH_CHECK(ks.has_value() == q8 && vs.has_value() == q8,
              q8 ? "a float8_e4m3fn cache needs k_scale and v_scale"
                 : "k_scale and v_scale go with a float8_e4m3fn cache");
  for (const Tensor* t : {&k, &v}) {
    TORCH_CHECK(t->stride(3) == 1 || t->size(3) <= 1, "the cache's head_dim must be contiguous");
    for (int i = 0; written && i < 3; ++i)
      TORCH_CHECK(t->size(i) <= 1 || t->stride(i) != 0, "the cache must not be an expanded view");
  }
  check_index(table, "block_table", 2, k);
  check_index(lens, "seq_lens", 1, k);
  TORCH_CHECK(table.size(0) == lens.size(0), "block_table and seq_lens must have the same batch");
  TORCH_CHECK(table.size(1) <= 1 || table.stride(1) == 1, "block_table's rows must be contiguous");
  TORCH_CHECK(lens.size(0) <= 1 || lens.stride(0) == 1, "seq_lens must be contiguous");
  fa_paged_cache c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.block_table = table.data_ptr<int32_t>();
  c.seq_lens = lens.data_ptr<int32_t>();
  c.batch = table.size(0);
  c.heads_kv = k.size(1);
  c.head_dim = k.size(3);
  c.num_pages = k.size(0);
  c.page_size = k.size(2);
  c.max_pages = table.size(1);
  c.block_table_stride = eff_stride(table, 0, table.size(1));
  const int64_t d = c.head_dim;
  c.k_stride_p = eff_stride(k, 0, 0); c.k_stride_h = eff_stride(k, 1, 0); c.k_stride_n = eff_stride(k, 2, d);
  c.v_stride_p = eff_stride(v, 0, 0); c.v_stride_h = eff_stride(v, 1, 0); c.v_stride_n = eff_stride(v, 2, d);
  if (q8) {
    for (const Tensor* t : {&*ks, &*vs}) {
      TORCH_CHECK(t->scalar_type() == torch::kFloat8_e8m0fnu, "k_scale and v_scale must be float8_e8m0fnu");
      TORCH_CHECK(t->device() == k.device(), "k_scale and v_scale must be on the cache's device");
      TORCH_CHECK(t->dim() == 3 && t->size(0) == k.size(0) && t->size(1) == k.size(1) &&
                      t->size(2) == k.size(2),
                  "k_scale and v_scale must be [pages, H_kv, page_size]");
      for (int i = 0; written && i < 3; ++i)
        TORCH_CHECK(t->size(i) <= 1 || t->stride(i) != 0, "the scales must not be an expanded view");
    }
    c.k_scale = static_cast<uint8_t*>(ks->data_ptr());
    c.v_scale = static_cast<uint8_t*>(vs->data_ptr());
    c.ks_stride_p = eff_stride(*ks, 0, 0); c.ks_stride_h = eff_stride(*ks, 1, 0);
    c.ks_stride_n = eff_stride(*ks, 2, 1);
    c.vs_stride_p = eff_stride(*vs, 0, 0); c.vs_stride_h = eff_stride(*vs, 1, 0);
    c.vs_stride_n = eff_stride(*vs, 2, 1);
  }
  return c;
}

// [tokens, heads, D] rows the kernels can read in place, else a copy.
Tensor rows_view(const Tensor& t) {
  const bool ok = t.stride(2) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0 &&
                  (t.size(0) <= 1 || (t.stride(0) >= 0 && t.stride(0) % 8 == 0)) &&
                  (t.size(1) <= 1 || (t.stride(1) >= 0 && t.stride(1) % 8 == 0));
  return ok ? t : t.contiguous();
}

// Whether no byte from a's first element to its last lies between b's (strides not
// negative).
bool spans_apart(const Tensor& a, const Tensor& b) {
  auto span = [](const Tensor& t) {
    int64_t last = 0;
    for (int i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    const auto first = reinterpret_cast<uintptr_t>(t.data_ptr());
    return std::pair<uintptr_t, uintptr_t>(first, first + (last + 1) * t.element_size());
  };
  if (a.numel() == 0 || b.numel() == 0) return true;
  const auto x = span(a), y = span(b);
  return x.second <= y.first || y.second <= x.first;
}

// Whether [tokens, heads, D] rows of one shape and type, a's and b's, share no memory: they
// lie apart, or interleave in a buffer that holds both, in every token's stretch of it or in
// every head's.  (False where neither can be seen from the strides.)
bool rows_apart(const Tensor& a, const Tensor& b) {
  if (spans_apart(a, b)) return true;
  const int64_t d = a.size(2), st = a.stride(0), sh = a.size(1) == 1 ? d : a.stride(1);
  const bool one = a.size(0) == 1;
  if (!one && (st <= 0 || st != b.stride(0))) return false;
  if (sh < d || (a.size(1) > 1 && sh != b.stride(1))) return false;
  const int64_t bytes = reinterpret_cast<intptr_t>(b.data_ptr()) - reinterpret_cast<intptr_t>(a.data_ptr());
  if (bytes % a.element_size() != 0) return false;
  const int64_t delta = bytes / a.element_size();
  // `width` elements of every `period`, b's delta behind a's.
  auto apart = [delta](int64_t period, int64_t width) {
    const int64_t r = (delta % period + period) % period;
    return r >= width && r + width <= period;
  };
  return (!one && apart(st, (a.size(1) - 1) * sh + d)) || ((one || st % sh == 0) && apart(sh, d));
}

const int32_t* cu_pointer(const OptTensor& cu, const Tensor& k_cache, int64_t batch, int64_t tokens) {
  if (!cu.has_value()) {
    TORCH_CHECK(tokens == batch, "without cu_seqlens there is one new token for each of the ", batch,
                " sequences, got ", tokens);
    return nullptr;
  }
  check_index(*cu, "cu_seqlens", 1, k_cache);
  TORCH_CHECK(cu->size(0) == batch + 1, "cu_seqlens must have batch + 1 = ", batch + 1, " entries");
  TORCH_CHECK(cu->stride(0) == 1, "cu_seqlens must be contiguous");
  return cu->data_ptr<int32_t>();
}

void* current_stream(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// Refuses tensors that carry a forward-mode tangent, which the call would drop.
void check_no_tangent(const char* name, std::initializer_list<const Tensor*> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t->_fw_grad(0).defined(), name, " has no forward-mode derivative: call it on the primals "
                "(torch.autograd.forward_ad.unpack_dual)");
}

// Tells autograd that a tensor was written to: a graph that kept its old values raises.
// (Tensors of inference mode count no versions and are in no graph.)
void written_to(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void paged_cache_write(Tensor K, Tensor V, Tensor k_cache, Tensor v_cache, Tensor block_table,
                       Tensor seq_lens, OptTensor cu_seqlens, OptTensor k_scale, OptTensor v_scale) {
  check_no_tangent("paged_cache_write", {&K, &V, &k_cache, &v_cache});
  const fa_paged_cache c = make_cache(k_cache, v_cache, block_table, seq_lens, k_scale, v_scale, true);
  for (const Tensor* t : {&K, &V}) {
    TORCH_CHECK(is_half_type(*t), "K and V must be FP16 or BF16");
    TORCH_CHECK(t->device() == k_cache.device(), "K and V must be on the cache's device");
    TORCH_CHECK(t->dim() == 3, "K and V must be [tokens, H_kv, D]");
  }
  TORCH_CHECK(K.sizes() == V.sizes(), "K and V must have identical shapes");
  TORCH_CHECK(K.scalar_type() == V.scalar_type(), "K and V must have the same dtype");
  TORCH_CHECK(c.k_scale != nullptr || K.scalar_type() == k_cache.scalar_type(),
              "K and V must have the cache's dtype");
  TORCH_CHECK(K.size(1) == c.heads_kv && K.size(2) == c.head_dim,
              "K and V must have the cache's heads and head_dim");
  fa_paged_rows r{};
  r.cu_seqlens = cu_pointer(cu_seqlens, k_cache, c.batch, K.size(0));
  const at::OptionalDeviceGuard guard(at::device_of(k_cache));
  if (K.numel() != 0) {
    K = rows_view(K);
    V = rows_view(V);
  }
  r.k = static_cast<const fa_half*>(K.data_ptr());
  r.v = static_cast<const fa_half*>(V.data_ptr());
  r.tokens = K.size(0);
  r.k_stride_t = eff_stride(K, 0, 0); r.k_stride_h = eff_stride(K, 1, 0);
  r.v_stride_t = eff_stride(V, 0, 0); r.v_stride_h = eff_stride(V, 1, 0);
  r.dtype = dtype_code(K.scalar_type());
  r.stream = current_stream(k_cache);
  const int st = fa_sm75_paged_write(&c, &r);
  TORCH_CHECK(st == FA_OK, "paged_cache_write: ", fa_sm75_last_error());
  written_to(k_cache);
  written_to(v_cache);
  if (k_scale.has_value()) {
    written_to(*k_scale);
    written_to(*v_scale);
  }
}

std::tuple<Tensor, Tensor> paged_cache_read(Tensor k_cache, Tensor v_cache, Tensor block_table,
                                            Tensor seq_lens, int64_t max_len, OptTensor k_scale,
                                            OptTensor v_scale, c10::optional<torch::ScalarType> dtype) {
  check_no_tangent("paged_cache_read", {&k_cache, &v_cache});
  const fa_paged_cache c = make_cache(k_cache, v_cache, block_table, seq_lens, k_scale, v_scale, false);
  TORCH_CHECK(max_len >= 0, "max_len must be non-negative, got ", max_len);
  TORCH_CHECK(dtype.has_value() || c.k_scale == nullptr, "a float8_e4m3fn cache needs a dtype to read to");
  const auto to = dtype.has_value() ? *dtype : k_cache.scalar_type();
  TORCH_CHECK(to == torch::kFloat16 || to == torch::kBFloat16, "dtype must be float16 or bfloat16");
  TORCH_CHECK(c.k_scale != nullptr || to == k_cache.scalar_type(),
              "a 16-bit cache is read in its own dtype");
  const at::OptionalDeviceGuard guard(at::device_of(k_cache));
  auto K = torch::empty({c.batch, c.heads_kv, max_len, c.head_dim}, k_cache.options().dtype(to));
  auto V = torch::empty_like(K);
  const int st = fa_sm75_paged_read(&c, static_cast<fa_half*>(K.data_ptr()),
                                    static_cast<fa_half*>(V.data_ptr()), max_len, dtype_code(to),
                                    current_stream(k_cache));
  TORCH_CHECK(st == FA_OK, "paged_cache_read: ", fa_sm75_last_error());
  return {K, V};
}

// Checks the queries of a call over a cache; Q becomes rows that the kernels can read.
void check_queries(Tensor& Q, const fa_paged_cache& c, const Tensor& k_cache) {
  TORCH_CHECK(is_half_type(Q), "Q must be FP16 or BF16");
  TORCH_CHECK(Q.device() == k_cache.device(), "Q must be on the cache's device");
  TORCH_CHECK(Q.dim() == 3, "Q must be [tokens, H_q, D]");
  TORCH_CHECK(c.k_scale != nullptr || Q.scalar_type() == k_cache.scalar_type(),
              "Q must have the cache's dtype");
  TORCH_CHECK(Q.size(2) == c.head_dim, "head_dim mismatch");
  TORCH_CHECK(c.heads_kv > 0 && Q.size(1) % c.heads_kv == 0, "heads mismatch: Q heads (", Q.size(1),
              ") not divisible by K/V heads (", c.heads_kv, ")");
}

// An attention call's parameters, checked, with the tensors they point into.
struct Forward {
  fa_paged_params p{};
  Tensor Q, O;
  OptTensor L;
};
Forward make_forward(const fa_paged_cache& c, Tensor Q, const Tensor& k_cache, const Tensor& v_cache,
                     const OptTensor& cu_seqlens, int64_t max_query_len, int64_t causal, double scale,
                     const OptTensor& k_scale, const OptTensor& v_scale, bool return_lse, const OptTensor& out) {
  check_queries(Q, c, k_cache);
  Forward f;
  fa_paged_params& p = f.p;
  p.cu_seqlens = cu_pointer(cu_seqlens, k_cache, c.batch, Q.size(0));
  if (Q.numel() != 0) Q = rows_view(Q);
  Tensor O;
  if (out.has_value()) {
    O = *out;
    TORCH_CHECK(O.sizes() == Q.sizes() && O.scalar_type() == Q.scalar_type() && O.device() == Q.device(),
                "out must have Q's shape, dtype and device");
    // (other workgroups still read Q when the first rows of O are written)
    for (int i = 0; i < 2; ++i)
      TORCH_CHECK(O.size(i) <= 1 || O.stride(i) != 0, "out must not be an expanded view");
    TORCH_CHECK(O.numel() == 0 || rows_view(O).is_same(O),
                "out must be 16-byte aligned, head_dim contiguous, its other strides multiples of 8");
    bool apart = rows_apart(O, Q) && spans_apart(O, k_cache) && spans_apart(O, v_cache);
    if (k_scale.has_value()) apart = apart && spans_apart(O, *k_scale) && spans_apart(O, *v_scale);
    TORCH_CHECK(apart, "out must not share Q's or the cache's memory");
  } else {
    O = torch::empty(Q.sizes(), Q.options());
  }
  if (return_lse) f.L = torch::empty({Q.size(1), Q.size(0)}, Q.options().dtype(torch::kFloat32));
  p.cache = &c;
  p.q = static_cast<const fa_half*>(Q.data_ptr());
  p.o = static_cast<fa_half*>(O.data_ptr());
  p.lse = return_lse ? f.L->data_ptr<float>() : nullptr;
  p.tokens = Q.size(0);
  p.heads_q = Q.size(1);
  p.q_stride_t = eff_stride(Q, 0, 0); p.q_stride_h = eff_stride(Q, 1, 0);
  p.o_stride_t = eff_stride(O, 0, 0); p.o_stride_h = eff_stride(O, 1, 0);
  p.max_query_len = max_query_len;
  p.scale = (float)scale;
  p.causal = (int)causal;
  p.dtype = dtype_code(Q.scalar_type());
  p.stream = current_stream(k_cache);
  f.Q = Q;
  f.O = O;
  return f;
}

// A workspace of the current stream's (stream-ordered reuse behind the launch).
Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? torch::empty({bytes}, like.options().dtype(torch::kUInt8)) : Tensor();
}

std::tuple<Tensor, OptTensor> flash_attention_paged(
    Tensor Q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor seq_lens,
    OptTensor cu_seqlens, int64_t max_query_len, int64_t causal, double scale, OptTensor k_scale,
    OptTensor v_scale, bool return_lse, OptTensor out) {
  check_no_tangent("flash_attention_paged", {&Q, &k_cache, &v_cache, out.has_value() ? &*out : &Q});
  const fa_paged_cache c = make_cache(k_cache, v_cache, block_table, seq_lens, k_scale, v_scale, false);
  const at::OptionalDeviceGuard guard(at::device_of(k_cache));
  Forward f = make_forward(c, Q, k_cache, v_cache, cu_seqlens, max_query_len, causal, scale, k_scale, v_scale,
                           return_lse, out);
  f.p.workspace_bytes = fa_sm75_paged_workspace_size(&f.p);
  const Tensor work = workspace(f.p.workspace_bytes, k_cache);
  f.p.workspace = work.defined() ? work.data_ptr() : nullptr;
  const int st = fa_sm75_paged_forward(&f.p);
  TORCH_CHECK(st == FA_OK, "flash_attention_paged: ", fa_sm75_last_error());
  if (out.has_value()) written_to(f.O);
  return {f.O, f.L};
}

std::tuple<Tensor, OptTensor> flash_attention_paged_prefix(
    Tensor Q, Tensor k_cache, Tensor v_cache, Tensor prefix_table, Tensor prefix_lens, Tensor block_table,
    Tensor seq_lens, OptTensor cu_seqlens, OptTensor cu_prefix, int64_t max_query_len,
    int64_t max_prefix_queries, int64_t causal, double scale, OptTensor k_scale, OptTensor v_scale,
    bool return_lse, OptTensor out) {
  check_no_tangent("flash_attention_paged_prefix", {&Q, &k_cache, &v_cache, out.has_value() ? &*out : &Q});
  const fa_paged_cache c = make_cache(k_cache, v_cache, block_table, seq_lens, k_scale, v_scale, false);
  check_index(prefix_table, "prefix_table", 2, k_cache);
  check_index(prefix_lens, "prefix_lens", 1, k_cache);
  TORCH_CHECK(prefix_table.size(0) == prefix_lens.size(0), "prefix_table and prefix_lens must have as many rows");
  TORCH_CHECK(prefix_table.size(1) <= 1 || prefix_table.stride(1) == 1, "prefix_table's rows must be contiguous");
  TORCH_CHECK(prefix_lens.size(0) <= 1 || prefix_lens.stride(0) == 1, "prefix_lens must be contiguous");
  fa_paged_prefix x{};
  x.block_table = prefix_table.data_ptr<int32_t>();
  x.lens = prefix_lens.data_ptr<int32_t>();
  x.count = prefix_table.size(0);
  x.max_pages = prefix_table.size(1);
  x.block_table_stride = eff_stride(prefix_table, 0, prefix_table.size(1));
  x.max_queries = max_prefix_queries;
  if (cu_prefix.has_value()) {
    check_index(*cu_prefix, "cu_prefix", 1, k_cache);
    TORCH_CHECK(cu_prefix->size(0) == x.count + 1, "cu_prefix must have prefixes + 1 = ", x.count + 1, " entries");
    TORCH_CHECK(cu_prefix->stride(0) == 1, "cu_prefix must be contiguous");
    x.cu_prefix = cu_prefix->data_ptr<int32_t>();
  } else {
    TORCH_CHECK(x.count == 1, "without cu_prefix there is one prefix, got ", x.count);
  }
  const at::OptionalDeviceGuard guard(at::device_of(k_cache));
  Forward f = make_forward(c, Q, k_cache, v_cache, cu_seqlens, max_query_len, causal, scale, k_scale, v_scale,
                           return_lse, out);
  f.p.workspace_bytes = fa_sm75_paged_prefix_workspace_size(&f.p, &x);
  const Tensor work = workspace(f.p.workspace_bytes, k_cache);
  f.p.workspace = work.defined() ? work.data_ptr() : nullptr;
  const int st = fa_sm75_paged_prefix_forward(&f.p, &x);
  TORCH_CHECK(st == FA_OK, "flash_attention_paged_prefix: ", fa_sm75_last_error());
  if (out.has_value()) written_to(f.O);
  return {f.O, f.L};
}

// Whether [B, H, n] rows of contiguous positions lie apart from each other.
bool rows_disjoint(const Tensor& t) {
  const int64_t n = t.size(2), b = t.size(0), h = t.size(1);
  const int64_t sb = t.stride(0), sh = t.stride(1);
  if (b <= 1) return h <= 1 || sh >= n;
  if (h <= 1) return sb >= n;
  return sb >= sh ? sh >= n && sb >= (h - 1) * sh + n : sb >= n && sh >= (b - 1) * sb + n;
}

Tensor paged_attention_weights(Tensor Q, Tensor LSE, Tensor k_cache, Tensor block_table, Tensor seq_lens,
                               OptTensor cu_seqlens, int64_t max_len, int64_t max_query_len, int64_t causal,
                               double scale, OptTensor k_scale, OptTensor add_to) {
  check_no_tangent("paged_attention_weights", {&Q, &LSE, &k_cache, add_to.has_value() ? &*add_to : &Q});
  const fa_paged_cache c = make_cache(k_cache, k_cache, block_table, seq_lens, k_scale, k_scale, false);
  check_queries(Q, c, k_cache);
  TORCH_CHECK(LSE.scalar_type() == torch::kFloat32, "LSE must be float32");
  TORCH_CHECK(LSE.device() == k_cache.device(), "LSE must be on the cache's device");
  TORCH_CHECK(LSE.dim() == 2 && LSE.size(0) == Q.size(1) && LSE.size(1) == Q.size(0),
              "LSE must be [H_q, tokens]");
  fa_paged_weigh_params p{};
  p.cu_seqlens = cu_pointer(cu_seqlens, k_cache, c.batch, Q.size(0));
  const at::OptionalDeviceGuard guard(at::device_of(k_cache));
  if (Q.numel() != 0) Q = rows_view(Q);
  // (views wider than fa_paged_weigh_params takes)
  if (Q.numel() != 0 && (eff_stride(Q, 0, 0) >= 1 << 23 || eff_stride(Q, 1, 0) >= 1 << 23 ||
                         33 * eff_stride(Q, 0, 0) + Q.size(1) / c.heads_kv * eff_stride(Q, 1, 0) >= 1 << 30))
    Q = Q.contiguous();
  LSE = LSE.contiguous();
  Tensor W;
  if (add_to.has_value()) {
    W = *add_to;
    TORCH_CHECK(W.scalar_type() == torch::kFloat32, "add_to must be float32");
    TORCH_CHECK(W.device() == k_cache.device(), "add_to must be on the cache's device");
    TORCH_CHECK(W.dim() == 3 && W.size(0) == c.batch && W.size(1) == c.heads_kv, "add_to must be [B, H_kv, max_len]");
    TORCH_CHECK(W.size(2) <= 1 || W.stride(2) == 1, "add_to's positions must be contiguous");
    TORCH_CHECK(W.numel() == 0 || rows_disjoint(W), "add_to's rows must not overlap");
    bool apart = spans_apart(W, Q) && spans_apart(W, LSE) && spans_apart(W, k_cache);
    if (k_scale.has_value()) apart = apart && spans_apart(W, *k_scale);
    TORCH_CHECK(apart, "add_to must not share Q's, LSE's or the cache's memory");
  } else {
    TORCH_CHECK(max_len >= 0, "max_len must be non-negative, got ", max_len);
    W = torch::empty({c.batch, c.heads_kv, max_len}, LSE.options());
  }
  p.cache = &c;
  p.q = static_cast<const fa_half*>(Q.data_ptr());
  p.lse = LSE.data_ptr<float>();
  p.weights = W.data_ptr<float>();
  p.weights_stride_b = eff_stride(W, 0, 0);
  p.weights_stride_h = eff_stride(W, 1, 0);
  p.max_len = W.size(2);
  p.add = add_to.has_value();
  p.tokens = Q.size(0);
  p.heads_q = Q.size(1);
  p.q_stride_t = eff_stride(Q, 0, 0); p.q_stride_h = eff_stride(Q, 1, 0);
  p.max_query_len = max_query_len;
  p.scale = (float)scale;
  p.causal = (int)causal;
  p.dtype = dtype_code(Q.scalar_type());
  p.stream = current_stream(k_cache);
  p.workspace_bytes = fa_sm75_paged_weigh_workspace_size(&p);
  const Tensor work = workspace(p.workspace_bytes, k_cache);
  p.workspace = work.defined() ? work.data_ptr() : nullptr;
  const int st = fa_sm75_paged_weigh(&p);
  TORCH_CHECK(st == FA_OK, "paged_attention_weights: ", fa_sm75_last_error());
  if (add_to.has_value()) written_to(W);
  return W;
}

std::tuple<Tensor, Tensor> paged_cache_evict(Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor seq_lens,
                                             Tensor weights, Tensor to_table, int64_t keep, int64_t recent,
                                             OptTensor k_scale, OptTensor v_scale) {
  check_no_tangent("paged_cache_evict", {&k_cache, &v_cache, &weights});
  const fa_paged_cache c = make_cache(k_cache, v_cache, block_table, seq_lens, k_scale, v_scale, true);
  check_index(to_table, "to_table", 2, k_cache);
  TORCH_CHECK(to_table.size(0) == c.batch, "to_table and block_table must have the same batch");
  TORCH_CHECK(to_table.size(1) <= 1 || to_table.stride(1) == 1, "to_table's rows must be contiguous");
  TORCH_CHECK(weights.scalar_type() == torch::kFloat32, "weights must be float32");
  TORCH_CHECK(weights.device() == k_cache.device(), "weights must be on the cache's device");
  TORCH_CHECK(weights.dim() == 3 && weights.size(0) == c.batch && weights.size(1) == c.heads_kv,
              "weights must be [B, H_kv, max_len]");
  TORCH_CHECK(keep >= 0, "keep must be non-negative, got ", keep);
  const at::OptionalDeviceGuard guard(at::device_of(k_cache));
  if (weights.size(2) > 1 && weights.stride(2) != 1) weights = weights.contiguous();
  const auto new_lens = torch::empty({c.batch}, seq_lens.options());
  const auto new_weights = torch::empty({c.batch, c.heads_kv, to_table.size(1) * c.page_size}, weights.options());
  fa_paged_evict_params p{};
  p.cache = &c;
  p.weights = weights.data_ptr<float>();
  p.weights_stride_b = eff_stride(weights, 0, 0);
  p.weights_stride_h = eff_stride(weights, 1, 0);
  p.weights_len = weights.size(2);
  p.to_table = to_table.data_ptr<int32_t>();
  p.to_pages = to_table.size(1);
  p.to_table_stride = eff_stride(to_table, 0, to_table.size(1));
  p.keep = keep;
  p.recent = recent;
  p.new_lens = new_lens.data_ptr<int32_t>();
  p.new_weights = new_weights.data_ptr<float>();
  p.stream = current_stream(k_cache);
  p.workspace_bytes = fa_sm75_paged_evict_workspace_size(&p);
  const Tensor work = workspace(p.workspace_bytes, k_cache);
  p.workspace = work.defined() ? work.data_ptr() : nullptr;
  const int st = fa_sm75_paged_evict(&p);
  TORCH_CHECK(st == FA_OK, "paged_cache_evict: ", fa_sm75_last_error());
  written_to(k_cache);
  written_to(v_cache);
  if (k_scale.has_value()) {
    written_to(*k_scale);
    written_to(*v_scale);
  }
  return {new_lens, new_weights};
}

}  // namespace

void bind_paged(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("paged_cache_write", &paged_cache_write, py::arg("K"), py::arg("V"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("block_table"), py::arg("seq_lens"),
        py::arg("cu_seqlens") = py::none(), py::arg("k_scale") = py::none(),
        py::arg("v_scale") = py::none());
  m.def("paged_cache_read", &paged_cache_read, py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("max_len"),
        py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(),
        py::arg("dtype") = py::none());
  m.def("flash_attention_paged", &flash_attention_paged, py::arg("Q"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("block_table"), py::arg("seq_lens"), py::arg("cu_seqlens"),
        py::arg("max_query_len"), py::arg("causal"), py::arg("scale"),
        py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(),
        py::arg("return_lse") = false, py::arg("out") = py::none());
  m.def("flash_attention_paged_prefix", &flash_attention_paged_prefix, py::arg("Q"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("prefix_table"), py::arg("prefix_lens"), py::arg("block_table"),
        py::arg("seq_lens"), py::arg("cu_seqlens"), py::arg("cu_prefix"), py::arg("max_query_len"),
        py::arg("max_prefix_queries"), py::arg("causal"), py::arg("scale"),
        py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(),
        py::arg("return_lse") = false, py::arg("out") = py::none());
  m.def("paged_attention_weights", &paged_attention_weights, py::arg("Q"), py::arg("LSE"), py::arg("k_cache"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("cu_seqlens"), py::arg("max_len"),
        py::arg("max_query_len"), py::arg("causal"), py::arg("scale"), py::arg("k_scale") = py::none(),
        py::arg("add_to") = py::none());
  m.def("paged_cache_evict", &paged_cache_evict, py::arg("k_cache"), py::arg("v_cache"), py::arg("block_table"),
        py::arg("seq_lens"), py::arg("weights"), py::arg("to_table"), py::arg("keep"), py::arg("recent"),
        py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none());
}
