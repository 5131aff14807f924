// C ABI of the paged key/value cache: argument checks (all before the first
// HIP call), then the launches.
#include <hip/hip_runtime.h>

#include <cmath>

#include "fa_capi_error.h"
#include "fa_paged.h"
#include "flash_attn_sm75.h"

namespace {

using fa::capi_fail;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_launch() {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return capi_fail(FA_ERR_HIP, "HIP launch failed: %s", hipGetErrorString(e));
  return FA_OK;
}

// Checks the cache's description; *a is filled from it.
int make_cache(const fa_paged_cache* c, int dtype, fa::PagedArgs* a) {
  *a = fa::PagedArgs{};
  if (c == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "cache must not be NULL");
  if (dtype != FA_DTYPE_FP16 && dtype != FA_DTYPE_BF16)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "dtype must be 0 (binary16) or 1 (bfloat16), got %d", dtype);
  if (c->batch < 0 || c->heads_kv < 0 || c->head_dim < 0 || c->num_pages < 0 || c->max_pages < 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "sizes must be non-negative");
  if (c->head_dim != 64 && c->head_dim != 128)
    return capi_fail(FA_ERR_UNSUPPORTED_HEAD_DIM, "a paged cache supports head_dim=64 or 128, got %lld",
                     (long long)c->head_dim);
  if (c->page_size < 16 || c->page_size > (1 << 20) || (c->page_size & (c->page_size - 1)) != 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT,
                     "page_size must be a power of two from 16 to 2^20, got %lld", (long long)c->page_size);
  if (c->batch > (1 << 20) || c->heads_kv > (1 << 16) || c->num_pages > INT32_MAX)
    return capi_fail(FA_ERR_TOO_LARGE, "batch, heads_kv or num_pages exceeds the supported maximum");
  if (c->max_pages > fa::kPagedMaxKeys / c->page_size)
    return capi_fail(FA_ERR_TOO_LARGE, "max_pages * page_size exceeds 2^30 tokens");
  const bool q8 = c->k_scale != nullptr || c->v_scale != nullptr;
  if (q8 && (c->k_scale == nullptr || c->v_scale == nullptr))
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "k_scale and v_scale go together");
  const bool empty = c->batch == 0 || c->heads_kv == 0;
  if (!empty && (c->seq_lens == nullptr || (c->max_pages > 0 && c->block_table == nullptr)))
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "block_table and seq_lens must not be NULL");
  if (!empty && c->num_pages > 0 && (c->k == nullptr || c->v == nullptr))
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "the cache's K and V pointers must not be NULL");
  if (!aligned(c->k, 16) || !aligned(c->v, 16))
    return capi_fail(FA_ERR_MISALIGNED, "the cache's K and V must be 16-byte aligned");
  if (!aligned(c->block_table, 4) || !aligned(c->seq_lens, 4))
    return capi_fail(FA_ERR_MISALIGNED, "block_table and seq_lens must be 4-byte aligned");
  if (c->block_table_stride < 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "strides must be non-negative");
  const int esize = q8 ? 1 : 2;
  const int64_t strides[6] = {c->k_stride_p, c->k_stride_h, c->k_stride_n,
                              c->v_stride_p, c->v_stride_h, c->v_stride_n};
  for (int64_t s : strides) {
    if (s < 0) return capi_fail(FA_ERR_INVALID_ARGUMENT, "strides must be non-negative");
    if (s * esize % 16 != 0)
      return capi_fail(FA_ERR_MISALIGNED, "page/head/row strides must be multiples of 16 bytes");
  }
  if (c->k_stride_n < c->head_dim || c->v_stride_n < c->head_dim)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "row stride must be at least head_dim");
  if (c->k_stride_n * esize > fa::kPagedMaxRowBytes || c->v_stride_n * esize > fa::kPagedMaxRowBytes)
    return capi_fail(FA_ERR_TOO_LARGE, "row stride exceeds 2^24 bytes");
  const int64_t scales[6] = {c->ks_stride_p, c->ks_stride_h, c->ks_stride_n,
                             c->vs_stride_p, c->vs_stride_h, c->vs_stride_n};
  if (q8) {
    for (int64_t s : scales)
      if (s < 0) return capi_fail(FA_ERR_INVALID_ARGUMENT, "strides must be non-negative");
    if (c->ks_stride_n < 1 || c->vs_stride_n < 1)
      return capi_fail(FA_ERR_INVALID_ARGUMENT, "the scales' row stride must be at least 1");
    if (c->ks_stride_n > fa::kPagedMaxRowBytes || c->vs_stride_n > fa::kPagedMaxRowBytes)
      return capi_fail(FA_ERR_TOO_LARGE, "the scales' row stride exceeds 2^24 bytes");
  }
  a->k = static_cast<uint8_t*>(c->k);
  a->v = static_cast<uint8_t*>(c->v);
  a->ks = c->k_scale;
  a->vs = c->v_scale;
  a->kp = c->k_stride_p * esize; a->kh = c->k_stride_h * esize; a->kn = c->k_stride_n * esize;
  a->vp = c->v_stride_p * esize; a->vh = c->v_stride_h * esize; a->vn = c->v_stride_n * esize;
  a->ksp = c->ks_stride_p; a->ksh = c->ks_stride_h; a->ksn = c->ks_stride_n;
  a->vsp = c->vs_stride_p; a->vsh = c->vs_stride_h; a->vsn = c->vs_stride_n;
  a->table = c->block_table;
  a->lens = c->seq_lens;
  a->table_stride = c->block_table_stride;
  a->num_pages = (int)c->num_pages;
  a->page_shift = __builtin_ctzll((unsigned long long)c->page_size);
  a->max_pages = (int)c->max_pages;
  a->batch = (int)c->batch;
  a->hkv = (int)c->heads_kv;
  a->bf16 = dtype == FA_DTYPE_BF16 ? 1 : 0;
  return FA_OK;
}

int check_tokens(const fa::PagedArgs& a, int64_t tokens, const int32_t* cu_seqlens) {
  if (tokens < 0) return capi_fail(FA_ERR_INVALID_ARGUMENT, "tokens must be non-negative");
  if (tokens > (1 << 24)) return capi_fail(FA_ERR_TOO_LARGE, "tokens exceeds 2^24");
  if (!aligned(cu_seqlens, 4)) return capi_fail(FA_ERR_MISALIGNED, "cu_seqlens must be 4-byte aligned");
  if (cu_seqlens == nullptr && tokens < a.batch)
    return capi_fail(FA_ERR_INVALID_ARGUMENT,
                     "without cu_seqlens there is a token for each of the %d sequences, got %lld",
                     a.batch, (long long)tokens);
  return FA_OK;
}

int check_rows(const void* p, int64_t stride_t, int64_t stride_h, const char* name) {
  if (p == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "%s must not be NULL", name);
  if (!aligned(p, 16)) return capi_fail(FA_ERR_MISALIGNED, "%s must be 16-byte aligned", name);
  if (stride_t < 0 || stride_h < 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "strides must be non-negative");
  if (stride_t % 8 != 0 || stride_h % 8 != 0)
    return capi_fail(FA_ERR_MISALIGNED, "token/head strides must be multiples of 8 elements (16 bytes)");
  return FA_OK;
}

// Checks a forward call and fills *a; *empty: no row to write.
int make_forward(const fa_paged_params* p, fa::PagedArgs* a, bool* empty) {
  if (p == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "params must not be NULL");
  if (int st = make_cache(p->cache, p->dtype, a)) return st;
  if (int st = check_tokens(*a, p->tokens, p->cu_seqlens)) return st;
  if (p->heads_q < 0) return capi_fail(FA_ERR_INVALID_ARGUMENT, "sizes must be non-negative");
  if (p->heads_q > (1 << 20)) return capi_fail(FA_ERR_TOO_LARGE, "heads_q exceeds 2^20");
  if (p->heads_q > 0 && a->hkv == 0)
    return capi_fail(FA_ERR_HEADS_NOT_DIVISIBLE, "heads_kv must be positive");
  if (a->hkv > 0 && p->heads_q % a->hkv != 0)
    return capi_fail(FA_ERR_HEADS_NOT_DIVISIBLE,
                     "heads mismatch: Q heads (%lld) not divisible by K/V heads (%d)",
                     (long long)p->heads_q, a->hkv);
  if (!std::isfinite(p->scale)) return capi_fail(FA_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (p->causal != FA_CAUSAL_NONE && p->causal != FA_CAUSAL_BOTTOM_RIGHT)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "causal must be 0 or 2 (bottom-right), got %d", p->causal);
  if (p->max_query_len < 0 || p->workspace_bytes < 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "max_query_len and workspace_bytes must be non-negative");
  *empty = p->tokens == 0 || a->batch == 0 || p->heads_q == 0;
  if (*empty) return FA_OK;
  if (int st = check_rows(p->q, p->q_stride_t, p->q_stride_h, "Q")) return st;
  if (int st = check_rows(p->o, p->o_stride_t, p->o_stride_h, "O")) return st;
  if (!aligned(p->lse, 4)) return capi_fail(FA_ERR_MISALIGNED, "lse must be 4-byte aligned");
  if (!aligned(p->workspace, 16))
    return capi_fail(FA_ERR_MISALIGNED, "workspace must be 16-byte aligned");
  // Workgroups of a launch that does not split: one for each unit of 16 rows at least.
  if (p->tokens * p->heads_q + (int64_t)a->batch * a->hkv * 32 > (1 << 27))
    return capi_fail(FA_ERR_TOO_LARGE, "tokens * heads_q + 32 * batch * heads_kv exceeds 2^27");
  a->tokens = (int)p->tokens;
  a->cu = p->cu_seqlens;
  a->q = reinterpret_cast<const _Float16*>(p->q);
  a->o = reinterpret_cast<_Float16*>(p->o);
  a->lse = p->lse;
  a->qt = p->q_stride_t; a->qh = p->q_stride_h;
  a->ot = p->o_stride_t; a->oh = p->o_stride_h;
  a->hq = (int)p->heads_q;
  a->group = (int)(p->heads_q / a->hkv);
  a->causal = p->causal != FA_CAUSAL_NONE ? 1 : 0;
  // A zero scale still has to give hidden keys no weight (2^(-inf c) = 0).
  a->c = std::fmax(std::fabs(p->scale) * 1.4426950408889634f, 1e-30f);
  a->negate_q = p->scale < 0.0f ? 1 : 0;
  return FA_OK;
}

// (a checked call's: tokens > 0)
int64_t longest_query(const fa_paged_params* p) {
  if (p->cu_seqlens == nullptr) return 1;
  return p->max_query_len > 0 && p->max_query_len < p->tokens ? p->max_query_len : p->tokens;
}

}  // namespace

extern "C" {

int fa_sm75_paged_write(const fa_paged_cache* cache, const fa_paged_rows* rows) {
  fa::capi_clear_error();
  fa::PagedArgs a;
  if (rows == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "rows must not be NULL");
  if (int st = make_cache(cache, rows->dtype, &a)) return st;
  if (int st = check_tokens(a, rows->tokens, rows->cu_seqlens)) return st;
  if (rows->tokens == 0 || a.batch == 0 || a.hkv == 0 || a.num_pages == 0 || a.max_pages == 0) return FA_OK;
  if (int st = check_rows(rows->k, rows->k_stride_t, rows->k_stride_h, "K")) return st;
  if (int st = check_rows(rows->v, rows->v_stride_t, rows->v_stride_h, "V")) return st;
  if (rows->tokens * a.hkv > (1 << 26))
    return capi_fail(FA_ERR_TOO_LARGE, "tokens * heads_kv exceeds 2^26 rows");
  a.tokens = (int)rows->tokens;
  a.cu = rows->cu_seqlens;
  a.k_new = reinterpret_cast<const _Float16*>(rows->k);
  a.v_new = reinterpret_cast<const _Float16*>(rows->v);
  a.knt = rows->k_stride_t; a.knh = rows->k_stride_h;
  a.vnt = rows->v_stride_t; a.vnh = rows->v_stride_h;
  fa::launch_paged_write(a, (int)cache->head_dim, static_cast<hipStream_t>(rows->stream));
  return check_launch();
}

int fa_sm75_paged_read(const fa_paged_cache* cache, fa_half* k, fa_half* v, int64_t max_len,
                       int dtype, void* stream) {
  fa::capi_clear_error();
  fa::PagedArgs a;
  if (int st = make_cache(cache, dtype, &a)) return st;
  if (max_len < 0) return capi_fail(FA_ERR_INVALID_ARGUMENT, "max_len must be non-negative");
  if (max_len == 0 || a.batch == 0 || a.hkv == 0) return FA_OK;
  if (max_len > (1 << 27) || (int64_t)a.batch * a.hkv > (1 << 27) ||
      max_len * a.batch * a.hkv > (1 << 27))
    return capi_fail(FA_ERR_TOO_LARGE, "batch * heads_kv * max_len exceeds 2^27 rows");
  if (k == nullptr || v == nullptr)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "K and V must not be NULL");
  if (!aligned(k, 16) || !aligned(v, 16))
    return capi_fail(FA_ERR_MISALIGNED, "K and V must be 16-byte aligned");
  a.k_out = reinterpret_cast<_Float16*>(k);
  a.v_out = reinterpret_cast<_Float16*>(v);
  a.max_len = (int)max_len;
  fa::launch_paged_read(a, (int)cache->head_dim, static_cast<hipStream_t>(stream));
  return check_launch();
}

int64_t fa_sm75_paged_workspace_size(const fa_paged_params* p) {
  const fa::SavedError keep;  // a size is no error report
  fa::PagedArgs a;
  bool empty = true;
  if (make_forward(p, &a, &empty) != FA_OK || empty) return 0;
  return fa::plan_paged(a, (int)p->cache->head_dim, longest_query(p), INT64_MAX).workspace_bytes;
}

int fa_sm75_paged_forward(const fa_paged_params* p) {
  fa::capi_clear_error();
  fa::PagedArgs a;
  bool empty = true;
  if (int st = make_forward(p, &a, &empty)) return st;
  if (empty) return FA_OK;
  const int head_dim = (int)p->cache->head_dim;
  const fa::PagedPlan plan = fa::plan_paged(a, head_dim, longest_query(p),
                                            p->workspace != nullptr ? p->workspace_bytes : 0);
  fa::launch_paged_attention(a, plan, head_dim, p->workspace, static_cast<hipStream_t>(p->stream));
  return check_launch();
}

}  // extern "C"
