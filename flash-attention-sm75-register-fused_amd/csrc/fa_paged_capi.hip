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

// Whether two ranges of bytes share none.
bool apart(const void* x, int64_t nx, const void* y, int64_t ny) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
  return nx == 0 || ny == 0 || a + nx <= b || b + ny <= a;
}

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

// Checks the prefixes of a forward call and fills both stages' arguments from its own ones.
int make_prefix(const fa_paged_prefix* x, const fa::PagedArgs& a, fa::PagedShared* prefix, fa::PagedShared* own) {
  if (x == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "prefix must not be NULL");
  if (x->count < 0 || x->max_pages < 0 || x->block_table_stride < 0 || x->max_queries < 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "the prefixes' sizes and strides must be non-negative");
  if (x->count > (1 << 20)) return capi_fail(FA_ERR_TOO_LARGE, "the prefixes exceed 2^20");
  if (x->max_pages > fa::kPagedMaxKeys >> a.page_shift)
    return capi_fail(FA_ERR_TOO_LARGE, "the prefixes' max_pages * page_size exceeds 2^30 tokens");
  if (x->count > 0 && (x->lens == nullptr || (x->max_pages > 0 && x->block_table == nullptr)))
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "the prefixes' block_table and lens must not be NULL");
  if (x->count != 1 && x->cu_prefix == nullptr)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "without cu_prefix there is one prefix, got %lld", (long long)x->count);
  if (!aligned(x->block_table, 4) || !aligned(x->lens, 4) || !aligned(x->cu_prefix, 4))
    return capi_fail(FA_ERR_MISALIGNED, "the prefixes' block_table, lens and cu_prefix must be 4-byte aligned");
  if ((int64_t)a.tokens * a.hq + x->count * a.hkv * 32 > (1 << 27))
    return capi_fail(FA_ERR_TOO_LARGE, "tokens * heads_q + 32 * prefixes * heads_kv exceeds 2^27");
  *own = fa::PagedShared{a};
  own->groups = x->cu_prefix;
  own->prefixes = (int)x->count;
  own->seqs = a.batch;
  own->pre_table = x->block_table;
  own->pre_lens = x->lens;
  own->pre_stride = x->block_table_stride;
  own->pre_pages = (int)x->max_pages;
  *prefix = *own;
  prefix->batch = (int)x->count;
  prefix->table = x->block_table;
  prefix->lens = x->lens;
  prefix->table_stride = x->block_table_stride;
  prefix->max_pages = (int)x->max_pages;
  prefix->causal = 0;
  prefix->lse = nullptr;
  return FA_OK;
}

// (a checked call's: tokens > 0)
int64_t longest_shared(const fa_paged_prefix* x, const fa::PagedArgs& a) {
  return x->max_queries > 0 && x->max_queries < a.tokens ? x->max_queries : a.tokens;
}

// Checks a call that sums weights; *nothing: no weight to write.
int make_weigh(const fa_paged_weigh_params* p, fa::WeighArgs* w, bool* nothing) {
  *w = fa::WeighArgs{};
  if (p == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "params must not be NULL");
  if (p->cache == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "cache must not be NULL");
  fa_paged_cache c = *p->cache;  // V is not looked at
  c.v = c.k;
  c.v_scale = c.k_scale;
  c.v_stride_p = c.k_stride_p; c.v_stride_h = c.k_stride_h; c.v_stride_n = c.k_stride_n;
  c.vs_stride_p = c.ks_stride_p; c.vs_stride_h = c.ks_stride_h; c.vs_stride_n = c.ks_stride_n;
  fa_paged_params f{};
  f.cache = &c;
  f.q = p->q;
  f.o = const_cast<fa_half*>(p->q);  // (none is written)
  f.lse = const_cast<float*>(p->lse);
  f.tokens = p->tokens;
  f.heads_q = p->heads_q;
  f.q_stride_t = f.o_stride_t = p->q_stride_t;
  f.q_stride_h = f.o_stride_h = p->q_stride_h;
  f.cu_seqlens = p->cu_seqlens;
  f.max_query_len = p->max_query_len;
  f.scale = p->scale;
  f.causal = p->causal;
  f.dtype = p->dtype;
  f.workspace = p->workspace;
  f.workspace_bytes = p->workspace_bytes;
  bool empty = true;
  if (int st = make_forward(&f, &w->p, &empty)) return st;
  if (!empty && p->lse == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "lse must not be NULL");
  // 64 rows of one KV head's queries (33 tokens, or of one head 64) are read through one window, by
  // products of 24 bits.
  constexpr int64_t kStride = 1 << 23;
  if (!empty && (p->q_stride_t >= kStride || p->q_stride_h >= kStride || w->p.group >= kStride ||
                 33 * p->q_stride_t + w->p.group * p->q_stride_h >= 1 << 30))
    return capi_fail(FA_ERR_TOO_LARGE, "Q's strides must be below 2^23, and a group's heads and 33 tokens within 2^30 elements");
  if (p->max_len < 0 || p->weights_stride_b < 0 || p->weights_stride_h < 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "max_len and the weights' strides must be non-negative");
  if (p->max_len > fa::kPagedMaxKeys) return capi_fail(FA_ERR_TOO_LARGE, "max_len exceeds 2^30");
  const int64_t pairs = (int64_t)w->p.batch * w->p.hkv;
  *nothing = pairs == 0 || p->max_len == 0 || (empty && p->add);
  if (*nothing) return FA_OK;
  if (pairs > (1 << 22) || pairs * ((p->max_len + 31) / 32) > (1 << 26))
    return capi_fail(FA_ERR_TOO_LARGE, "batch * heads_kv exceeds 2^22, or batch * heads_kv * max_len 2^31");
  if (p->weights == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "weights must not be NULL");
  if (!aligned(p->weights, 4)) return capi_fail(FA_ERR_MISALIGNED, "weights must be 4-byte aligned");
  if (empty) {  // no row: every weight is 0
    w->p.tokens = 0;
    w->p.group = 1;
    w->p.c = 1.0f;
  }
  w->lse = p->lse;
  w->out = p->weights;
  w->sb = p->weights_stride_b;
  w->sh = p->weights_stride_h;
  w->max_len = (int)p->max_len;
  w->add = p->add ? 1 : 0;
  return FA_OK;
}

// Checks an eviction; *nothing: no sequence.
int make_evict(const fa_paged_evict_params* p, fa::EvictArgs* e, bool* nothing) {
  *e = fa::EvictArgs{};
  if (p == nullptr) return capi_fail(FA_ERR_INVALID_ARGUMENT, "params must not be NULL");
  if (int st = make_cache(p->cache, FA_DTYPE_FP16, &e->p)) return st;  // (rows are copied as they are)
  const fa::PagedArgs& a = e->p;
  if (a.hkv == 0) return capi_fail(FA_ERR_INVALID_ARGUMENT, "heads_kv must be positive");
  if (p->keep < 0 || p->recent < 0 || p->to_pages < 0 || p->weights_len < 0 || p->workspace_bytes < 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "keep, recent and sizes must be non-negative");
  if (p->recent > p->keep)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "recent (%lld) must not exceed keep (%lld)", (long long)p->recent,
                     (long long)p->keep);
  if (p->weights_stride_b < 0 || p->weights_stride_h < 0 || p->to_table_stride < 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "strides must be non-negative");
  if (p->to_pages > fa::kPagedMaxKeys >> a.page_shift)
    return capi_fail(FA_ERR_TOO_LARGE, "to_pages * page_size exceeds 2^30 tokens");
  const int64_t room = (int64_t)a.max_pages << a.page_shift, to_room = p->to_pages << a.page_shift;
  const int64_t slots = p->keep < room ? p->keep : room;
  if (to_room < slots)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "to_table has room for %lld rows, up to %lld stay", (long long)to_room,
                     (long long)slots);
  if (p->weights_len < room)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "weights must have block_table's room, %lld positions, got %lld",
                     (long long)room, (long long)p->weights_len);
  const int64_t pairs = (int64_t)a.batch * a.hkv;
  *nothing = pairs == 0;
  if (*nothing) return FA_OK;
  if (pairs > (1 << 20) || pairs * slots > (1 << 29))
    return capi_fail(FA_ERR_TOO_LARGE, "batch * heads_kv exceeds 2^20, or the rows that stay 2^29");
  if (p->new_lens == nullptr || (to_room > 0 && p->new_weights == nullptr) ||
      (room > 0 && p->weights == nullptr) || (p->to_pages > 0 && p->to_table == nullptr))
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "weights, to_table, new_lens and new_weights must not be NULL");
  if (!aligned(p->weights, 4) || !aligned(p->to_table, 4) || !aligned(p->new_lens, 4) || !aligned(p->new_weights, 4))
    return capi_fail(FA_ERR_MISALIGNED, "weights, to_table, new_lens and new_weights must be 4-byte aligned");
  e->weights = p->weights;
  e->wb = p->weights_stride_b;
  e->wh = p->weights_stride_h;
  e->to_table = p->to_table;
  e->to_stride = p->to_table_stride;
  e->to_pages = (int)p->to_pages;
  e->keep = (int)slots;
  e->recent = (int)(p->recent < INT32_MAX ? p->recent : INT32_MAX);
  e->new_lens = p->new_lens;
  e->new_weights = p->new_weights;
  e->slots = (int)slots;
  return FA_OK;
}

// (a checked call's: tokens > 0)
int64_t longest_query(const int32_t* cu_seqlens, int64_t max_query_len, int64_t tokens) {
  if (cu_seqlens == nullptr) return 1;
  return max_query_len > 0 && max_query_len < tokens ? max_query_len : tokens;
}
int64_t longest_query(const fa_paged_params* p) {
  return longest_query(p->cu_seqlens, p->max_query_len, p->tokens);
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

int64_t fa_sm75_paged_prefix_workspace_size(const fa_paged_params* p, const fa_paged_prefix* x) {
  const fa::SavedError keep;  // a size is no error report
  fa::PagedArgs a;
  fa::PagedShared prefix, own;
  bool empty = true;
  if (make_forward(p, &a, &empty) != FA_OK || empty || make_prefix(x, a, &prefix, &own) != FA_OK) return 0;
  if (x->count == 0) return fa_sm75_paged_workspace_size(p);
  const int d = (int)p->cache->head_dim;
  if (fa::joins_prefixes(own, d, longest_query(p)))
    return fa::plan_joined(own, d, longest_query(p), INT64_MAX).workspace_bytes;
  return fa::plan_prefix(prefix, d, longest_shared(x, a)).workspace_bytes +
         fa::plan_paged(own, d, longest_query(p), INT64_MAX, fa::kOwn).workspace_bytes;
}

int fa_sm75_paged_prefix_forward(const fa_paged_params* p, const fa_paged_prefix* x) {
  fa::capi_clear_error();
  fa::PagedArgs a;
  fa::PagedShared prefix, own;
  bool empty = true;
  if (int st = make_forward(p, &a, &empty)) return st;
  if (empty) return FA_OK;
  if (int st = make_prefix(x, a, &prefix, &own)) return st;
  if (x->count == 0) return fa_sm75_paged_forward(p);
  const int d = (int)p->cache->head_dim;
  const hipStream_t stream = static_cast<hipStream_t>(p->stream);
  const int64_t bytes = p->workspace != nullptr ? p->workspace_bytes : 0;
  if (fa::joins_prefixes(own, d, longest_query(p))) {
    fa::launch_paged_joined(own, fa::plan_joined(own, d, longest_query(p), bytes), d, p->workspace, stream);
    return check_launch();
  }
  const fa::PagedPlan first = fa::plan_prefix(prefix, d, longest_shared(x, a));
  const int64_t rest = bytes - first.workspace_bytes;
  if (rest < 0)
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "the workspace must hold %lld bytes at least, got %lld",
                     (long long)first.workspace_bytes, (long long)bytes);
  fa::launch_paged_prefix(prefix, own, first, d, p->workspace, stream);
  const fa::PagedPlan plan = fa::plan_paged(own, d, longest_query(p), rest, fa::kOwn);
  fa::launch_paged_attention(own, plan, d, static_cast<char*>(p->workspace) + first.workspace_bytes, stream);
  return check_launch();
}

int64_t fa_sm75_paged_weigh_workspace_size(const fa_paged_weigh_params* p) {
  const fa::SavedError keep;  // a size is no error report
  fa::WeighArgs w;
  bool nothing = true;
  if (make_weigh(p, &w, &nothing) != FA_OK || nothing) return 0;
  return fa::plan_weigh(w, longest_query(p->cu_seqlens, p->max_query_len, p->tokens), INT64_MAX).workspace_bytes;
}

int fa_sm75_paged_weigh(const fa_paged_weigh_params* p) {
  fa::capi_clear_error();
  fa::WeighArgs w;
  bool nothing = true;
  if (int st = make_weigh(p, &w, &nothing)) return st;
  if (nothing) return FA_OK;
  const fa::WeighPlan plan = fa::plan_weigh(w, longest_query(p->cu_seqlens, p->max_query_len, p->tokens),
                                            p->workspace != nullptr ? p->workspace_bytes : 0);
  fa::launch_weigh(w, plan, (int)p->cache->head_dim, p->workspace, static_cast<hipStream_t>(p->stream));
  return check_launch();
}

int64_t fa_sm75_paged_evict_workspace_size(const fa_paged_evict_params* p) {
  const fa::SavedError keep;  // a size is no error report
  fa::EvictArgs e;
  bool nothing = true;
  return make_evict(p, &e, &nothing) != FA_OK || nothing ? 0 : fa::evict_workspace_bytes(e);
}

int fa_sm75_paged_evict(const fa_paged_evict_params* p) {
  fa::capi_clear_error();
  fa::EvictArgs e;
  bool nothing = true;
  if (int st = make_evict(p, &e, &nothing)) return st;
  if (nothing) return FA_OK;
  const int64_t need = fa::evict_workspace_bytes(e);
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need))
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "the workspace must hold %lld bytes, got %lld", (long long)need,
                     (long long)(p->workspace != nullptr ? p->workspace_bytes : 0));
  if (!aligned(p->workspace, 16)) return capi_fail(FA_ERR_MISALIGNED, "workspace must be 16-byte aligned");
  // (a row's workgroups read a length and weights while others write what stays)
  const fa::PagedArgs& a = e.p;
  const int64_t pairs = (int64_t)a.batch * a.hkv, room = (int64_t)a.max_pages << a.page_shift;
  const int64_t span = room > 0 ? (a.batch - 1) * e.wb + (a.hkv - 1) * e.wh + room : 0;
  if (!apart(e.new_lens, 4ll * a.batch, a.lens, 4ll * a.batch))
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "new_lens must not share seq_lens' memory");
  if (!apart(e.new_weights, 4 * pairs * (p->to_pages << a.page_shift), e.weights, 4 * span))
    return capi_fail(FA_ERR_INVALID_ARGUMENT, "new_weights must not share the weights' memory");
  fa::launch_evict(e, (int)p->cache->head_dim, p->workspace, static_cast<hipStream_t>(p->stream));
  return check_launch();
}

}  // extern "C"
