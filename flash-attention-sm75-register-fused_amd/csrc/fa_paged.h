// Paged key/value cache: kernel arguments, and the pieces its kernels share
// (fa_paged_cache.hip: writing and reading rows, fa_paged_attn.h: attention
// over the cache, fa_paged.hip: launchers).
//
// Positions of a sequence are cut into pages of 2^page_shift tokens; entry i of
// its row of the block table names the page of positions [i << page_shift,
// (i + 1) << page_shift).  An entry outside [0, num_pages) names no page (one
// that is gone, or a wrong one): nothing is read or written there.  All of it
// lives on the device, so a captured call sees the tables of each replay, and
// every value read from it is held to the ranges the launch was made for before
// it reaches an address.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fa {

struct PagedArgs {
  // The cache: page p, KV head h, row r of K at k + p * kp + h * kh + r * kn
  // (strides in bytes); e4m3: its scale at ks + p * ksp + h * ksh + r * ksn.
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;  // nullptr: 16-bit rows
  uint8_t* vs;
  int64_t kp, kh, kn;
  int64_t vp, vh, vn;
  int64_t ksp, ksh, ksn;
  int64_t vsp, vsh, vsn;
  const int32_t* table;  // [batch, max_pages], rows table_stride apart
  const int32_t* lens;   // [batch]
  const int32_t* cu;     // [batch + 1], or nullptr: one token in every sequence
  int64_t table_stride;
  int num_pages, page_shift, max_pages;
  int tokens, batch, hkv;
  int bf16;  // element type of the 16-bit tensors

  // New rows of a write, the padded tensors of a read (strides in elements).
  const _Float16* k_new;
  const _Float16* v_new;
  int64_t knt, knh, vnt, vnh;
  _Float16* k_out;
  _Float16* v_out;
  int max_len;

  // Attention.
  const _Float16* q;
  _Float16* o;
  float* lse;  // [hq, tokens] or nullptr
  int64_t qt, qh, ot, oh;
  int hq, group;
  int causal;    // token i of n of a sequence of len tokens sees key j iff j <= len - n + i
  float c;       // |scale| * log2(e), clamped away from 0
  int negate_q;  // scale < 0
  // Quotients that every workgroup would begin with.
  float inv_group;  // 1 / group
  float rescale;    // kRescaleLog2 / c
  // Plan: `classes` (2^class_shift) sequences of workgroups, class x holding the `heads` KV
  // heads x, x + classes, ...; wgs of them in each class (split), or one for each unit.
  int classes, class_shift, heads, wgs;
  int split;
  float* part_o;
  float* part_ml;
  uint64_t* flags;  // one for each of the two records of a workgroup, and one more
  uint64_t mark;    // what a written record's flag holds (merge_mark)
  int units;        // the most units a class can have
  int resident;     // the chunk kernel's workgroups of a class that run at once
  int pieces;       // most pieces the chunk kernel may cut a unit into, 0: any number
  int stream_v;     // the chunk kernel reads V non-temporally
};

// Largest key count a block table may cover, and row stride (bytes) of a cache
// tensor: a window over 64 of its rows stays within 31 bits.
constexpr int64_t kPagedMaxKeys = 1 << 30;
constexpr int64_t kPagedMaxRowBytes = (int64_t)1 << 24;

int launch_paged_write(const PagedArgs& a, int head_dim, hipStream_t stream);
int launch_paged_read(const PagedArgs& a, int head_dim, hipStream_t stream);

// Attention over the cache.
struct PagedPlan {
  int classes, wgs, rows;  // rows: query columns of a unit
  bool split;
  bool combine;       // some unit may have more partials than the kernel merges itself
  int units, y;       // of the combine kernel's grid
  bool chunk;         // units of 128 rows (fa_paged_chunk.h)
  int resident, pieces;
  bool stream_v;
  int64_t workspace_bytes;
};
PagedPlan plan_paged(const PagedArgs& a, int head_dim, int64_t max_query_len,
                     int64_t workspace_bytes);
int launch_paged_attention(const PagedArgs& a, const PagedPlan& plan, int head_dim,
                           void* workspace, hipStream_t stream);
template <int D, bool BF16, bool FP8>
void launch_paged_attn(const PagedArgs& a, int rows, int64_t grid, hipStream_t stream);
template <int D, bool BF16, bool FP8>
void launch_paged_chunk(const PagedArgs& a, int64_t grid, hipStream_t stream);
template <int D, bool BF16>
void launch_paged_combine(const PagedArgs& a, int rows, int y, hipStream_t stream);

}  // namespace fa

#ifdef __HIPCC__
#include "fa_kernel_common.h"

namespace fa {
namespace {

typedef const __attribute__((address_space(4))) int32_t cint32;

// A device table read through the scalar cache; the address has to be the
// same in every lane.
__device__ __forceinline__ int load_scalar(const int32_t* p) { return *(cint32*)(uintptr_t)p; }

__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return max(lo, min(x, hi)); }

// A value that is the same in every lane, in a scalar register: a clamp is done in
// vector ones (v_med3), and a buffer window made of it would be taken for a
// different one in each lane, its loads for a loop over them.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// One sequence: its rows [t0, t0 + n) of the new tokens, its length with them
// and the keys its pages can hold of it.
struct PagedSeq {
  int t0, n, len, keys;
};
template <class Load>
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int b, Load load) {
  PagedSeq s;
  const int len = load(a.lens + b);  // (all loads together)
  if (a.cu != nullptr) {
    const int t0 = load(a.cu + b), t1 = load(a.cu + b + 1);
    s.t0 = clamp_int(t0, 0, a.tokens);
    s.n = clamp_int(t1, s.t0, a.tokens) - s.t0;
  } else {
    s.t0 = min(b, a.tokens);
    s.n = b < a.tokens ? 1 : 0;
  }
  s.len = max(0, len);
  s.keys = min(s.len, a.max_pages << a.page_shift);
  return s;
}
// (b the same in every lane; all of it in scalar registers)
__device__ __forceinline__ PagedSeq scalar_seq(const PagedArgs& a, int b) {
  const PagedSeq s = paged_seq(a, uniform(b), load_scalar);
  return {uniform(s.t0), uniform(s.n), uniform(s.len), uniform(s.keys)};
}

// The factor an e8m0 scale stands for (127: 1).  Only its exponent is used.
__device__ __forceinline__ float scale_of(unsigned byte) {
  return __builtin_bit_cast(float, byte << 23);
}

// 8 codes (two words) times a power of two, as 16-bit values: exact for rows
// that paged_cache_write wrote in this type.
template <bool BF16>
__device__ __forceinline__ half8 dequantise8(unsigned w0, unsigned w1, float scale) {
  uint4v r;
  if constexpr (BF16) {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true));
  } else {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, true));
  }
  return __builtin_bit_cast(half8, r);
}

}  // namespace
}  // namespace fa
#endif
