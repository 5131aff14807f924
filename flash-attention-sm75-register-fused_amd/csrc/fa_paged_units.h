// What the two attention kernels over a paged cache (fa_paged_attn.h, fa_paged_chunk.h)
// share: a sequence's rows, wave broadcasts, and merging partial results.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_paged.h"

namespace fa {
namespace {

__device__ __forceinline__ int wave_bcast(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ int64_t wave_bcast(int64_t x, int lane) {
  return (int64_t)(uint32_t)wave_bcast((int)x, lane) |
         ((int64_t)wave_bcast((int)(x >> 32), lane) << 32);
}

// Blocks of R rows of a sequence: its units for one KV head.
template <int R>
__device__ __forceinline__ int paged_blocks(const PagedArgs& a, const PagedSeq& s) {
  return (int)(((int64_t)s.n * a.group + R - 1) / R);
}

// Row r of a sequence's rows: the addresses of its Q, O and LSE.
struct PagedRow {
  int token, head;
};
__device__ __forceinline__ PagedRow paged_row(const PagedArgs& a, const PagedSeq& s, int hkv, int r) {
  const int i = r / a.group;
  return {s.t0 + i, hkv * a.group + (r - i * a.group)};
}

__device__ __forceinline__ float natural_lse(float m2, float l) {
  return ((m2 == -__builtin_inff() ? 0.0f : m2) + __builtin_log2f(l)) * 0.69314718055994530942f;
}

// A merge of partials: the running maximum (log2 units), sum and O.  Where the
// maximum is -inf every partial so far saw no key, with sum and O zero, or only
// NaN scores, with both NaN; relative to 0 the weight of either is 2^-inf = 0, which
// leaves the zeros and keeps the NaN.
__device__ __forceinline__ float over_zero(float m) { return m == -__builtin_inff() ? 0.0f : m; }

constexpr int kPCoherent = 16;  // cache policy: the sc1 bit, coherent over the device's L2s
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

// O and LSE of row r of a sequence from its merged state, 4 dimensions.
template <bool BF16>
__device__ __forceinline__ void store_row(const PagedArgs& a, const PagedSeq& s, int hkv, int r, int dim,
                                          float m2, float l, float4v x) {
  const PagedRow pr = paged_row(a, s, hkv, r);
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  half4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = Elem<BF16>::round(x[e] * inv);
  *(half4*)(a.o + pr.token * a.ot + pr.head * a.oh + dim) = y;
  if (a.lse != nullptr && dim == 0) a.lse[(int64_t)pr.head * a.tokens + pr.token] = natural_lse(m2, l);
}

// Folds up to BATCH partials, step apart from i0, into (m, l, x): all their loads
// are in flight together.  `load` gives the record's (max, sum) and 4 dimensions.
template <int BATCH, class LoadML, class LoadO>
__device__ __forceinline__ void fold_partials(int i0, int step, int count, float& m, float& l, float4v& x,
                                              LoadML load_ml, LoadO load_o) {
  v2f ml[BATCH];
  float4v o[BATCH];
#pragma unroll
  for (int u = 0; u < BATCH; ++u) {
    const int i = min(i0 + u * step, count - 1);
    ml[u] = load_ml(i);
    o[u] = load_o(i);
  }
  float m_new = m;
#pragma unroll
  for (int u = 0; u < BATCH; ++u) {
    if (i0 + u * step >= count) {  // the last one again: no weight
      ml[u] = v2f{-__builtin_inff(), 0.0f};
      o[u] = (float4v)0.0f;
    }
    m_new = fmaxf(m_new, ml[u][0]);
  }
  const float f = __builtin_amdgcn_exp2f(m - over_zero(m_new));
  l *= f;
  x *= f;
#pragma unroll
  for (int u = 0; u < BATCH; ++u) {
    const float w = __builtin_amdgcn_exp2f(ml[u][0] - over_zero(m_new));
    l += w * ml[u][1];
    x += w * o[u];
  }
  m = m_new;
}

}  // namespace
}  // namespace fa
