// Writing new tokens' K and V rows into the pages of a cache, and reading a
// batch's rows back.  Both are bound by memory: a write reads a row once and
// writes it once, a read writes the padded tensor once.
//
// 8-bit rows.  A row (one token, one head; D values x) is held as e4m3 codes q and
// one scale 2^e, x ~ q 2^e, e the smallest exponent with max |x| <= 448 2^e
// over the row's finite values (e4m3's largest value is 448), from -126 to the
// largest with which 448 2^e is finite in the rows' 16-bit type (7 for float16,
// 119 for bfloat16; larger values are stored as that).  A power of two costs
// e4m3 nothing (its own exponent takes it up, and no finite row loses more than
// the binade of range by which 448 2^e exceeds its maximum) and makes q 2^e a
// 16-bit number exactly: codes have 4 significant bits, and a float16 row's are
// multiples of float16's smallest step, as the row is.  So the attention feeds
// its matrix instructions q 2^e unrounded, and one conversion instruction takes
// the scale along.  An infinity or NaN is stored as NaN (e4m3 has no infinity).
// The only rounding is x 2^-e to e4m3, to nearest even: at most 2^-4 of a value
// not below 2^(e-6), 2^(e-10) below.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_kernel_common.h"
#include "fa_paged.h"

namespace fa {
namespace {

typedef unsigned uint2v __attribute__((ext_vector_type(2)));

constexpr int kCacheThreads = 256;

__device__ __forceinline__ int load_plain(const int32_t* p) { return *p; }

// 8 consecutive values of a row as 8 codes, given its scale exponent.
template <bool BF16>
__device__ __forceinline__ uint2v quantise8(half8 x, int e) {
  const float inv = __builtin_bit_cast(float, (127 - e) << 23);  // 2^-e; e in [-126, 119]
  int w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float y[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float f = Elem<BF16>::to_f32(x[i + u]);
      // |f| < inf fails for NaN too
      y[u] = __builtin_fabsf(f) < __builtin_inff() ? fminf(fmaxf(f * inv, -448.0f), 448.0f)
                                                   : __builtin_nanf("");
    }
    if (i & 2) w[i >> 2] = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w[i >> 2], true);
    else w[i >> 2] = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w[i >> 2], false);
  }
  return uint2v{(unsigned)w[0], (unsigned)w[1]};
}

// Thread layout of both kernels: D / 8 lanes a row, 16 bytes of a 16-bit row each.
template <int D, bool BF16, bool FP8>
__global__ void __launch_bounds__(kCacheThreads) fa_paged_write_kernel(const PagedArgs a) {
  constexpr int LANES = D / 8;
  constexpr int ROWS = kCacheThreads / LANES;
  const int part = threadIdx.x % LANES;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;  // (token, head, K or V)
  const int64_t rows = (int64_t)a.tokens * a.hkv * 2;
  if (row >= rows) return;  // whole rows, whose lanes alone exchange values
  const int th = (int)(row >> 1);
  const bool is_v = row & 1;
  const int t = th / a.hkv;
  const int h = th - t * a.hkv;
  int b = t;
  if (a.cu != nullptr) {  // the last b with cu[b] <= t
    int lo = 0, hi = a.batch;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid + 1] <= t) lo = mid + 1;
      else hi = mid;
    }
    b = lo;
  }
  if (b >= a.batch) return;  // behind the last sequence
  const PagedSeq s = paged_seq(a, b, load_plain);
  const int i = t - s.t0;
  const int pos = s.len - s.n + i;
  if (i < 0 || i >= s.n || pos < 0 || pos >= s.keys) return;
  const int page = a.table[b * a.table_stride + (pos >> a.page_shift)];
  if (page < 0 || page >= a.num_pages) return;
  const int r = pos & ((1 << a.page_shift) - 1);
  const half8 x = is_v ? *(const half8*)(a.v_new + t * a.vnt + h * a.vnh + 8 * part)
                       : *(const half8*)(a.k_new + t * a.knt + h * a.knh + 8 * part);
  uint8_t* const dst = is_v ? a.v + page * a.vp + h * a.vh + r * a.vn
                            : a.k + page * a.kp + h * a.kh + r * a.kn;
  if constexpr (!FP8) {
    *(half8*)(dst + 16 * part) = x;
  } else {
    float m = 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float f = __builtin_fabsf(Elem<BF16>::to_f32(x[u]));
      m = fmaxf(m, f < __builtin_inff() ? f : 0.0f);
    }
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    // m = 1.f 2^k: 448 2^e >= m first at e = k - 8 where 1.f <= 1.75, else k - 7.
    const unsigned bits = __builtin_bit_cast(unsigned, m);
    const int k = (int)(bits >> 23) - 127;
    const int e = clamp_int(k - ((bits & 0x7fffff) <= 0x600000 ? 8 : 7), -126, BF16 ? 119 : 7);
    *(uint2v*)(dst + 8 * part) = quantise8<BF16>(x, e);
    if (part == 0) {
      uint8_t* const sc = is_v ? a.vs + page * a.vsp + h * a.vsh + r * a.vsn
                               : a.ks + page * a.ksp + h * a.ksh + r * a.ksn;
      *sc = (uint8_t)(e + 127);
    }
  }
}

// Rows of [batch, hkv, max_len, D] out of the pages; zeros where a sequence
// has no token or its page is gone.
template <int D, bool BF16, bool FP8>
__global__ void __launch_bounds__(kCacheThreads) fa_paged_read_kernel(const PagedArgs a) {
  constexpr int LANES = D / 8;
  constexpr int ROWS = kCacheThreads / LANES;
  const int part = threadIdx.x % LANES;
  const int j = (int)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (j >= a.max_len) return;
  const int h = (int)blockIdx.y % a.hkv;
  const int b = (int)blockIdx.y / a.hkv;
  const bool is_v = blockIdx.z != 0;
  half8 x = (half8)(_Float16)0;
  if (j < a.lens[b] && (j >> a.page_shift) < a.max_pages) {
    const int page = a.table[b * a.table_stride + (j >> a.page_shift)];
    if (page >= 0 && page < a.num_pages) {
      const int r = j & ((1 << a.page_shift) - 1);
      const uint8_t* const src = is_v ? a.v + page * a.vp + h * a.vh + r * a.vn
                                      : a.k + page * a.kp + h * a.kh + r * a.kn;
      if constexpr (!FP8) {
        x = *(const half8*)(src + 16 * part);
      } else {
        const uint8_t* const sc = is_v ? a.vs + page * a.vsp + h * a.vsh + r * a.vsn
                                       : a.ks + page * a.ksp + h * a.ksh + r * a.ksn;
        const uint2v w = *(const uint2v*)(src + 8 * part);
        x = dequantise8<BF16>(w[0], w[1], scale_of(*sc));
      }
    }
  }
  _Float16* const dst = is_v ? a.v_out : a.k_out;
  *(half8*)(dst + (((int64_t)b * a.hkv + h) * a.max_len + j) * D + 8 * part) = x;
}

}  // namespace

int launch_paged_write(const PagedArgs& a, int head_dim, hipStream_t stream) {
  const int64_t rows = (int64_t)a.tokens * a.hkv * 2;
  const int per = kCacheThreads / (head_dim / 8);
  const dim3 grid((unsigned)((rows + per - 1) / per));
#define FA_WRITE(D, BF, F8) \
  hipLaunchKernelGGL((fa_paged_write_kernel<D, BF, F8>), grid, dim3(kCacheThreads), 0, stream, a)
#define FA_WRITE_D(D)                                             \
  if (a.ks != nullptr) {                                          \
    if (a.bf16) FA_WRITE(D, true, true); else FA_WRITE(D, false, true);   \
  } else {                                                        \
    FA_WRITE(D, false, false); /* a copy: the type does not matter */     \
  }
  if (head_dim == 64) { FA_WRITE_D(64) } else { FA_WRITE_D(128) }
#undef FA_WRITE_D
#undef FA_WRITE
  return 0;
}

int launch_paged_read(const PagedArgs& a, int head_dim, hipStream_t stream) {
  const int per = kCacheThreads / (head_dim / 8);
  const dim3 grid((unsigned)((a.max_len + per - 1) / per), (unsigned)(a.batch * a.hkv), 2);
#define FA_READ(D, BF, F8) \
  hipLaunchKernelGGL((fa_paged_read_kernel<D, BF, F8>), grid, dim3(kCacheThreads), 0, stream, a)
#define FA_READ_D(D)                                              \
  if (a.ks != nullptr) {                                          \
    if (a.bf16) FA_READ(D, true, true); else FA_READ(D, false, true);     \
  } else {                                                        \
    FA_READ(D, false, false);                                     \
  }
  if (head_dim == 64) { FA_READ_D(64) } else { FA_READ_D(128) }
#undef FA_READ_D
#undef FA_READ
  return 0;
}

}  // namespace fa
