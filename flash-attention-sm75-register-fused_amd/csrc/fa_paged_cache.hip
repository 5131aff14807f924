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

#include <algorithm>

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

// Maximum over the D / 8 lanes of a row (8 or 16, aligned): xor 1, xor 2, then the
// mirrored half and the mirrored row, whose quads agree already.
template <int LANES>
__device__ __forceinline__ float row_lanes_max(float x) {
  auto step = [](float v, int other) { return fmaxf(v, __builtin_bit_cast(float, other)); };
#define FA_DPP(V, CTRL) __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, V), CTRL, 0xf, 0xf, true)
  x = step(x, FA_DPP(x, 0xb1));   // quad_perm [1, 0, 3, 2]
  x = step(x, FA_DPP(x, 0x4e));   // quad_perm [2, 3, 0, 1]
  x = step(x, FA_DPP(x, 0x141));  // row_half_mirror
  if constexpr (LANES == 16) x = step(x, FA_DPP(x, 0x140));  // row_mirror
#undef FA_DPP
  return x;
}

// D / 8 lanes a row, 16 bytes of a 16-bit row each; a thread takes its part of K and V of
// kWriteHeads heads of one token.  The rows are asked for first: where they go takes
// three dependent reads (cu_seqlens, the sequence's entries, its page), which run
// under them, once for all the token's rows of the thread.  8000 tokens of 8 heads
// d128 bfloat16 to 8 bits, 49 MB: 17.5 us with a row a thread and a search of cu_seqlens
// for each, 13.4 so (3.7 TB/s; with one head a thread 14.2, with four 13.5).
constexpr int kWriteHeads = 2;
template <int D, bool BF16, bool FP8>
__global__ void __launch_bounds__(kCacheThreads) fa_paged_write_kernel(const PagedArgs a) {
  constexpr int LANES = D / 8;
  constexpr int TOKENS = kCacheThreads / LANES;
  constexpr int WAVE_TOKENS = 64 / LANES;
  const int lane = threadIdx.x & 63;
  const int part = lane % LANES;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int t_wave = (int)blockIdx.x * TOKENS + wave * WAVE_TOKENS;
  if (t_wave >= a.tokens) return;
  const int t = t_wave + lane / LANES;
  const int tr = min(t, a.tokens - 1);
  const int h0 = (int)blockIdx.y * kWriteHeads;
  half8 x[kWriteHeads][2];
#pragma unroll
  for (int u = 0; u < kWriteHeads; ++u) {
    const int h = min(h0 + u, a.hkv - 1);
    x[u][0] = *(const half8*)(a.k_new + tr * a.knt + h * a.knh + 8 * part);
    x[u][1] = *(const half8*)(a.v_new + tr * a.vnt + h * a.vnh + 8 * part);
  }
  // The token's sequence: as many as end at or before it (cu_seqlens rises).
  int b = t;
  if (a.cu != nullptr) {
    b = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      const int end = b0 + lane < a.batch ? a.cu[b0 + lane + 1] : INT32_MAX;
#pragma unroll
      for (int u = 0; u < WAVE_TOKENS; ++u) {
        const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(end <= t_wave + u));
        if (lane / LANES == u) b += n;
      }
    }
  }
  if (t >= a.tokens || b >= a.batch) return;  // behind the last sequence
  const PagedSeq s = paged_seq(a, b, load_plain);
  const int i = t - s.t0;
  const int pos = s.len - s.n + i;
  if (i < 0 || i >= s.n || pos < 0 || pos >= s.keys) return;
  const int page = a.table[b * a.table_stride + (pos >> a.page_shift)];
  if (page < 0 || page >= a.num_pages) return;
  const int r = pos & ((1 << a.page_shift) - 1);
#pragma unroll
  for (int u = 0; u < kWriteHeads; ++u) {
    const int h = h0 + u;
    if (h >= a.hkv) break;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const half8 y = x[u][kv];
      uint8_t* const dst = kv ? a.v + page * a.vp + h * a.vh + r * a.vn : a.k + page * a.kp + h * a.kh + r * a.kn;
      if constexpr (!FP8) {
        *(half8*)(dst + 16 * part) = y;
      } else {
        float m = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = __builtin_fabsf(Elem<BF16>::to_f32(y[e]));
          m = fmaxf(m, f < __builtin_inff() ? f : 0.0f);
        }
        m = row_lanes_max<LANES>(m);
        // m = 1.f 2^k: 448 2^e >= m first at e = k - 8 where 1.f <= 1.75, else k - 7.
        const unsigned bits = __builtin_bit_cast(unsigned, m);
        const int k = (int)(bits >> 23) - 127;
        const int e = clamp_int(k - ((bits & 0x7fffff) <= 0x600000 ? 8 : 7), -126, BF16 ? 119 : 7);
        *(uint2v*)(dst + 8 * part) = quantise8<BF16>(y, e);
        if (part == 0) {
          uint8_t* const sc = kv ? a.vs + page * a.vsp + h * a.vsh + r * a.vsn
                                 : a.ks + page * a.ksp + h * a.ksh + r * a.ksn;
          *sc = (uint8_t)(e + 127);
        }
      }
    }
  }
}

// Rows of [batch, hkv, max_len, D] out of the pages; zeros where a sequence
// has no token or its page is gone.  D / 8 lanes a row, 16 bytes of the output each; a
// thread has one row, whose reads depend on each other (length, page, row), and it is the
// many waves that keep the memory busy: 4 sequences to 8192 tokens of 8 heads d128, 235 MB,
// 46.6 us (5.0 TB/s, what a large copy reaches); 7 to 8191 of 2 heads d64 8 bits, 38 MB,
// 8.6 us (4.4 TB/s).
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
  const int per = kCacheThreads / (head_dim / 8);
  const dim3 grid((unsigned)((a.tokens + per - 1) / per), (unsigned)((a.hkv + kWriteHeads - 1) / kWriteHeads));
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

int launch_paged_read(const PagedArgs& args, int head_dim, hipStream_t stream) {
  constexpr int kGridY = 65535;
  const int per = kCacheThreads / (head_dim / 8);
  // Whole sequences, as many as have their heads in one dimension of the grid, in a launch; of
  // more heads than that (2^16 at most) one sequence, in two.  (As one grid, heads running on
  // along z, every read paid for it: 38 MB of 8 bits 8.9 us, so 8.6, 235 MB 47.3, so 46.8.)
  const int seqs = std::max(1, std::min(args.batch, kGridY / args.hkv));
  const int heads = std::min(args.hkv, kGridY);
  for (int b0 = 0; b0 < args.batch; b0 += seqs) {
    for (int h0 = 0; h0 < args.hkv; h0 += heads) {
      PagedArgs a = args;
      a.batch = std::min(seqs, args.batch - b0);
      a.hkv = std::min(heads, args.hkv - h0);
      a.lens += b0;
      a.table += b0 * a.table_stride;
      a.k += h0 * a.kh;
      a.v += h0 * a.vh;
      if (a.ks != nullptr) {
        a.ks += h0 * a.ksh;
        a.vs += h0 * a.vsh;
      }
      const int64_t row = ((int64_t)b0 * args.hkv + h0) * a.max_len;
      a.k_out += row * head_dim;
      a.v_out += row * head_dim;
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
    }
  }
  return 0;
}

}  // namespace fa
