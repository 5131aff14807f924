// The weights that attention gave the rows of a paged cache: for each sequence, KV head
// and key j, the sum over the sequence's rows r that see it (token r / group of query head
// kv_head * group + r % group) of p_rj = exp(scale q_r k_j - lse_r), where lse_r is the row's
// log-sum-exp: the probabilities the attention used, computed again from Q and K.
//
//   S = Q K^T   rows on the M side of 16x16x32 MFMAs, keys on N: a lane has one key
//               of a 16-key piece and four rows of each 16, so that a key's sum over
//               rows is a sum in the lane and, once a tile, over the four lane groups
//
// p = 2^(c s - lse log2 e), c = scale log2 e: no maximum is looked for, the lse is one already.
// Everything from S on is in 32 bits.  Each key has one owner, which adds its rows' terms in
// their order: the same call gives the same bits.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_paged_units.h"

namespace fa {
namespace {

constexpr int kWTile = 32;  // keys of a wave's step: two 16-key pieces, each in one page

// A row's log-sum-exp in log2 units.  -inf (a row that saw no key) as +inf: it gives
// every key 2^-inf = 0.
__device__ __forceinline__ float weigh_lse2(float lse) {
  return lse == -__builtin_inff() ? __builtin_inff() : lse * 1.4426950408889634f;
}

// A wave takes `run` tiles of one (sequence, KV head): K goes to registers, the next
// tile's under the current one's work.  Runs are dealt by their place in the sequence,
// those of all sequences and heads before the next, so that what lies behind the shorter
// sequences' ends is dealt last.
template <int D, bool BF16, bool FP8, int NT>
__global__ void __launch_bounds__(kThreads) fa_paged_weigh_kernel(const WeighArgs w) {
  using E = Elem<BF16>;
  constexpr int R = 16 * NT;
  constexpr int KS = D / 32;             // contraction steps of S
  constexpr int KL = FP8 ? KS / 2 : KS;  // K loads of a 16-key piece
  const PagedArgs& a = w.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l16 = lane & 15;
  const int g4 = lane >> 4;
  const int pairs = a.batch * a.hkv;
  const unsigned item = (unsigned)blockIdx.x * kWaves + wave;
  const int at = uniform((int)(item / (unsigned)pairs));
  const int bh = uniform((int)(item - (unsigned)at * pairs));
  const int tiles = (int)((unsigned)(w.max_len + kWTile - 1) / kWTile);
  const int t_begin = at * w.run;
  if (t_begin >= tiles) return;
  const int b = uniform((int)((unsigned)bh / (unsigned)a.hkv));
  const int hkv = bh - b * a.hkv;
  const PagedSeq s = scalar_seq(a, b);
  const int t_end = min(t_begin + w.run, tiles);

  // Keys some row sees end at `sees`; those before `full` every row sees.
  const int nrows = s.n * a.group;
  const int past = s.len - s.n;  // tokens before the new ones
  const int sees = s.n > 0 ? uniform(min(s.keys, w.max_len)) : 0;
  const int full = a.causal ? uniform(clamp_int(past + 1, 0, sees)) : sees;
  const int t_stop = uniform(clamp_int((sees + kWTile - 1) / kWTile, t_begin, t_end));
  float* const out = w.out + b * w.sb + hkv * w.sh;
  const float c2 = a.c;

  // Rows rb R .. + R - 1: their Q, and of each of the lane's four rows of a 16 its lse
  // and the last key it sees.
  const int blocks = (nrows + R - 1) / R;
  half8 qf[NT][KS];
  float lse2[NT][4];
  int last[NT][4];
  auto load_rows = [&](int rb) {
    const PagedRows row_of(a, s, hkv, rb * R);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int c = 16 * nt + l16;
      const bool ok = rb * R + c < nrows;
      const PagedRow pr = row_of(ok ? c : 0);
      const _Float16* const qp = a.q + pr.token * a.qt + pr.head * a.qh;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        // (the dimensions of a K row's bytes, see fa_paged_attn.h)
        const int dim = FP8 ? 64 * (kk >> 1) + 16 * g4 + 8 * (kk & 1) : 32 * kk + 8 * g4;
        const half8 x = *(const half8*)(qp + dim);
        qf[nt][kk] = ok ? (a.negate_q ? negate16(x) : x) : (half8)(_Float16)0;
      }
      const float lse = ok ? weigh_lse2(w.lse[(int64_t)pr.head * a.tokens + pr.token]) : __builtin_inff();
      const int most = !ok ? -1 : a.causal ? min(sees - 1, past + (pr.token - s.t0)) : sees - 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lse2[nt][i] = __shfl(lse, 4 * g4 + i);
        last[nt][i] = __shfl(most, 4 * g4 + i);
      }
    }
  };

  struct Tile {
    int rows[2];  // keys of the two pieces
    uint4v k[2][KL];
    unsigned ks[2];
  };
  const int k_off = l16 * (int)a.kn + 16 * g4;
  const int32_t* const entries = a.table + b * a.table_stride;
  const uint8_t* const kh = a.k + hkv * a.kh;
  auto look_up = [&](int t, int (&e)[2]) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
      e[p] = load_scalar(entries + min((t * kWTile + 16 * p) >> a.page_shift, a.max_pages - 1));
  };
  // (a piece in no page or past the keys reads through an empty window)
  auto load = [&](int t, const int (&e)[2], Tile& x) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int key = t * kWTile + 16 * p;
      const bool paged = e[p] >= 0 && e[p] < a.num_pages;
      x.rows[p] = uniform(paged && t < t_stop ? clamp_int(sees - key, 0, 16) : 0);
      const int64_t page = paged ? e[p] : 0;
      const int off = key & ((1 << a.page_shift) - 1);
      const __amdgpu_buffer_rsrc_t rk = make_rsrc(kh + page * a.kp + off * a.kn, x.rows[p] * (int)a.kn);
#pragma unroll
      for (int i = 0; i < KL; ++i)
        x.k[p][i] = __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + 64 * i, 0, 0));
      if constexpr (FP8) {
        const __amdgpu_buffer_rsrc_t rs =
            make_rsrc(a.ks + page * a.ksp + hkv * a.ksh + off * a.ksn, x.rows[p] * (int)a.ksn);
        x.ks[p] = __builtin_amdgcn_raw_buffer_load_b8(rs, l16 * (int)a.ksn, 0, 0);
      }
    }
  };
  auto step = [&](int t, const Tile& x) {
    float acc[2] = {0.0f, 0.0f};
    half8 kf[2][KS];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        if constexpr (FP8) {
          const uint4v c = x.k[p][kk / 2];
          const float ks = scale_of(x.ks[p]);
          kf[p][kk] = kk & 1 ? dequantise8<BF16>(c[2], c[3], ks) : dequantise8<BF16>(c[0], c[1], ks);
        } else {
          kf[p][kk] = __builtin_bit_cast(half8, x.k[p][kk]);
        }
      }
    for (int rb = 0; rb < blocks; ++rb) {
      if (blocks > 1) load_rows(rb);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int key = t * kWTile + 16 * p + l16;
        const bool masked = (t + 1) * kWTile > full || x.rows[p] < 16;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float4v st = (float4v)0.0f;
#pragma unroll
          for (int kk = 0; kk < KS; ++kk) st = E::mfma16(qf[nt][kk], kf[p][kk], st);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float y = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i], c2, -lse2[nt][i]));
            if (masked) y = key <= last[nt][i] ? y : 0.0f;
            acc[p] += y;
          }
        }
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      acc[p] += __shfl_xor(acc[p], 16);
      acc[p] += __shfl_xor(acc[p], 32);
      if (x.rows[p] == 0) acc[p] = 0.0f;  // (in no page)
    }
    // Lanes 0 .. 31 have the tile's keys.
    const int j = t * kWTile + lane;
    const float y = lane < 16 ? acc[0] : acc[1];
    const int rows = lane < 16 ? x.rows[0] : x.rows[1];
    if (lane < kWTile && j < w.max_len) {
      if (!w.add) out[j] = y;
      else if (l16 < rows) out[j] += y;
    }
  };

  if (t_begin < t_stop) {
    int e[2];
    Tile xa, xb;
    look_up(t_begin, e);
    load(t_begin, e, xa);
    look_up(t_begin + 1, e);
    if (blocks <= 1) load_rows(0);
    int t = t_begin;
    for (; t + 1 < t_stop; t += 2) {
      load(t + 1, e, xb);
      look_up(t + 2, e);
      step(t, xa);
      load(t + 2, e, xa);
      look_up(t + 3, e);
      step(t + 1, xb);
    }
    if (t < t_stop) step(t, xa);
  }
  if (!w.add) {
    for (int j = t_stop * kWTile + lane; j < min(t_end * kWTile, w.max_len); j += 64) out[j] = 0.0f;
  }
}

}  // namespace

template <int D, bool BF16, bool FP8>
void launch_weigh_few(const WeighArgs& a, int rows, int64_t grid, hipStream_t stream) {
  if (rows == 16)
    hipLaunchKernelGGL((fa_paged_weigh_kernel<D, BF16, FP8, 1>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((fa_paged_weigh_kernel<D, BF16, FP8, 2>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
}

}  // namespace fa
