// The weights that attention gave the rows of a paged cache: for each sequence, KV head
// and key j, the sum over the sequence's rows r that see it (token r / group of query head
// kv_head * group + r % group) of p_rj = exp(scale q_r k_j - lse_r), where lse_r is the row's
// log-sum-exp: the probabilities the attention used, computed again from Q and K.
//
//   S = Q K^T   rows on the M side of the MFMAs, keys on N: a lane has one key and
//               several rows, so that a key's sum over rows is a sum in the lane, and
//               over the lane groups once, at the end
//
// p = 2^(c s - lse log2 e), c = scale log2 e: no maximum is looked for, the lse is one already.
// Everything from S on is in 32 bits, and sums go by tiles of 32 rows (one accumulator over 2048
// rows was off by 1.4e-6 of a weight, twelve of the sum's own roundings).  Which rows a sum takes, and in which order, follows from
// the sizes and lengths: the same call gives the same bits.
//
// Two kernels: up to 32 rows (one generated token, a few drafted ones) K is the work, which
// streams through registers; more rows meet a block of keys that stays in registers.
#pragma once

#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include "fa_internal.h"
#include "fa_paged_units.h"

namespace fa {
namespace {

constexpr int kWTile = 32;    // keys of a wave's step: two 16-key pieces, each in one page
constexpr int kWBlock = 256;  // keys of a unit of the kernel for more rows

constexpr float kWLog2e = 1.4426950408889634f;

// The steps of STEP keys that hold keys some row sees, up to max_len: of every sequence, those of its
// KV heads.  And the blocks of 256 positions behind them.  Called by whole waves.
template <int STEP>
struct WeighLine {
  const WeighArgs& w;
  int lane;
  PagedSeq own;  // sequence `lane`
  __device__ __forceinline__ WeighLine(const WeighArgs& args, int ln) : w(args), lane(ln) { own = look(ln); }
  __device__ __forceinline__ PagedSeq look(int b) const {
    PagedSeq s = paged_seq(w.p, min(b, w.p.batch - 1), [](const int32_t* p) { return *p; });
    if (b >= w.p.batch) s.n = 0;
    return s;
  }
  __device__ __forceinline__ int steps(const PagedSeq& s) const {  // for each KV head
    return s.n > 0 ? (int)((unsigned)(min(s.keys, w.max_len) + STEP - 1) / STEP) : 0;
  }
  __device__ __forceinline__ int empty(const PagedSeq& s) const {
    return (int)((unsigned)(max(0, w.max_len - STEP * steps(s)) + kWBlock - 1) / kWBlock);
  }
  // Those of sequences b0 .. b0 + lane.
  __device__ __forceinline__ int prefix(int b0, bool behind) const {
    const PagedSeq s = b0 == 0 ? own : look(b0 + lane);
    return wave_prefix((b0 + lane < w.p.batch ? behind ? empty(s) : steps(s) : 0) * w.p.hkv);
  }
  __device__ __forceinline__ int total(bool behind) const {
    int sum = 0;
    for (int b0 = 0; b0 < w.p.batch; b0 += 64) sum += wave_bcast(prefix(b0, behind), 63);
    return uniform(sum);
  }
  // The sequence of number `at` (below the total), which becomes its number in the sequence.
  __device__ __forceinline__ int find(int& at, bool behind) const {
    for (int b0 = 0;; b0 += 64) {
      const int x = prefix(b0, behind);
      const uint64_t past = __builtin_amdgcn_ballot_w64(x > at);
      if (past != 0 || b0 + 64 >= w.p.batch) {
        const int l = past != 0 ? __builtin_ctzll(past) : 63;
        if (l > 0) at -= wave_bcast(x, l - 1);
        return uniform(min(b0 + l, w.p.batch - 1));
      }
      at -= wave_bcast(x, 63);
    }
  }
  // Zeros into block number `at` of those behind the keys, `threads` threads.
  __device__ __forceinline__ void clear(int at, int thread, int threads) const {
    const int b = find(at, true);
    const int block = (int)((unsigned)at / (unsigned)w.p.hkv), h = at - block * w.p.hkv;
    const int j0 = STEP * steps(scalar_seq(w.p, b)) + block * kWBlock;
    float* const out = w.out + b * w.sb + h * w.sh;
    for (int j = j0 + thread; j < min(j0 + kWBlock, w.max_len); j += threads) out[j] = 0.0f;
  }
};

// The tiles of all (sequence, KV head) end to end are a line, of which each of `waves` waves takes an
// equal stretch, whatever heads and sequences it covers: as many waves as run at once, or one for
// each tile.  K goes to registers, the next tile's under the current one's work.  (Runs of 8 tiles
// a wave, as the GPU got round to them, left a last round of half the waves: 88 us for 80 at 32 sequences
// of 4096 .. 8192 rows of 128, 8 KV heads.)
//
// Bound: K comes from HBM once, 403 MB in 79 us (5.1 TB/s, as fast as a copy moves bytes); at 8 bits
// 211 MB in 46 us with cold caches (4.5 TB/s), 36 where the 256 MB cache has part of it.  A token over a
// few thousand rows is latency, 5 us.
template <int D, bool BF16, bool FP8, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : 3) fa_paged_weigh_kernel(const WeighArgs w) {
  using E = Elem<BF16>;
  constexpr int R = 16 * NT;
  constexpr int KS = D / 32;             // contraction steps of S
  constexpr int KL = FP8 ? KS / 2 : KS;  // K loads of a 16-key piece
  const PagedArgs& a = w.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l16 = lane & 15;
  const int g4 = lane >> 4;
  const WeighLine<kWTile> line(w, lane);
  const int total = line.total(false);
  const int wv = uniform((int)blockIdx.x * kWaves + wave);
  const int waves = min(w.waves, total);
  if (wv >= waves) {  // blocks behind the keys
    if (!w.add && wv - waves < line.total(true)) line.clear(wv - waves, lane, 64);
    return;
  }
  int pos = (int)((int64_t)total * wv / waves);
  const int end = uniform((int)((int64_t)total * (wv + 1) / waves));

  while (pos < end) {
  int at = pos;
  const int b = line.find(at, false);
  const PagedSeq s = scalar_seq(a, b);
  const int tiles = uniform(line.steps(s));
  if (tiles == 0) return;  // (the lengths changed meanwhile)
  const int hkv = uniform((int)((unsigned)at / (unsigned)tiles));
  const int t_begin = uniform(at - hkv * tiles);
  const int t_stop = uniform(min(tiles, t_begin + end - pos));
  pos = uniform(pos + t_stop - t_begin);
  if (hkv >= a.hkv) return;

  // Keys some row sees end at `sees`.
  const int nrows = s.n * a.group;
  const int past = s.len - s.n;  // tokens before the new ones
  const int sees = s.n > 0 ? uniform(min(s.keys, w.max_len)) : 0;
  float* const out = w.out + b * w.sb + hkv * w.sh;
  const float c2 = a.negate_q ? -a.c : a.c;

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
        qf[nt][kk] = ok ? *(const half8*)(qp + dim) : (half8)(_Float16)0;
      }
      // Rows of LSE -inf and places without a row see no key: their products with one that is not finite may be
      // NaN.
      const float lse = ok ? w.lse[(int64_t)pr.head * a.tokens + pr.token] : -__builtin_inff();
      const int most = lse == -__builtin_inff() ? -1 : a.causal ? min(sees - 1, past + (pr.token - s.t0)) : sees - 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lse2[nt][i] = __shfl(lse * kWLog2e, 4 * g4 + i);
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
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float4v st = (float4v)0.0f;
#pragma unroll
          for (int kk = 0; kk < KS; ++kk) st = E::mfma16(qf[nt][kk], kf[p][kk], st);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i], c2, -lse2[nt][i]));
            acc[p] += key <= last[nt][i] ? y : 0.0f;
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
  }
}

// ---- more than 32 rows ------------------------------------------------------------
//
// A unit is 256 keys of one (sequence, KV head), a wave's 64 of them in its registers as the B
// operand of 32x32x16 MFMAs; the sequence's rows that see them come by, 64 at a time, through LDS
// (four buffers, loaded directly, two steps ahead; each row's -lse log2 e beside them), the
// probabilities of 32 rows between the MFMAs of the next 32.  Where units are many, each is a
// workgroup's; else their row tiles (under the causal rule a unit of new keys has fewer) are a line, of
// which each workgroup takes an equal stretch; the workgroups of a unit leave their sums, and the last
// of them to finish adds those up in their order (each unit's rows dealt to whole parts left a second
// round and idle CUs: at a prompt of 4096 tokens 116 us for 97, at five of 700 .. 2000 of 14 heads of
// 64 42 for 35; where the parts came to two whole rounds the line costs 4%).
//
// Bound: the matrix units, the exponentials and the sums share a SIMD's two waves.  The last 2048
// tokens of 8192, 32 heads of 128 on 8, are 120 GFLOP in 142 us (0.85 PFLOP/s), the matrix units 42%
// busy, 8-bit keys 136; rows loaded through registers, one step ahead, 154.
constexpr int kWRows = 64;      // rows of a tile, two of S
constexpr int kWMinTiles = 8;   // tiles a stretch has at least

// How many of a sequence's row tiles see its blocks of keys: `tiles` for those before block k0,
// where the new tokens begin; block k from there on is hidden from the first 4 group k - c
// (row r sees key j iff r >= (j - past) group).
struct WeighTiles {
  int tiles, k0, group;
  int64_t c;
  __device__ __forceinline__ WeighTiles(const PagedArgs& a, const PagedSeq& s) {
    const int past = s.len - s.n;  // tokens before the new ones
    group = a.group;
    tiles = (int)((unsigned)(s.n * a.group + kWRows - 1) / kWRows);
    k0 = a.causal ? max(0, (int)(((int64_t)past + kWBlock - 1) / kWBlock)) : INT32_MAX;
    const int64_t rows = (int64_t)past * a.group;
    c = rows > 0 ? (rows + kWRows - 1) / kWRows : -(-rows / kWRows);
  }
  // The first tile that sees block k, and all those of blocks before it (below 2^31 where there
  // are fewer units than workgroups).
  __device__ __forceinline__ int first(int k) const { return k < k0 ? 0 : (int)(4ll * group * k - c); }
  __device__ __forceinline__ int before(int k) const {
    if (k <= k0) return k * tiles;
    return (int)((int64_t)k0 * tiles + (k - k0) * (tiles + c) - 2ll * group * ((int64_t)k * (k - 1) - (int64_t)k0 * (k0 - 1)));
  }
};

template <int D>
__device__ __forceinline__ int weigh_swizzle(int r) {
  if constexpr (D == 64) return dense_swizzle(r);
  return r & 15;
}

template <int D, bool BF16, bool FP8>
__global__ void __launch_bounds__(kThreads, 2) fa_paged_weigh_chunk_kernel(const WeighArgs w) {
  using E = Elem<BF16>;
  constexpr int KK = D / 16;               // contraction steps of S
  constexpr int QL = kWRows * D * 2 / 1024 / kWaves;  // 1 KB loads of a wave's 16 rows
  constexpr int NS = 2 * KK;               // MFMAs of 32 rows
  constexpr int PF = 3;                    // Q operand reads run this many steps ahead
  // Tile t's rows are in buffer t % 4.  (Distinct objects, so that the compiler sees that loads in
  // flight into one do not touch those being read.)  Chunk c of 8 dimensions of row r is at
  // c ^ weigh_swizzle(r): 16 rows' chunks of one number are in 16 different places of the banks.
  __shared__ __attribute__((aligned(1024))) _Float16 q_lds0[kWRows * D];
  __shared__ __attribute__((aligned(1024))) _Float16 q_lds1[kWRows * D];
  __shared__ __attribute__((aligned(1024))) _Float16 q_lds2[kWRows * D];
  __shared__ __attribute__((aligned(1024))) _Float16 q_lds3[kWRows * D];
  __shared__ __attribute__((aligned(16))) float lse_lds[4][kWRows];
  __shared__ int scratch[kWaves];
  const PagedArgs& a = w.p;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wg = (int)blockIdx.x;
  // The line of row tiles and its workgroups, or one for each unit.  (The sequences are looked at again
  // for each unit, not kept in registers through its tiles.)
  auto length_of = [&](const WeighLine<kWBlock>& line, int b0) {  // of sequence b0 + lane
    const PagedSeq s = b0 == 0 ? line.own : line.look(b0 + line.lane);
    return s.n > 0 ? WeighTiles(a, s).before(line.steps(s)) * a.hkv : 0;
  };
  int total = 0, cuts = 0;
  {
    const WeighLine<kWBlock> line(w, threadIdx.x & 63);
    const int units = line.total(false);
    if (w.wgs > units) {
      for (int b0 = 0; b0 < a.batch; b0 += 64) total += wave_bcast(wave_prefix(length_of(line, b0)), 63);
      total = uniform(total);
      cuts = uniform(min(w.wgs, (int)((unsigned)total / kWMinTiles)));
      if (cuts >= kNumXcds) cuts &= -kNumXcds;
      if (cuts <= units) cuts = 0;
    }
    const int active = cuts > 0 ? cuts : units;
    if (wg >= active) {  // blocks behind the keys
      if (!w.add && wg - active < line.total(true)) line.clear(wg - active, threadIdx.x, kThreads);
      return;
    }
  }
  // Stretch number i is [start(i), start(i + 1)) of the line; an XCD's are next to each other, so that it
  // reads few heads' rows.
  auto start = [&](int i) { return (int)((int64_t)total * i / cuts); };
  auto holder = [&](int pos) { return (int)(((int64_t)(pos + 1) * cuts + total - 1) / total) - 1; };
  const int place = cuts >= kNumXcds ? (wg & (kNumXcds - 1)) * (cuts / kNumXcds) + wg / kNumXcds : wg;
  int pos = 0, end = 1;
  if (cuts > 0) {
    pos = uniform(start(place));
    end = uniform(start(place + 1));
  }
  while (pos < end) {
  // The unit, and its tiles [t0, t1) that are this workgroup's, at [u0, u1) of the line.
  int b, block, hkv, t0 = 0, t1, u0 = 0, u1 = 0;
  // What depends on the thread is derived for each unit from an opaque index, so that none of it is kept
  // in registers from one to the next.
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63, hi = lane >> 5, l32 = lane & 31;
  const WeighLine<kWBlock> line(w, lane);
  if (cuts > 0) {
    int before = 0;
    for (int b0 = 0;; b0 += 64) {
      const int x = wave_prefix(length_of(line, b0));
      const uint64_t past = __builtin_amdgcn_ballot_w64(before + x > pos);
      if (past != 0 || b0 + 64 >= a.batch) {
        const int l = past != 0 ? __builtin_ctzll(past) : 63;
        if (l > 0) before += wave_bcast(x, l - 1);
        b = uniform(min(b0 + l, a.batch - 1));
        break;
      }
      before += wave_bcast(x, 63);
    }
    u0 = before;
  } else {
    int at = wg;
    b = line.find(at, false);
    block = uniform((int)((unsigned)at / (unsigned)a.hkv));
    hkv = uniform(at - block * a.hkv);
  }
  const PagedSeq s = scalar_seq(a, b);
  const WeighTiles rows(a, s);
  if (cuts > 0) {
    const int blocks = line.steps(s), head = rows.before(blocks);
    if (head <= 0) return;  // (the lengths changed meanwhile)
    hkv = uniform((int)((unsigned)(pos - u0) / (unsigned)head));
    const int rel = pos - u0 - hkv * head;
    int lo = 0, hi_k = blocks;  // before(lo) <= rel < before(hi_k)
    while (hi_k - lo > 1) {
      const int mid = (lo + hi_k) / 2;
      if (rows.before(mid) <= rel) lo = mid;
      else hi_k = mid;
    }
    block = uniform(lo);
    u0 = uniform(u0 + hkv * head + rows.before(lo));
    u1 = uniform(u0 + rows.before(lo + 1) - rows.before(lo));
    t0 = pos - u0;
    t1 = min(u1, end) - u0;
    pos = uniform(min(u1, end));
    if (hkv >= a.hkv || t1 <= t0) return;
  } else {
    t1 = rows.tiles - rows.first(block);
    pos = end;
  }
  const int nrows = s.n * a.group;
  const int past = s.len - s.n;
  const int sees = min(s.keys, w.max_len);
  const int key0 = block * kWBlock;

  // This lane's two keys.
  const int key = key0 + 64 * wave + l32;
  half8 kf[2][KK];
  bool held[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int j = key + 32 * t;
    const int page = j < sees ? a.table[b * a.table_stride + (j >> a.page_shift)] : -1;
    held[t] = page >= 0 && page < a.num_pages;
    const int64_t off = j & ((1 << a.page_shift) - 1);
    const uint8_t* const row = a.k + page * a.kp + hkv * a.kh + off * a.kn + 16 * hi;
    const float ks = FP8 && held[t] ? scale_of(a.ks[page * a.ksp + hkv * a.ksh + off * a.ksn]) : 0.0f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if constexpr (FP8) {  // (16 codes are two steps' dimensions)
        if (kk & 1) continue;
        const uint4v c = held[t] ? *(const uint4v*)(row + 16 * kk) : (uint4v)0u;
        kf[t][kk] = dequantise8<BF16>(c[0], c[1], ks);
        kf[t][kk + 1] = dequantise8<BF16>(c[2], c[3], ks);
      } else {
        kf[t][kk] = held[t] ? *(const half8*)(row + 32 * kk) : (half8)(_Float16)0;
      }
    }
  }
  // Row r sees key j iff r >= (j - past) group, its token's number not below j - past: from row
  // `from` on this lane's first key, and 32 tokens later the second.
  const int64_t from64[2] = {(int64_t)(key - past) * a.group, (int64_t)(key + 32 - past) * a.group};
  int from[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) from[t] = a.causal ? (int)min(max(from64[t], (int64_t)0), (int64_t)nrows) : 0;
  // From this row on all of the unit's keys are seen.
  const int all_from = a.causal ? (int)min((int64_t)max(0, key0 + kWBlock - 1 - past) * a.group, (int64_t)nrows) : 0;

  const int tile0 = uniform(rows.first(block) + t0);
  const int count = uniform(max(0, t1 - t0));
  const float c2 = a.negate_q ? -a.c : a.c;
  // Loads of a tile's rows go through windows from its first row's token and the first head of the
  // group on, with offsets below 2^31 bytes (the launcher sees to it), whose factors have 24 bits.
  float lse_next;
  const int q_tok = 2 * (int)a.qt, q_head = 2 * (int)a.qh;  // in bytes
  const int tok_step = uniform((int)((unsigned)kWRows / (unsigned)a.group));
  const int rem_step = kWRows - tok_step * a.group;
  int ld_row = uniform(tile0 * kWRows);  // of the tile that is loaded next; its token and what is left
  int ld_tok = uniform((int)((unsigned)ld_row / (unsigned)a.group));
  int ld_rem = ld_row - ld_tok * a.group;
  // Offsets of the lane's rows: they follow from what is left of the tile's first token, which often is
  // the same for all tiles, and, of the last tile, from where the rows end (the last row again for those
  // behind it).
  int q_off[QL], lse_off = 0, aimed = -1;
  auto q_buf = [&](auto t_c) -> _Float16* {
    constexpr int B = decltype(t_c)::value % 4;
    return B == 0 ? q_lds0 : B == 1 ? q_lds1 : B == 2 ? q_lds2 : q_lds3;
  };
  auto load = [&](auto t_c) {  // (t_c: the tile's number, modulo 4)
    const int end = nrows - 1 - ld_row;
    if (ld_rem != aimed || end < kWRows - 1) {
      aimed = ld_rem;
      auto place = [&](int r, int& tok, int& head) {
        const int x = ld_rem + min(r, end);
        tok = (int)(((float)x + 0.5f) * a.inv_group);
        head = x - (int)__umul24(tok, a.group);
      };
      int tok, head;
#pragma unroll
      for (int u = 0; u < QL; ++u) {
        const int at = 1024 * u + 16 * lane, r = 16 * wave + at / (2 * D);
        place(r, tok, head);
        q_off[u] = __umul24(tok, q_tok) + __umul24(head, q_head) + 16 * (((at >> 4) & (D / 8 - 1)) ^ weigh_swizzle<D>(r));
      }
      place(lane, tok, head);
      lse_off = head * a.tokens + tok;
    }
    const float* const lse = w.lse + (int64_t)hkv * a.group * a.tokens + s.t0 + ld_tok;
    lse_next = lse[lse_off];
    fence_schedule();  // (the LSE is waited for first)
    const __amdgpu_buffer_rsrc_t rq =
        make_rsrc(a.q + (int64_t)(s.t0 + ld_tok) * a.qt + (int64_t)hkv * a.group * a.qh, INT32_MAX);
#pragma unroll
    for (int u = 0; u < QL; ++u) {
      int off = (QL * wave + u) * 512;
      asm volatile("" : "+s"(off));  // recomputed at each load, not kept in a register
      direct_load16(rq, (lds_void*)(q_buf(t_c) + off), q_off[u]);
    }
    ld_row += kWRows;
    ld_tok += tok_step;
    ld_rem += rem_step;
    if (ld_rem >= a.group) {
      ld_rem -= a.group;
      ++ld_tok;
    }
  };
  // Of rows of LSE -inf, which are left out, +inf; bit `buf` of `out_tiles` says that its tile has one (every
  // wave has all the tile's LSE).  Their products with a key that is not finite may be NaN.  Copies of the last row
  // behind it get a finite least, with which a score that the row itself makes 0, infinite or NaN stays so.
  int out_tiles = 0;
  auto store_lse = [&](int buf, int tile) {
    const bool out = lse_next == -__builtin_inff();
    const float nl = -lse_next * kWLog2e;
    const bool copy = tid > nrows - 1 - (tile0 + tile) * kWRows;
    if (tid < kWRows)
      lse_lds[buf][tid] = out ? __builtin_inff() : copy ? -FLT_MAX : nl == __builtin_inff() ? FLT_MAX : nl;
    out_tiles = uniform((out_tiles & ~(1 << buf)) | (__builtin_amdgcn_ballot_w64(out) != 0 ? 1 << buf : 0));
  };
  int q_base[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    q_base[kk] = l32 * D + 8 * ((FP8 ? 4 * (kk >> 1) + 2 * hi + (kk & 1) : 2 * kk + hi) ^ weigh_swizzle<D>(l32));
  auto read_q = [&](const _Float16* buf, int half, int kk) -> half8 {
    return *(const half8*)(buf + q_base[kk] + 32 * half * D);
  };
  float sum[2] = {0.0f, 0.0f};
  float16v st[2][2];
  // Half H of step i (I: modulo 4): the probabilities of these 32 rows, whose S is st[H], between the
  // MFMAs of the next 32's (behind the last tile: of what is there, for nobody).  Tile i + 3 is loaded
  // to where tile i - 1 was, straight to LDS.  MASK: 1 where keys may be hidden from rows, 2 where rows may be
  // left out as well (a variant of its own: that select in 1 too cost all steps 4 to 10%).
  auto half_step = [&](int i, auto i_t, auto half_t, auto mask_t) {
    constexpr int I = decltype(i_t)::value;
    constexpr int H = decltype(half_t)::value;
    constexpr int MASK = decltype(mask_t)::value;
    half8 qf[KK];
    const _Float16* const buf = q_buf(std::integral_constant<int, I + H>{});
    static_for<PF>([&](auto k_c) { qf[decltype(k_c)::value] = read_q(buf, 1 - H, decltype(k_c)::value); });
    float4v nl[4];
    auto read_lse = [&](int g) { return *(const float4v*)(lse_lds[I] + 32 * H + 8 * g + 4 * hi); };
    nl[0] = read_lse(0);
    const int row0 = (tile0 + i) * kWRows + 32 * H + 4 * hi;
    const int lim[2] = {from[0] - row0, from[1] - row0};
    float add[2] = {0.0f, 0.0f};
    fence_schedule();
    static_for<NS>([&](auto slot_c) {
      constexpr int slot = decltype(slot_c)::value;
      constexpr int kk = slot / 2, v = slot % 2;
      if constexpr (v == 0 && kk + PF < KK) qf[kk + PF] = read_q(buf, 1 - H, kk + PF);
      if constexpr (slot % (NS / 4) == 1 && slot / (NS / 4) < 3) nl[slot / (NS / 4) + 1] = read_lse(slot / (NS / 4) + 1);
      if constexpr (H == 0 && slot == NS / 4) {
        if (i + 2 < count) store_lse((I + 2) % 4, i + 2);
      }
      if constexpr (H == 0 && slot == NS / 2) {
        if (i + 3 < count) load(std::integral_constant<int, I + 3>{});
      }
      st[1 - H][v] = E::mfma(qf[kk], kf[v][kk], kk == 0 ? (float16v)0.0f : st[1 - H][v]);
      // Rows 8 g + 4 hi + r of the 32 in register 4 g + r.
      static_for<32>([&](auto e_c) {
        constexpr int e = decltype(e_c)::value;
        if constexpr (e * NS / 32 == slot) {
          constexpr int k = e & 1, x = e >> 1;
          float y = __builtin_amdgcn_exp2f(__builtin_fmaf(st[H][k][x], c2, nl[x >> 2][x & 3]));
          if constexpr (MASK != 0) y = 8 * (x >> 2) + (x & 3) >= lim[k] ? y : 0.0f;
          if constexpr (MASK == 2) {
            asm volatile("" : "+v"(y));
            y = nl[x >> 2][x & 3] != __builtin_inff() ? y : 0.0f;
          }
          add[k] += y;
          asm volatile("" : "+v"(add[k]));  // keeps the sum in this slot
        }
      });
      fence_schedule();
    });
    sum[0] += add[0];
    sum[1] += add[1];
  };
  if (count > 0) {
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    load(I0{});
    store_lse(0, 0);
    if (count > 1) {
      load(I1{});
      store_lse(1, 1);
    }
    if (count > 2) load(I2{});
    barrier_after_loads<0>();
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      st[0][v] = (float16v)0.0f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) st[0][v] = E::mfma(read_q(q_lds0, 0, kk), kf[v][kk], st[0][v]);
    }
    // Tiles before `all_from` hide a key from some row.
    const int hiding = uniform((int)((unsigned)(max(0, all_from - tile0 * kWRows) + kWRows - 1) / kWRows));
    auto step = [&](int i, auto i_t) {
      if (out_tiles >> decltype(i_t)::value & 1) {
        half_step(i, i_t, I0{}, std::integral_constant<int, 2>{});
        half_step(i, i_t, I1{}, std::integral_constant<int, 2>{});
      } else if (i < hiding) {
        half_step(i, i_t, I0{}, std::integral_constant<int, 1>{});
        half_step(i, i_t, I1{}, std::integral_constant<int, 1>{});
      } else {
        half_step(i, i_t, I0{}, std::integral_constant<int, 0>{});
        half_step(i, i_t, I1{}, std::integral_constant<int, 0>{});
      }
      // Tile i + 2 has landed, tile i + 3 need not have.
      if (i + 3 < count) barrier_after_loads<QL>();
      else barrier_after_loads<0>();
    };
    for (int i = 0;; i += 4) {
      step(i, I0{});
      if (i + 1 >= count) break;
      step(i + 1, I1{});
      if (i + 2 >= count) break;
      step(i + 2, I2{});
      if (i + 3 >= count) break;
      step(i + 3, I3{});
      if (i + 4 >= count) break;
    }
  }
  // Thread: a key of its wave's 64.
  sum[0] = halves_sum(sum[0]);
  sum[1] = halves_sum(sum[1]);
  const bool mine = hi ? held[1] : held[0];
  const float x = mine ? (hi ? sum[1] : sum[0]) : 0.0f;
  const int j = key0 + tid;
  float* const out = w.out + b * w.sb + hkv * w.sh + j;
  if (cuts == 0 || (t0 == 0 && u0 + t1 == u1)) {
    if (j < w.max_len && (mine || !w.add)) *out = w.add ? *out + x : x;
    barrier_after_loads<63>();  // the next unit's rows go into these buffers
    continue;
  }
  // A record for each workgroup's piece of a unit that it begins and of one that it does not, and one of
  // what the first piece's finds there; coherent over the L2s.
  const __amdgpu_buffer_rsrc_t rec = make_rsrc(w.partial, 3 * w.wgs * kWBlock * 4);
  auto at_record = [&](int r) { return (r * kWBlock + tid) * 4; };
  const int record = 2 * place + (t0 == 0 ? 1 : 0);
  const int from_place = uniform(holder(u0)), pieces = uniform(holder(u1 - 1)) - from_place + 1;
  __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), rec, at_record(record), 0, kPCoherent);
  if (t0 == 0 && w.add) {
    const float before = j < w.max_len ? *out : 0.0f;
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, before), rec, at_record(2 * w.wgs + place), 0,
                                          kPCoherent);
  }
  // (see last_to_finish, fa_paged_units.h: whoever sets the last flag sees them all)
  const __amdgpu_buffer_rsrc_t rf = make_rsrc(w.flags, 2 * w.wgs * 8);
  auto piece = [&](int p) { return 2 * (from_place + p) + (p == 0 ? 1 : 0); };
  wait_loads<0>();
  __syncthreads();
  if (tid == 0) {
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, w.mark), rf, record * 8, 0, kPCoherent);
    wait_loads<0>();
  }
  __syncthreads();
  bool set = true;
  for (int p = tid; p < pieces; p += kThreads)
    set = set && __builtin_bit_cast(uint64_t, __builtin_amdgcn_raw_buffer_load_b64(rf, piece(p) * 8, 0, kPCoherent)) ==
                     w.mark;
  const bool all = __builtin_amdgcn_ballot_w64(!set) == 0;
  if (lane == 0) scratch[wave] = all;
  __syncthreads();
  const bool last = scratch[0] && scratch[1] && scratch[2] && scratch[3];
  __syncthreads();
  if (!last) continue;
  // Two that both get here store the same values.
  auto get = [&](int r) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rec, at_record(r), 0, kPCoherent));
  };
  float y = 0.0f;
  for (int p = 0; p < pieces; p += 8) {
    float z[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) z[u] = get(piece(min(p + u, pieces - 1)));
#pragma unroll
    for (int u = 0; u < 8; ++u) y += p + u < pieces ? z[u] : 0.0f;
  }
  if (w.add) y += get(2 * w.wgs + from_place);
  if (j < w.max_len && (mine || !w.add)) *out = y;
  }
}

}  // namespace

template <int D, bool BF16, bool FP8>
void launch_weigh_chunk(const WeighArgs& a, int64_t grid, hipStream_t stream) {
  hipLaunchKernelGGL((fa_paged_weigh_chunk_kernel<D, BF16, FP8>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
}

template <int D, bool BF16, bool FP8>
void launch_weigh_few(const WeighArgs& a, int rows, int64_t grid, hipStream_t stream) {
  if (rows == 16)
    hipLaunchKernelGGL((fa_paged_weigh_kernel<D, BF16, FP8, 1>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((fa_paged_weigh_kernel<D, BF16, FP8, 2>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
}

}  // namespace fa
