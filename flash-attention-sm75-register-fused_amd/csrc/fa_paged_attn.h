// Attention of new tokens over a paged cache, for units of at most 32 query
// columns: one generated token of every sequence, or a few drafted ones.
//
// A unit is one (sequence, KV head, block of 16 NT query columns); column c of
// the block is row r = 16 NT rb + c of the sequence's n * group rows, row r being
// token r / group of query head kv_head * group + r % group.  All of them read
// the same K and V rows, which is the work: streaming those from HBM once.
//
//   S^T = K Q^T     keys on the M side of 16x16x32 MFMAs, columns on N
//   O^T = V^T P^T   P stays in the registers S^T left it in (the key order
//                   inside a 32-key step is a permutation shared by P and V)
//
// 16x16x32 and not 32x32x16, as the other decode kernel has it: a K operand
// read is then 16 rows of 64 bytes, and 16 consecutive keys lie in one page
// whatever the page size (16 or more), so each read goes through one buffer
// window whose base is scalar; and up to 16 columns cost half the matrix time.
//
// The four waves of a workgroup take every fourth 32-key tile of its key range
// and run independently; their (max, sum, O) meet in LDS at the end.
//
// Softmax: running maximum per column, raised when some score outgrew it by more
// than 2^kRescaleLog2 (the sums and O share the stale maximum, so nothing else
// changes); sums of the unrounded P in 32 bits; P rounded to the 16-bit type for
// the second product, at most half a step of it each.
//
// The plan.  The units of one class of KV heads (every classes-th head, so that
// the workgroups of one XCD share heads) are laid end to end as a line of 32-key
// tiles, and each of the class's workgroups takes an equal stretch of the line,
// whatever mixture of sequences it covers: a batch of very different lengths
// keeps every CU busy to the end.  (Units that are all equally long are cut each for
// itself instead, see PagedStretch.)  A unit cut by a stretch's border leaves
// partials (O, max, sum) in the workspace, at most two for each workgroup.  Where
// they are few bytes the unit's last workgroup to finish merges them, else
// a second kernel does.  Stretches follow from the lengths alone, and partials
// are merged in order, so the same call gives the same bits.
//
// What bounds it: HBM where there are many keys (32 sequences of 4096 to 8192 keys, 8 KV
// heads d128, 807 MB: 130 us, 6.2 TB/s; 8 bits, 406 MB: 73 us, 5.6 TB/s; 4 tokens over 131072
// keys 8 bits: 52 us with its merge kernel, 5.2 TB/s), else the chain of one workgroup (its
// plan, two tiles a wave, two merges: one token of 4097 keys, 2 KV heads d64, 8.7 us).
// 8-bit tiles cost conversions and LDS stores, whose instructions are not what bounds them:
// laid out without the stores' bank conflicts, or with deeper loads, they took as long.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_paged_units.h"

namespace fa {
namespace {

constexpr int kPTile = 32;       // keys of a wave's tile
constexpr int kPMinTiles = 8;    // tiles a stretch is not cut below (but see PagedStretch)
// Another unit's cost, in tiles (us without and with: 4 sequences of 2048 to 4096 keys d128
// 8 bits 19.6 / 16.0, 32 of 4096 to 8192 132.0 / 130.5, 8 bits 68.8 / 68.0, 16 of 16384 to
// 32768 d64 36.6 / 37.2; 8 of 8192 each d128, where it does not count, 45.2, with it 47.8).
constexpr int kPAhead = 3;

// Whether a unit's last workgroup merges its partials: one workgroup reads them
// at about 50 bytes/ns, and the second kernel costs a launch 2.5 us where it has
// nothing to do (16 sequences to 32768 keys d64 39.3 -> 36.9 us, 8 bits 32.9 -> 30.3,
// without it).
constexpr int kPMergeBytes = 256 << 10;
__host__ __device__ constexpr bool paged_merges_itself(int pieces, int rows, int d) {
  return pieces <= kThreads && (int64_t)pieces * rows * d * 4 <= kPMergeBytes;
}

// A class's stretches: of units where all are equally long and that leaves a workgroup at
// most kPAhead tiles more, what its beginning another unit costs (us, of the line and of
// units: one token of 3 sequences of 4128 keys d128 8 bits 19.4 / 14.7, of 16 34.6 / 30.7,
// of 32 16 bits 86.0 / 82.1).
template <class Line>
__device__ __forceinline__ PagedStretch<kPMinTiles> paged_stretch(const PagedArgs& a, const Line& line) {
  const int total = line.total(), same = line.same;
  PagedStretch<kPMinTiles> s(a, total);
  if (!a.split) {
    s.active = s.cuts = min(a.wgs, total);
  } else if (same > 0 && s.active > 0) {
    const int count = s.units(same);
    const int q = min(s.small_quotient(a.wgs, count), (int)((unsigned)(same + kPMinTiles - 1) / kPMinTiles));
    if (q > 0 && same <= (int64_t)q * ((int)((unsigned)total / (unsigned)s.active) + kPAhead))
      s.cut_units(count, same, q);
  }
  return s;
}

template <int D, bool BF16, bool FP8, int NT>
__global__ void __launch_bounds__(kThreads, 2) fa_paged_attn_kernel(const PagedArgs a) {
  using E = Elem<BF16>;
  constexpr int R = 16 * NT;
  constexpr int KS = D / 32;  // contraction steps of S^T
  constexpr int MT = D / 16;  // 16-dimension tiles of O^T
  constexpr int KL = FP8 ? KS / 2 : KS;         // K loads of a 16-key piece
  constexpr int RL = FP8 ? D / 16 : D / 8;      // lanes that hold a V row, 16 bytes each
  constexpr int VL = 16 * RL / 64;              // V loads of a piece
  // A wave's V tile: 32 rows of D halves, 32-byte piece p of row r at p ^ swz(r)
  // (the transposing reads take 32 bytes of 8 consecutive rows at once: eight
  // different pieces of the 256-byte sweep of the banks).  Two arrays, so that
  // the compiler sees that loads in flight into one do not touch the other;
  // an 8-bit cache's rows pass through registers and need one.
  constexpr int VT = kPTile * D;
  constexpr bool TWO = !FP8 || NT == 2;
  __shared__ __attribute__((aligned(1024))) _Float16 v_lds0[4 * VT];
  __shared__ __attribute__((aligned(1024))) _Float16 v_lds1[TWO ? 4 * VT : 1];
  static_assert(16 * D * 4 <= VT * 2, "a wave's O of 16 columns fits its V tile");
  __shared__ float ml_lds[4][2][R];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l16 = lane & 15;
  const int g4 = lane >> 4;
  const int cls = (int)blockIdx.x & (a.classes - 1);
  const int wg = (int)(blockIdx.x >> a.class_shift);

  const PagedLine<R, kPTile, kPAhead> line(a, lane, a.split != 0);
  auto stretch = paged_stretch(a, line);
  if (wg >= stretch.active) return;
  int pos, end;
  stretch.of(wg, pos, end);
  asm volatile("" : "+v"(stretch.len), "+v"(stretch.cuts));  // (few scalar registers are left)
  int seq_start;
  int b = uniform(line.find(pos, seq_start));

  auto swz = [](int r) { return D == 128 ? (r & 7) : ((r >> 1) & 3); };
  _Float16* const vt0 = v_lds0 + wave * VT;
  _Float16* const vt1 = v_lds1 + (TWO ? wave * VT : 0);
  const float c2 = a.c;

  // Offsets inside a 16-key piece of what this lane loads: row l16 of K, 16 bytes
  // at 16 g4 of each 64; VL times 64 / RL rows of V, RL lanes a row, in the
  // order of the tile (16-bit rows go to LDS directly, lane l's 16 bytes at
  // 16 l of each KB).
  const int k_off = l16 * (int)a.kn + 16 * g4;
  int v_off[VL];
#pragma unroll
  for (int i = 0; i < VL; ++i) {
    const int row = (64 * i + lane) / RL, ch = (64 * i + lane) % RL;
    v_off[i] = row * (int)a.vn + 16 * (FP8 ? ch : ch ^ (2 * swz(row)));
  }
  // Bases of the transposing reads: lane i of a 16-lane group names 4 dimensions
  // of row i / 4 of the group's four; it receives dimension i of all four.
  const int r0 = 4 * g4 + (l16 >> 2);

  while (pos < end) {
    const PagedSeq s = line.seq(b);
    const int blocks = paged_blocks<R>(a, s);
    const int unit_len = line.unit_of(s);
    const int len = line.length_of(s);
    if (pos >= seq_start + len || len == 0) {  // on to the next sequence
      seq_start += len;
      if (++b >= a.batch) return;
      continue;
    }
    const int unit = line.unit_at(pos - seq_start, unit_len, blocks);
    const int u0 = seq_start + unit * unit_len + line.ahead;  // its first tile on the line
    const int u1 = seq_start + (unit + 1) * unit_len;
    const int first = max(0, pos - u0);  // tiles [first, stop) of it are this stretch's
    if (u1 <= pos) return;  // (wrapped round)
    pos = min(u1, end);
    const int stop = pos - u0;
    if (stop <= 0) break;
    const int hc = blocks == 1 ? unit : (int)((unsigned)unit / (unsigned)blocks);
    const int rb = unit - hc * blocks;
    const int hkv = hc * a.classes + cls;
    const bool whole = first == 0 && pos == u1;
    const int t_begin = first;
    const int t_end = a.split ? stop : (s.keys + kPTile - 1) / kPTile;

    // Columns of this lane, one for each nt: whether they hold a row, and the last
    // key it sees.
    const int nrows = s.n * a.group;
    const PagedRows row_of(a, s, hkv, rb * R);
    const int past = s.len - s.n;  // tokens before the new ones
    int last[NT];
    half8 qf[NT][KS];
    auto load_q = [&] {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int c = 16 * nt + l16;
        const bool ok = rb * R + c < nrows;
        const PagedRow pr = row_of(ok ? c : 0);
        last[nt] = a.causal ? min(s.keys - 1, past + (pr.token - s.t0)) : s.keys - 1;
        const _Float16* qp = a.q + pr.token * a.qt + pr.head * a.qh;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          // Dimensions of step kk that lane group g4 contracts: 8 of a 16-bit
          // row's 64 bytes; of an 8-bit row's 64 bytes 16, over two steps.
          const int dim = FP8 ? 64 * (kk >> 1) + 16 * g4 + 8 * (kk & 1) : 32 * kk + 8 * g4;
          qf[nt][kk] = ok ? *(const half8*)(qp + dim) : (half8)(_Float16)0;
        }
      }
    };
    // (behind the first tile's loads: it waits for Q)
    auto sign_q = [&] {
      fence_schedule();
      if (a.negate_q) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int kk = 0; kk < KS; ++kk) qf[nt][kk] = negate16(qf[nt][kk]);
      }
    };
    // Keys no row of the block sees are not read (past `sees`); tiles up to `full`
    // hide nothing from any of them.
    const int tok_first = uniform(row_of(0).token) - s.t0;
    const int tok_last = uniform(row_of(min(nrows - rb * R, R) - 1).token) - s.t0;
    const int sees = a.causal ? uniform(clamp_int(past + tok_last + 1, 0, s.keys)) : s.keys;
    const int full = a.causal ? uniform(clamp_int(past + tok_first + 1, 0, s.keys)) : s.keys;
    const int t_stop = min(t_end, (sees + kPTile - 1) / kPTile);

    float4v o[NT][MT];
    float m_run[NT], l_run[NT], thr[NT], mc[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[nt][mt] = (float4v)0.0f;
      m_run[nt] = thr[nt] = -__builtin_inff();
      l_run[nt] = mc[nt] = 0.0f;
    }

    // A tile in flight: which of its two pieces hold keys, and the registers that
    // its loads fill.
    struct Tile {
      int rows[2];
      uint4v k[2][KL];
      uint4v v[FP8 ? 2 : 1][FP8 ? VL : 1];
      unsigned ks[2], vs[2][FP8 ? VL : 1];
    };
    const int32_t* const entries = a.table + b * a.table_stride;
    const uint8_t* const kh = a.k + hkv * a.kh;
    const uint8_t* const vh = a.v + hkv * a.vh;
    // Table entries of a tile's pieces (of the last page, past the table).
    auto look_up = [&](int t, int (&e)[2]) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
        e[p] = load_scalar(entries + min((t * kPTile + 16 * p) >> a.page_shift, a.max_pages - 1));
    };
    // Issues a tile's loads.  A piece in no page or past the keys reads through an
    // empty window: zeros, and no traffic.
    auto load = [&](int t, const int (&e)[2], Tile& x, _Float16* vt) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int key = t * kPTile + 16 * p;
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
        const __amdgpu_buffer_rsrc_t rv = make_rsrc(vh + page * a.vp + off * a.vn, x.rows[p] * (int)a.vn);
        if constexpr (FP8) {
          const __amdgpu_buffer_rsrc_t rs =
              make_rsrc(a.vs + page * a.vsp + hkv * a.vsh + off * a.vsn, x.rows[p] * (int)a.vsn);
#pragma unroll
          for (int i = 0; i < VL; ++i) {
            // Non-temporal, as the 16-bit rows' direct loads: whole lines that nobody
            // reads again.  K's are read in halves and stay cached.
            x.v[p][i] = __builtin_bit_cast(
                uint4v, __builtin_amdgcn_raw_buffer_load_b128(rv, v_off[i], 0, kPStreamed));
            x.vs[p][i] =
                __builtin_amdgcn_raw_buffer_load_b8(rs, (64 * i + lane) / RL * (int)a.vsn, 0, 0);
          }
        } else {
#pragma unroll
          for (int i = 0; i < VL; ++i)
            direct_load16_nt(rv, (lds_void*)(vt + (16 * p * RL + 64 * i) * 8), v_off[i]);
        }
      }
    };

    // Scores to probabilities of one tile, then P V.
    auto compute = [&](int t, const int (&rows)[2], float4v (&st)[2][NT], const _Float16* vt, auto wait) {
      // Lane group g4 holds keys 16 p + 4 g4 + i of column l16.
      if ((t + 1) * kPTile > full || rows[0] == 0 || rows[1] == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (t * kPTile + 16 * p + 4 * g4 + i > last[nt] || rows[p] == 0)
                st[p][nt][i] = -__builtin_inff();
      }
      half8 pf[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mx = -__builtin_inff();
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, st[p][nt][i]);
        if (__builtin_amdgcn_ballot_w64(mx > thr[nt]) != 0) {
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float m_new = fmaxf(m_run[nt], mx);
          const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
          const float alpha = m_run[nt] == -__builtin_inff()
                                  ? 0.0f
                                  : __builtin_amdgcn_exp2f((m_run[nt] - m_use) * c2);
          l_run[nt] *= alpha;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) o[nt][mt] *= alpha;
          m_run[nt] = m_new;
          mc[nt] = m_use * c2;
          thr[nt] = m_new + a.rescale;
        }
        uint4v pw;
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[p][nt][i], c2, -mc[nt]));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[p][nt][i + 1], c2, -mc[nt]));
            l_run[nt] += p0;
            l_run[nt] += p1;
            pw[2 * p + (i >> 1)] = __builtin_bit_cast(unsigned, E::pack(p0, p1));
          }
        pf[nt] = __builtin_bit_cast(half8, pw);
      }
      wait();
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const half4 lo = ds_read_tr16(vt + r0 * D + 16 * (mt ^ swz(r0)) + 4 * (l16 & 3));
        const half4 hi = ds_read_tr16(vt + (r0 + 16) * D + 16 * (mt ^ swz(r0)) + 4 * (l16 & 3));
        const half8 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[nt][mt] = E::mfma16(vf, pf[nt], o[nt][mt]);
      }
    };

    int t = t_begin + wave;
    if (t < t_stop) {
      int e[2];
      look_up(t, e);
      load_q();
      if constexpr (FP8) {
        // The tile's codes are converted, K's in registers and V's into LDS, and the
        // next tile's loads go into the registers they leave.
        Tile x;
        load(t, e, x, nullptr);
        look_up(t + 4, e);
        sign_q();
        for (; t < t_stop; t += 4) {
          float4v st[2][NT];
          const int rows[2] = {x.rows[0], x.rows[1]};
#pragma unroll
          for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int i = 0; i < VL; ++i) {
              const int row = 16 * p + (64 * i + lane) / RL, q = (64 * i + lane) % RL;
              const float vs = scale_of(x.vs[p][i]);
              _Float16* const dst = vt0 + row * D + 16 * (q ^ swz(row));
              *(half8*)dst = dequantise8<BF16>(x.v[p][i][0], x.v[p][i][1], vs);
              *(half8*)(dst + 8) = dequantise8<BF16>(x.v[p][i][2], x.v[p][i][3], vs);
            }
            const float ks = scale_of(x.ks[p]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) st[p][nt] = (float4v)0.0f;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
              const uint4v w = x.k[p][kk / 2];
              const half8 kf = kk & 1 ? dequantise8<BF16>(w[2], w[3], ks) : dequantise8<BF16>(w[0], w[1], ks);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) st[p][nt] = E::mfma16(kf, qf[nt][kk], st[p][nt]);
            }
          }
          load(t + 4, e, x, nullptr);
          look_up(t + 8, e);
          compute(t, rows, st, vt0, [] {});
        }
      } else {
        Tile xa, xb;
        load(t, e, xa, vt0);
        look_up(t + 4, e);
        sign_q();
        auto step = [&](int tt, Tile& cur, Tile& nxt, const _Float16* vc, _Float16* vn) {
          load(tt + 4, e, nxt, vn);
          look_up(tt + 8, e);
          float4v st[2][NT];
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              st[p][nt] = (float4v)0.0f;
#pragma unroll
              for (int kk = 0; kk < KS; ++kk)
                st[p][nt] = E::mfma16(__builtin_bit_cast(half8, cur.k[p][kk]), qf[nt][kk], st[p][nt]);
            }
          // V of this tile has landed once only the next tile's loads are in flight.
          compute(tt, cur.rows, st, vc, [] { wait_loads<2 * (KL + VL)>(); });
        };
        for (; t + 4 < t_stop; t += 8) {
          step(t, xa, xb, vt0, vt1);
          step(t + 4, xb, xa, vt1, vt0);
        }
        if (t < t_stop) step(t, xa, xb, vt0, vt1);
      }
    }

    // ---- the four waves' shares meet in LDS ---------------------------------
    // No direct load is in flight into a V tile any more, and no wave reads one.
    if constexpr (!FP8) wait_loads<0>();
    __syncthreads();
    // What depends on the thread from here on is derived from an opaque index, so that none
    // of it is made ready ahead of the tiles or kept through them.
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int t16 = tid & 15, t4 = (tid & 63) >> 4;
    // O of column c (16 of them to an array), 16-byte chunk d at d ^ c.
    auto o_at = [&](int w, int c, int chunk) -> float4v* {
      float* const base = (float*)(c < 16 || !TWO ? v_lds0 : v_lds1) + w * 16 * D;
      return (float4v*)(base + (c & 15) * D + 4 * (chunk ^ (c & 15)));
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float l = l_run[nt];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      const int c = 16 * nt + t16;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) *o_at(wave, c, 4 * mt + t4) = o[nt][mt];
      if (t4 == 0) {
        ml_lds[wave][0][c] = m_run[nt];
        ml_lds[wave][1][c] = l;
      }
    }
    __syncthreads();
    // Thread: 4 dimensions of one column, columns in turns.
    for (int it = tid; it < R * (D / 4); it += kThreads) {
      const int c = it / (D / 4), ch = it - c * (D / 4), dim = 4 * ch;
      const int r = rb * R + c;
      if (r >= nrows) continue;
      float mw[4], m = -__builtin_inff(), l = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        mw[w] = ml_lds[w][0][c];
        m = fmaxf(m, mw[w]);
      }
      const float m_use = m == -__builtin_inff() ? 0.0f : m;
      float4v x = (float4v)0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f((mw[w] - m_use) * c2);
        l += f * ml_lds[w][1][c];
        x += f * *o_at(w, c, ch);
      }
      const float m2 = m == -__builtin_inff() ? m : m * c2;
      if (whole) {
        store_row<BF16>(a, row_of(c), dim, m2, l, x);
      } else {
        // Coherent over the L2s: the merging workgroup may be on another XCD.
        const int64_t rec = (int64_t)(2 * (int)blockIdx.x + (first == 0 ? 1 : 0)) * R;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4v, x), make_rsrc(a.part_o + rec * D, R * D * 4),
                                               (c * D + dim) * 4, 0, kPCoherent);
        if (dim == 0)
          __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, v2f{m2, l}),
                                                make_rsrc(a.part_ml + rec * 2, R * 8), c * 8, 0, kPCoherent);
      }
    }
    if (whole) {
      __syncthreads();  // the next unit's loads go into these tiles
      continue;
    }

    // ---- the unit's last workgroup merges its partials -------------------------
    const PagedPieces pieces(stretch, a.wgs, u0, u1);
    const int nr = min(R, nrows - rb * R);
    if (!paged_merges_itself(pieces.count, nr, D)) {
      ask_combine(a);
      __syncthreads();
      continue;
    }
    if (!last_to_finish(a, pieces, cls, 2 * (int)blockIdx.x + (first == 0 ? 1 : 0), (int*)v_lds0)) continue;
    // Thread: 4 dimensions of a row, pieces grp, grp + groups, ...; the groups
    // meet in LDS.  More items than threads: one group, items in turns.
    const int items = nr * (D / 4);
    const int groups = max(1, min(kThreads / items, pieces.count));
    const int grp = groups > 1 ? tid / items : 0;
    float4v* const xo = (float4v*)v_lds0;
    float* const xm = (float*)(v_lds0 + 8 * kThreads);  // max, then sum
    static_assert(kThreads * 24 <= 4 * VT * 2, "the merge's states fit the V tiles");
    for (int it = tid - grp * items; grp < groups && it < items; it += kThreads) {
      const int c = it / (D / 4), ch = it - c * (D / 4);
      float m = -__builtin_inff(), l = 0.0f;
      float4v x = (float4v)0.0f;
      for (int i = grp; i < pieces.count; i += 12 * groups)
        fold_partials<12>(
            i, groups, pieces.count, m, l, x,
            [&](int i) {
              const int64_t rec = (int64_t)pieces.slot(a, cls, i) * R + c;
              return __builtin_bit_cast(v2f, __builtin_amdgcn_raw_buffer_load_b64(make_rsrc(a.part_ml, INT32_MAX),
                                                                                  (int)(rec * 8), 0, kPCoherent));
            },
            [&](int i) {
              const int64_t rec = (int64_t)pieces.slot(a, cls, i) * R + c;
              return __builtin_bit_cast(
                  float4v, __builtin_amdgcn_raw_buffer_load_b128(make_rsrc(a.part_o, INT32_MAX),
                                                                 (int)((rec * D + 4 * ch) * 4), 0, kPCoherent));
            });
      if (groups > 1) {
        xo[tid] = x;
        xm[tid] = m;
        xm[kThreads + tid] = l;
      } else {
        store_row<BF16>(a, row_of(c), 4 * ch, m, l, x);
      }
    }
    __syncthreads();
    if (groups > 1 && tid < items) {
      float m = -__builtin_inff(), l = 0.0f;
      float4v x = (float4v)0.0f;
      for (int g = 0; g < groups; ++g) m = fmaxf(m, xm[g * items + tid]);
      for (int g = 0; g < groups; ++g) {
        const float w = __builtin_amdgcn_exp2f(xm[g * items + tid] - over_zero(m));
        l += w * xm[kThreads + g * items + tid];
        x += w * xo[g * items + tid];
      }
      const int c = tid / (D / 4);
      store_row<BF16>(a, row_of(c), 4 * (tid - c * (D / 4)), m, l, x);
    }
    __syncthreads();
  }
}

// Merges the partials of units whose last workgroup does not: a workgroup for each
// unit of a class (blockIdx.x) and row (blockIdx.y, and every gridDim.y-th on).
// The four waves take every fourth piece, D / 4 lanes each piece's row (with
// several pieces at once where D / 4 < 64 lanes), and meet in LDS.
template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(kThreads) fa_paged_combine_kernel(const PagedArgs a) {
  constexpr int R = 16 * NT;
  constexpr int LR = D / 4;               // lanes of a row
  constexpr int GROUPS = kThreads / LR;   // pieces at once
  __shared__ float4v xo[kThreads];
  __shared__ float xm[2][kThreads];
  if (!combine_asked(a)) return;
  const int cls = (int)blockIdx.x & (a.classes - 1);
  const int index = (int)(blockIdx.x >> a.class_shift);  // of the class's units
  const PagedLine<R, kPTile, kPAhead> line(a, threadIdx.x & 63, true);
  const PagedLine<R, kPTile, kPAhead> units(a, threadIdx.x & 63, false);
  if (index >= units.total()) return;
  int unit_start;
  const int b = uniform(units.find(index, unit_start));
  const PagedSeq s = line.seq(b);
  const int unit_len = line.unit_of(s);
  const int unit = index - unit_start;
  const int u0 = line.start_of(b) + unit * unit_len;
  const auto stretch = paged_stretch(a, line);
  const PagedPieces pieces(stretch, a.wgs, u0 + line.ahead, u0 + unit_len);
  if (pieces.count == 1) return;
  const int blocks = paged_blocks<R>(a, s);
  const int hc = unit / blocks;
  const int rb = unit - hc * blocks;
  const int hkv = hc * a.classes + cls;
  const int nr = min(R, s.n * a.group - rb * R);
  if (paged_merges_itself(pieces.count, nr, D)) return;
  const int grp = (int)threadIdx.x / LR, ch = (int)threadIdx.x % LR;
  for (int c = blockIdx.y; c < nr; c += gridDim.y) {
    float m = -__builtin_inff(), l = 0.0f;
    float4v x = (float4v)0.0f;
    for (int i = grp; i < pieces.count; i += 8 * GROUPS)
      fold_partials<8>(
          i, GROUPS, pieces.count, m, l, x,
          [&](int i) { return *(const v2f*)(a.part_ml + ((int64_t)pieces.slot(a, cls, i) * R + c) * 2); },
          [&](int i) {
            return *(const float4v*)(a.part_o + ((int64_t)pieces.slot(a, cls, i) * R + c) * D + 4 * ch);
          });
    xo[threadIdx.x] = x;
    xm[0][threadIdx.x] = m;
    xm[1][threadIdx.x] = l;
    __syncthreads();
    if (grp == 0) {
      for (int g = 1; g < GROUPS; ++g) m = fmaxf(m, xm[0][g * LR + ch]);
      l = 0.0f;
      x = (float4v)0.0f;
      for (int g = 0; g < GROUPS; ++g) {
        const float w = __builtin_amdgcn_exp2f(xm[0][g * LR + ch] - over_zero(m));
        l += w * xm[1][g * LR + ch];
        x += w * xo[g * LR + ch];
      }
      store_row<BF16>(a, PagedRows(a, s, hkv, rb * R)(c), 4 * ch, m, l, x);
    }
    __syncthreads();
  }
}

}  // namespace

template <int D, bool BF16, bool FP8>
void launch_paged_attn(const PagedArgs& a, int rows, int64_t grid, hipStream_t stream) {
  if (rows == 16)
    hipLaunchKernelGGL((fa_paged_attn_kernel<D, BF16, FP8, 1>), dim3((unsigned)grid), dim3(kThreads), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((fa_paged_attn_kernel<D, BF16, FP8, 2>), dim3((unsigned)grid), dim3(kThreads), 0,
                       stream, a);
}

}  // namespace fa
