// Attention of a chunk of new tokens over a paged cache: units of 128 query rows.
//
// A unit is one (sequence, KV head, block of 128 rows), row r of a sequence being
// token r / group of query head kv_head * group + r % group, so that a chunk of few
// tokens fills a block with its heads, and all rows of a block read the same K and V.
// One workgroup = 4 waves, wave w rows 32 w .. 32 w + 31; keys stream through LDS
// in double-buffered tiles of 64.  The matrix formulation, the LDS layouts and the
// step's schedule are the dense forward's (fa_fwd_kernel.h): S^T = K Q^T and O^T =
// V^T P^T in 32x32x16 MFMAs, one query per lane, step j issuing the MFMAs of S_{j+1}
// and P_j V_j slot by slot with the softmax of S_j, the operand reads and the
// loads of K_{j+2} and V_{j+1} between them.
//
// Pages.  Each wave brings 16 consecutive keys of every tile, which lie in one page
// whatever its size (16 or more): one table entry and one buffer window, whose base
// is scalar, for all its loads.  Table entries are read through the scalar cache a
// tile ahead.  Pieces that name no page read through an empty window (zeros) and
// are masked.
//
// 8-bit rows go through registers: a wave converts its 16 rows of a tile once for the
// workgroup (the codes times a power of two are 16-bit numbers) and writes them to LDS
// in the layout the 16-bit rows arrive in.
//
// The plan.  Where the units do not fill the GPU (SPLIT), each workgroup takes an equal
// stretch of the class's line of 64-key tiles, as in the kernel for few columns, or where
// all units are equally long a piece of one (chunk_stretch); the partials of units that are
// cut are merged by the unit's last workgroup where they are few, else by a second
// kernel.  Else a workgroup takes a unit, each head's from its last block (under the causal
// rule the longest) to its first; where all of them run at once, two a CU, the second half
// of them in reverse, so that a CU gets a long and a short one.
//
// What bounds it: as in the dense forward, the step (a tile's 32 MFMAs a wave, its softmax
// and 168 KB of LDS traffic a workgroup, two workgroups a CU: 1555 cycles each where the
// MFMAs alone take 1024 at d128; of one workgroup alone 2558), 2048 tokens behind 6144 of 32
// heads d128 232 to 248 us from one card to the next, 970 to 1040 TFLOP/s; in short launches
// what a workgroup does before its first tile and after its last (7 us) and the merges (3 to 5
// us); with 8-bit rows VALU instructions: three sequences of 1777 to 4000 keys, 777 new tokens
// each, 14 heads d64, 47 to 51 us, issue 254 a wave and tile, of which the softmax is 112
// (16-bit rows d128 179), and every 128-row unit converts all its K and V again.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_paged_units.h"

namespace fa {
namespace {

constexpr int kChunkRows = 128;
// Tiles a stretch is not cut below (us with 4, 5 and 6: one prompt of 320 tokens d128 17.9 /
// 14.8 / 14.8, of 384 18.3 / 18.4 / 15.7, of 640 24.9 / 23.0 / 23.0, 64 tokens behind 936
// 20.4 / 20.5 / 21.0).
constexpr int kChunkMinTiles = 6;
// Another unit's cost, in tiles (us without and with: 512 tokens of one sequence among 15
// single ones of 1000 to 4096 keys d128 63.5 / 61.5, 777 of three of 1777 to 4000 d64
// 51.9 / 51.3).
constexpr int kChunkAhead = 3;

// Rounds and stores two groups of 8 dimensions of a row.  The half-waves hold 4
// dimensions each of both; the lower takes the first whole and the upper the
// second: one 16-byte store.  `to`: the lane's 8.
template <bool BF16>
__device__ __forceinline__ void store_pair(_Float16* to, float4v x, float4v y, float inv) {
  uint4v v;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const unsigned u0 =
        __builtin_bit_cast(unsigned, Elem<BF16>::pack(x[2 * e] * inv, x[2 * e + 1] * inv));
    const unsigned u1 =
        __builtin_bit_cast(unsigned, Elem<BF16>::pack(y[2 * e] * inv, y[2 * e + 1] * inv));
    const auto z = __builtin_amdgcn_permlane32_swap(u0, u1, false, false);
    v[e] = z[0];
    v[2 + e] = z[1];
  }
  *(uint4v*)to = v;
}

// Whether a unit's last workgroup merges its partials (it reads them at about 50
// bytes/ns, 6 us for these many), or the second kernel.  Where a launch has units enough
// (plan_chunks), stretches are made long enough that none has more, and the second
// kernel is not launched.
constexpr int kChunkMergeBytes = 320 << 10;
constexpr int chunk_pieces(int d) { return kChunkMergeBytes / (kChunkRows * d * 4); }

// A record of the workspace: a block's partials in the order its waves' registers
// hold them, so that 64 lanes store and load 1 KB at once (row by row, 16 bytes of
// 32 rows at once, coherent stores took half of a short launch).  Group 4 mt + g of a wave:
// dimensions 32 mt + 8 g + 4 (lane / 32) .. + 3 of its row lane % 32.
template <int D>
struct ChunkRecord {
  static constexpr int Groups = D / 8;
  __amdgpu_buffer_rsrc_t o, ml;
  __device__ __forceinline__ ChunkRecord(const PagedArgs& a) {
    o = make_rsrc(a.part_o, INT32_MAX);
    ml = make_rsrc(a.part_ml, INT32_MAX);
  }
  __device__ __forceinline__ int o_at(int record, int wave, int group, int lane) const {
    return (((record * 4 + wave) * Groups + group) * 64 + lane) * 16;
  }
  __device__ __forceinline__ int ml_at(int record, int wave, int ql) const {
    return ((record * 4 + wave) * 32 + ql) * 8;
  }
};

// Merges pairs of groups pair0 .. pair0 + 3 of a unit's partials, wave w its rows
// 32 w .. + 31 (of `rows`), and stores them: O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M)
// l_i, M = max_i m_i.
template <int D, bool BF16>
__device__ __forceinline__ void merge_chunk(const PagedArgs& a, const PagedPieces& pieces, int cls,
                                            const PagedRows& row_of, int rows, int pair0) {
  constexpr int PAIRS = 4, AT = 4;  // at once; pieces at once
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int hi = lane >> 5, ql = lane & 31;
  const int r = 32 * wave + ql;
  if (r >= rows) return;
  const ChunkRecord<D> rec(a);
  auto load_ml = [&](int i) {
    return __builtin_bit_cast(v2f, __builtin_amdgcn_raw_buffer_load_b64(
                                       rec.ml, rec.ml_at(pieces.slot(a, cls, i), wave, ql), 0, kPCoherent));
  };
  float m = -__builtin_inff();
  for (int i0 = 0; i0 < pieces.count; i0 += 8) {
    v2f ml[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) ml[u] = load_ml(min(i0 + u, pieces.count - 1));
#pragma unroll
    for (int u = 0; u < 8; ++u) m = fmaxf(m, ml[u][0]);
  }
  float l = 0.0f;
  float4v x[PAIRS][2];
#pragma unroll
  for (int q = 0; q < PAIRS; ++q) x[q][0] = x[q][1] = (float4v)0.0f;
  for (int i0 = 0; i0 < pieces.count; i0 += AT) {
    v2f ml[AT];
    float4v o[AT][PAIRS][2];
#pragma unroll
    for (int u = 0; u < AT; ++u) {
      const int i = min(i0 + u, pieces.count - 1);
      const int record = pieces.slot(a, cls, i);
      ml[u] = load_ml(i);
#pragma unroll
      for (int q = 0; q < PAIRS; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          o[u][q][e] = __builtin_bit_cast(
              float4v, __builtin_amdgcn_raw_buffer_load_b128(
                           rec.o, rec.o_at(record, wave, 2 * (pair0 + q) + e, lane), 0, kPCoherent));
    }
#pragma unroll
    for (int u = 0; u < AT; ++u) {
      if (i0 + u >= pieces.count) break;  // (the last one again)
      const float w = __builtin_amdgcn_exp2f(ml[u][0] - over_zero(m));
      l += w * ml[u][1];
#pragma unroll
      for (int q = 0; q < PAIRS; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) x[q][e] += w * o[u][q][e];
    }
  }
  const PagedRow pr = row_of(r);
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  _Float16* const op = a.o + pr.token * a.ot + pr.head * a.oh;
#pragma unroll
  for (int q = 0; q < PAIRS; ++q) store_pair<BF16>(op + 16 * (pair0 + q) + 8 * hi, x[q][0], x[q][1], inv);
  if (a.lse != nullptr && hi == 0 && pair0 == 0)
    a.lse[(int64_t)pr.head * a.tokens + pr.token] = natural_lse(m, l);
}

// A class's stretches.  Where all units are equally long, of units, each into the number q
// of pieces that costs least, unless along the line it costs less yet.  The costs are in
// tiles, fitted to timings (us at q = 1, 2, 3, ..: one prompt of 512 tokens d128 17.8, 19.2;
// of 900 24.6, 28.0; 500 tokens behind 1500 -, 32.6, 35.6, 34.5; 64 behind 936 -, 23.4, 21.0,
// 20.1; one prompt of 800 d64 18.4, 17.5, 16.1; along the line against units: one prompt of
// 1700 tokens d128 50.2 / 42.7, three of 900 d64 32.4 / 24.6, 800 tokens behind 3200 d128
// 66.2 / 68.2): two workgroups on a CU slow each other down by a quarter; the merge costs so
// much a piece, the more the more workgroups do it, at most what the second kernel does;
// along the line a workgroup begins two units and most are cut.
template <int D, class Line>
__device__ __forceinline__ PagedStretch<kChunkMinTiles> chunk_stretch(const PagedArgs& a, const Line& line) {
  const int total = line.total(), same = line.same;
  PagedStretch<kChunkMinTiles> s(a, total);
  if (a.pieces > 0 && s.active > 0) {
    // (a unit as long as pieces - 1 stretches lies in one more at most)
    const int least = (int)((unsigned)(line.longest() + a.pieces - 2) / (unsigned)(a.pieces - 1));
    s.active = s.cuts = uniform(min(s.active, max(1, (int)((unsigned)total / (unsigned)least))));
  }
  if (same > 0 && s.active > 0) {
    const int count = s.units(same);
    const int q = line.lane + 1;  // a lane each
    const float full = 1.0f / (float)a.wgs;
    auto slowed = [&](int wgs) { return 1.0f + 0.25f * fmaxf(0.0f, 2.0f * (float)wgs * full - 1.0f); };
    const int most = s.small_quotient(same + q - 1, q);
    const float piece = D == 128 ? 1.0f + 2.5f * (float)(count * q) * full : 1.7f;
    float cost = (float)most * slowed(count * q) + (q > 1 ? fminf(piece * (float)q, 14.0f) : 0.0f);
    if (count > a.wgs / q || (a.pieces > 0 && q > a.pieces)) cost = __builtin_inff();
    float least = cost;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) least = fminf(least, __shfl_xor(least, m));
    const float along = (float)total / (float)s.active * slowed(s.active) + 10.0f;
    const uint64_t at = __builtin_amdgcn_ballot_w64(cost == least);
    if (least < along) s.cut_units(count, same, __builtin_ctzll(at) + 1);
  }
  return s;
}

// STREAM: V's rows are read non-temporally (a sequence's only block is the one that reads them).
template <int D, bool BF16, bool FP8, bool SPLIT, bool STREAM>
__global__ void __launch_bounds__(kThreads, 2) fa_paged_chunk_kernel(const PagedArgs a) {
  constexpr bool DENSE = D == 64;
  using L = std::conditional_t<DENSE, LdsDense<D>, Lds<D>>;
  using E = Elem<BF16>;
  constexpr int KK = D / 16;       // 16-wide contraction steps of S^T
  constexpr int MT = D / 32;       // 32-row output tiles of O^T
  constexpr int NS = 2 * KK;       // S^T MFMAs per tile
  constexpr int NPV = 4 * MT;      // P V MFMAs per tile
  constexpr int PFK = 3;           // K operand reads run this many MFMAs ahead
  constexpr int PFV = 2;           // V operand reads run this many MFMAs ahead
  constexpr int SEGQ = L::Segs / 4;            // 1 KB segments of a wave's 16 rows
  constexpr int RL = D / 16;                   // FP8: lanes that hold a row's codes
  constexpr int LQ = 16 * RL / 64;             // FP8: 16-byte loads of 16 rows
  constexpr int LPW = FP8 ? 2 * LQ : 2 * SEGQ; // loads per wave and step
  static_assert(SEGQ * 1024 == 16 * L::Pitch * 2, "a wave's segments are its 16 rows");

  // Distinct objects, so that the compiler sees that loads in flight into one do
  // not touch the tiles being read.
  __shared__ __attribute__((aligned(1024))) _Float16 k_lds0[L::Tile];
  __shared__ __attribute__((aligned(1024))) _Float16 k_lds1[L::Tile];
  __shared__ __attribute__((aligned(1024))) _Float16 v_lds0[L::Tile];
  __shared__ __attribute__((aligned(1024))) _Float16 v_lds1[L::Tile];

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int cls = (int)blockIdx.x & (a.classes - 1);
  const int wg = (int)(blockIdx.x >> a.class_shift);
  const PagedLine<kChunkRows, kBlockN, kChunkAhead> line(a, threadIdx.x & 63, SPLIT);
  const auto stretch = [&] {
    if constexpr (SPLIT) return chunk_stretch<D>(a, line);
    else return PagedStretch<1>(a, line.total());
  }();
  if (wg >= stretch.active) return;
  int pos, end;
  stretch.of(wg, pos, end);
  if constexpr (!SPLIT) {
    if (a.causal && stretch.len <= a.resident && pos >= a.resident / 2)
      pos = stretch.len - 1 + a.resident / 2 - pos;
  }
  int seq_start;
  int b = uniform(line.find(pos, seq_start));

  do {
  const PagedSeq s = line.seq(b);
  const int blocks = paged_blocks<kChunkRows>(a, s);
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
  if (SPLIT && u1 <= pos) return;  // (wrapped round)
  pos = SPLIT ? min(u1, end) : u1;
  const int stop = pos - u0;
  if (SPLIT && stop <= 0) break;
  const bool whole = !SPLIT || (first == 0 && pos == u1);
  const int hc = blocks == 1 ? unit : (int)((unsigned)unit / (unsigned)blocks);
  const int rb = blocks - 1 - (unit - hc * blocks);
  const int hkv = hc * a.classes + cls;

  // What depends on the lane is derived for each segment from an opaque lane index, so
  // that none of it is kept in registers from one to the next.
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  const int hi = lane >> 5;   // which half of the wave
  const int ql = lane & 31;   // query column owned by this lane
  const int grp = lane >> 4;  // 16-lane group (transposing reads)
  const int gi = lane & 15;
  const int nrows = s.n * a.group;
  const int q0 = rb * kChunkRows;
  const int qw = q0 + 32 * wave;
  const int row = qw + ql;
  const int past = s.len - s.n;  // tokens before the new ones

  // Keys the block's rows see, and this segment's tiles of them.
  const PagedRows row_of(a, s, hkv, q0);
  const int last_tok = uniform(row_of(min(nrows - q0, kChunkRows) - 1).token) - s.t0;
  const int kv_len = a.causal ? uniform(clamp_int(past + last_tok + 1, 0, s.keys)) : s.keys;
  const int block_tiles = (kv_len + kBlockN - 1) / kBlockN;
  const int tile0 = SPLIT ? first : 0;
  const int tile_end = SPLIT ? min(block_tiles, stop) : block_tiles;
  // The last key this lane's row sees; keys below wave_full are seen by every row of
  // the wave.
  const int tok = row_of(min(row, nrows - 1) - q0).token - s.t0;
  const int last_key = a.causal ? min(s.keys - 1, past + tok) : s.keys - 1;
  const int wave_full =
      a.causal ? uniform(clamp_int(past + row_of(min(qw, nrows - 1) - q0).token - s.t0 + 1, 0, s.keys)) : s.keys;

  // Q^T fragments (B operand of S^T), resident for the whole kernel.
  half8 qf[KK];
  auto load_q = [&] {
    const PagedRow pr = row_of(min(row, nrows - 1) - q0);
    const _Float16* qp = a.q + pr.token * a.qt + pr.head * a.qh + 8 * hi;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[kk] = *(const half8*)(qp + 16 * kk);
  };
  auto sign_q = [&] {  // (behind the first tiles' loads: it waits for Q)
    if (a.negate_q) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) qf[kk] = negate16(qf[kk]);
    }
  };

  // What a lane loads of its wave's 16 rows: byte offsets from the first row.
  // 16-bit rows go to LDS directly (lane l's 16 bytes at 16 l of each KB; padding
  // lanes: past any window).
  int koff[FP8 ? 1 : SEGQ], voff[FP8 ? 1 : SEGQ];
  if constexpr (!FP8) {
#pragma unroll
    for (int i = 0; i < SEGQ; ++i) {
      const int at = 1024 * i + 16 * lane;
      const int r = at / (2 * L::Pitch);
      const int within = at - r * (2 * L::Pitch);
      if (DENSE || within < 2 * D) {
        const int c = (within >> 4) ^ (DENSE ? dense_swizzle(r) : ((r >> 2) & 3));
        koff[i] = r * (int)a.kn + 16 * c;
        voff[i] = r * (int)a.vn + 16 * c;
      } else {
        koff[i] = voff[i] = -16;
      }
    }
  }

  // Table entries of a tile's four 16-key pieces, and what they say: the page of
  // this wave's piece (-1: none) and which pieces are in no page.
  const int32_t* const entries = a.table + b * a.table_stride;
  auto look_up = [&](int j, int (&e)[4]) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
      e[p] = load_scalar(entries + min((j * kBlockN + 16 * p) >> a.page_shift, a.max_pages - 1));
  };
  struct Pages {
    int own;
    unsigned gone;
  };
  auto pages_of = [&](const int (&e)[4]) -> Pages {
    Pages x;
    x.gone = 0;
#pragma unroll
    for (int p = 0; p < 4; ++p) x.gone |= (unsigned)e[p] < (unsigned)a.num_pages ? 0u : 1u << p;
    x.own = wave < 2 ? (wave == 0 ? e[0] : e[1]) : (wave == 2 ? e[2] : e[3]);
    if ((x.gone >> wave) & 1) x.own = -1;
    return x;
  };
  const uint8_t* const kh = a.k + hkv * a.kh;
  const uint8_t* const vh = a.v + hkv * a.vh;
  // Window of this wave's rows of tile j (empty past the piece's keys).
  auto rows_of = [&](int j, int page) -> int {
    return uniform(page >= 0 && j < tile_end ? clamp_int(kv_len - (j * kBlockN + 16 * wave), 0, 16) : 0);
  };
  auto window = [&](const uint8_t* base, int64_t sp, int64_t sn, int j, int page) {
    const int off = (j * kBlockN + 16 * wave) & ((1 << a.page_shift) - 1);
    return make_rsrc(base + (int64_t)max(page, 0) * sp + off * sn, rows_of(j, page) * (int)sn);
  };

  auto kbuf = [&](auto st) -> _Float16* { return decltype(st)::value % 2 == 0 ? k_lds0 : k_lds1; };
  auto vbuf = [&](auto st) -> _Float16* { return decltype(st)::value % 2 == 0 ? v_lds0 : v_lds1; };
  auto lds_seg = [&](_Float16* tile, int i) -> lds_void* {
    int off = (SEGQ * wave + i) * 512;
    asm volatile("" : "+s"(off));  // recomputed at each load, not kept in a register
    return (lds_void*)(tile + off);
  };

  auto load_v16 = [](const __amdgpu_buffer_rsrc_t r, lds_void* to, int off) {
    if constexpr (STREAM) direct_load16_nt(r, to, off);
    else direct_load16(r, to, off);
  };

  // 8-bit rows in flight: this wave's 16 rows of a K tile and of a V tile.
  constexpr int LF = FP8 ? LQ : 1;
  uint4v kr[LF], vr[LF];
  unsigned ksr[LF], vsr[LF];
  auto load_codes = [&](const uint8_t* base, int64_t sp, int64_t sn, const uint8_t* sbase, int64_t ssp,
                        int64_t ssn, int j, int page, uint4v (&w)[LF], unsigned (&sc)[LF], auto policy) {
    const __amdgpu_buffer_rsrc_t r = window(base, sp, sn, j, page);
    const __amdgpu_buffer_rsrc_t rs = window(sbase, ssp, ssn, j, page);
#pragma unroll
    for (int i = 0; i < LF; ++i) {
      const int rr = (64 * i + lane) / RL;
      w[i] = __builtin_bit_cast(
          uint4v, __builtin_amdgcn_raw_buffer_load_b128(r, rr * (int)sn + 16 * (lane % RL), 0,
                                                        decltype(policy)::value));
      sc[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, rr * (int)ssn, 0, 0);
    }
  };
  // Half `h` of load i (8 codes) into its place of the tile.
  auto store_codes = [&](_Float16* tile, const uint4v& w, unsigned sc, int i, int h) {
    const int rr = 16 * wave + (64 * i + lane) / RL;
    const int c = (2 * (lane % RL) + h) ^ (DENSE ? dense_swizzle(rr) : ((rr >> 2) & 3));
    *(half8*)(tile + rr * L::Pitch + 8 * c) = dequantise8<BF16>(w[2 * h], w[2 * h + 1], scale_of(sc));
  };
  const uint8_t* const ksh = FP8 ? a.ks + hkv * a.ksh : nullptr;
  const uint8_t* const vsh = FP8 ? a.vs + hkv * a.vsh : nullptr;
  auto load_k8 = [&](int j, int page) {
    load_codes(kh, a.kp, a.kn, ksh, a.ksp, a.ksn, j, page, kr, ksr, std::integral_constant<int, 0>{});
  };
  auto load_v8 = [&](int j, int page) {
    load_codes(vh, a.vp, a.vn, vsh, a.vsp, a.vsn, j, page, vr, vsr,
               std::integral_constant<int, STREAM ? kPStreamed : 0>{});
  };

  // Per-lane LDS bases of the operand reads (as in the dense forward).
  const int sK = (ql >> 2) & 3;
  const int k_base_even = ql * L::Pitch + 8 * (hi ^ sK);
  const int k_base_odd = ql * L::Pitch + 8 * ((2 + hi) ^ sK);
  const int v_row = 4 * hi + (gi >> 2);
  const int v_c = 2 * (grp & 1) + ((gi & 3) >> 1);
  const int v_base0 = v_row * L::Pitch + 8 * (v_c ^ hi) + 4 * (gi & 1);
  const int v_base1 = (v_row + 8) * L::Pitch + 8 * (v_c ^ (hi + 2)) + 4 * (gi & 1);
  int kd_base[DENSE ? KK : 1], vd_base0[DENSE ? MT : 1], vd_base1[DENSE ? MT : 1];
  if constexpr (DENSE) {
    const int sw = dense_swizzle(ql);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) kd_base[kk] = ql * L::Pitch + 8 * ((2 * kk + hi) ^ sw);
    const int sw0 = dense_swizzle(v_row), sw1 = dense_swizzle(v_row + 8);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      vd_base0[mt] = v_row * L::Pitch + 8 * ((v_c + 4 * mt) ^ sw0) + 4 * (gi & 1);
      vd_base1[mt] = (v_row + 8) * L::Pitch + 8 * ((v_c + 4 * mt) ^ sw1) + 4 * (gi & 1);
    }
  }
  auto read_k = [&](const _Float16* Ks, int i) -> half8 {
    const int t = i / KK, kk = i % KK;
    if constexpr (DENSE) return *(const half8*)(Ks + kd_base[kk] + 32 * t * L::Pitch);
    const int off = ((kk & 1) ? k_base_odd : k_base_even) + 32 * t * L::Pitch + 32 * (kk >> 1);
    return *(const half8*)(Ks + off);
  };
  auto read_v = [&](const _Float16* Vs, int v) -> half8 {
    const int ks = v / MT, mt = v % MT;
    const int imm = 16 * ks * L::Pitch + (DENSE ? 0 : 32 * mt);
    const half4 lo = ds_read_tr16(Vs + (DENSE ? vd_base0[DENSE ? mt : 0] : v_base0) + imm);
    const half4 hi4 = ds_read_tr16(Vs + (DENSE ? vd_base1[DENSE ? mt : 0] : v_base1) + imm);
    return __builtin_shufflevector(lo, hi4, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  float16v oacc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) oacc[mt] = (float16v)0.0f;
  float m_run = -__builtin_inff();
  float l_run = 0.0f;  // the lane's part of its row sum
  const float c2 = a.c;
  float16v s_buf[2][2];  // S^T of two tiles in flight
  float mc = 0.0f;       // running max times c2 (exp2 offset)
  float thr = -__builtin_inff();

  // Masks tile j's scores where it hides a key from some row of the wave, and
  // raises the running max when some row outgrew it by more than 2^kRescaleLog2.
  // mx: the lane's max over its half of the row.
  auto prepare = [&](int j, float16v (&sc)[2], float mx, unsigned gone) {
    const int kstart = j * kBlockN;
    if (kstart + kBlockN > wave_full || gone != 0) {
      const int lim = last_key - kstart - 4 * hi;
      static_for<32>([&](auto e_c) {
        constexpr int e = decltype(e_c)::value;
        constexpr int t = e >> 4, i = e & 15;
        constexpr int off = 32 * t + 8 * (i >> 2) + (i & 3);
        if (off > lim || ((gone >> (off >> 4)) & 1)) sc[t][i] = -__builtin_inff();
      });
      mx = -__builtin_inff();
      static_for<32>([&](auto e_c) {
        constexpr int e = decltype(e_c)::value;
        mx = fmaxf(mx, sc[e >> 4][e & 15]);
      });
    }
    if (__builtin_amdgcn_ballot_w64(mx > thr) != 0) {
      const float m_new = fmaxf(m_run, halves_max(mx));
      const float m_use = (m_new == -__builtin_inff()) ? 0.0f : m_new;
      const float alpha =
          (m_run == -__builtin_inff()) ? 0.0f : __builtin_amdgcn_exp2f((m_run - m_use) * c2);
      l_run *= alpha;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) oacc[mt] *= alpha;
      m_run = m_new;
      mc = m_use * c2;
      thr = m_new + a.rescale;
    }
  };

  // Pages of tiles j + 1 and j + 2 at the start of step j, and the entries of
  // tile j + 3 (in flight).
  Pages pg1, pg2;
  int ahead[4];

  auto step = [&](int j, auto has_next_t, auto u_t) {
    constexpr bool HAS_NEXT = decltype(has_next_t)::value;
    constexpr int U = decltype(u_t)::value;
    constexpr int ns = HAS_NEXT ? NS : 0;  // S MFMAs this step
    const _Float16* Kn = kbuf(std::integral_constant<int, U + 1>{});
    const _Float16* Vc = vbuf(std::integral_constant<int, U>{});
    float16v (&s_cur)[2] = s_buf[U];
    float16v (&s_nxt)[2] = s_buf[1 - U];

    // Loads of K_{j+2} (into the buffer K_j used) and V_{j+1} (into V_{j-1}'s), one
    // after each of the first MFMAs.  8-bit rows: those tiles' codes, loaded a step
    // ago, are converted and stored, and the next tiles' loads follow.
    __amdgpu_buffer_rsrc_t rk_next, rv_next;
    const Pages now1 = pg1, now2 = pg2;
    if constexpr (HAS_NEXT) {
      pg1 = pg2;
      pg2 = pages_of(ahead);
      look_up(j + 4, ahead);
      if constexpr (!FP8) {
        rk_next = window(kh, a.kp, a.kn, j + 2, now2.own);
        rv_next = window(vh, a.vp, a.vn, j + 1, now1.own);
      }
    }
    _Float16* const k_dst = kbuf(std::integral_constant<int, U>{});
    _Float16* const v_dst = vbuf(std::integral_constant<int, U + 1>{});
    auto issue_load = [&](auto q_c) {
      constexpr int q = decltype(q_c)::value;
      if constexpr (FP8) {  // half a load's codes to LDS
        constexpr int i = q / 4, h = q & 1;
        if constexpr ((q & 2) == 0) store_codes(k_dst, kr[i], ksr[i], i, h);
        else store_codes(v_dst, vr[i], vsr[i], i, h);
        if constexpr (q == 4 * LQ - 1) {
          load_k8(j + 3, pg2.own);
          load_v8(j + 2, pg1.own);
        }
      } else if constexpr (q < SEGQ) {
        direct_load16(rk_next, lds_seg(k_dst, q), koff[q]);
      } else {
        load_v16(rv_next, lds_seg(v_dst, q - SEGQ), voff[q - SEGQ]);
      }
    };
    constexpr int NL = FP8 ? 4 * LQ : LPW;

    constexpr int NB = ns + NPV;            // MFMA slots
    constexpr int PV_FIRST = ns;            // slot of the first P V MFMA
    constexpr int PAIR_SLOTS = NB - MT;     // slots available to pairs
    half8 kf[NS];
    uint4v pf[4];
    half8 vf[NPV];
    constexpr auto pair_slot = [](int p) constexpr {
      const int spread = (p * PAIR_SLOTS) / 16;
      const int last_ok = PV_FIRST + (p / 4) * MT - 1;
      return spread < last_ok ? spread : last_ok;
    };
    constexpr auto max_slot = [](int e) constexpr {
      const int t = e >> 4, i = e & 15;
      const int first = (t + 1) * KK + 2;
      const int span = (t == 0 ? KK : NB - 1 - first);
      const int sl = first + (i * span) / 16;
      return sl < NB - 1 ? sl : NB - 1;
    };
    constexpr auto last_max_slot = [max_slot]() constexpr {
      int m = 0;
      for (int e = 0; e < 32; ++e) m = max_slot(e) > m ? max_slot(e) : m;
      return m;
    };
    auto softmax_pair = [&](auto p_c) {
      constexpr int p = decltype(p_c)::value;
      constexpr int e = 2 * p;
      constexpr int t = e >> 4, i = e & 15;
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s_cur[t][i], c2, -mc));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s_cur[t][i + 1], c2, -mc));
      pf[2 * t + (i >> 3)][(i & 7) >> 1] = __builtin_bit_cast(unsigned, E::pack(p0, p1));
      l_run += p0 + p1;
      asm volatile("" : "+v"(l_run));  // keeps the sum in this slot
    };
    static_for<16>([&](auto p_c) {
      if constexpr (pair_slot(decltype(p_c)::value) < 0) softmax_pair(p_c);
    });
    if constexpr (D == 128) __builtin_amdgcn_s_setprio(1);
    static_for<(PFK < ns ? PFK : ns)>([&](auto i_c) {
      kf[decltype(i_c)::value] = read_k(Kn, decltype(i_c)::value);
    });
    float mx_next = -__builtin_inff();
    static_for<NB>([&](auto slot_c) {
      constexpr int slot = decltype(slot_c)::value;
      if constexpr (slot == (PV_FIRST >= PFV ? PV_FIRST - PFV : 0)) {
        static_for<PFV>([&](auto v_c) {
          vf[decltype(v_c)::value] = read_v(Vc, decltype(v_c)::value);
        });
      }
      if constexpr (slot >= PV_FIRST && slot - PV_FIRST + PFV < NPV)
        vf[slot - PV_FIRST + PFV] = read_v(Vc, slot - PV_FIRST + PFV);
      if constexpr (slot < PV_FIRST) {
        constexpr int i = slot;
        if constexpr (i + PFK < ns) kf[i + PFK] = read_k(Kn, i + PFK);
        constexpr int t = i / KK, kk = i % KK;
        s_nxt[t] = E::mfma(kf[i], qf[kk], kk == 0 ? (float16v)0.0f : s_nxt[t]);
      } else {
        constexpr int v = slot - PV_FIRST;
        constexpr int ks = v / MT, mt = v % MT;
        oacc[mt] = E::mfma(vf[v], __builtin_bit_cast(half8, pf[ks]), oacc[mt]);
      }
      if constexpr (HAS_NEXT) {
        static_for<NL>([&](auto q_c) {
          constexpr int q = decltype(q_c)::value;
          if constexpr ((q * (NB / 2)) / NL == slot) issue_load(q_c);
        });
        static_for<32>([&](auto e_c) {
          constexpr int e = decltype(e_c)::value;
          if constexpr (max_slot(e) == slot) mx_next = fmaxf(mx_next, s_nxt[e >> 4][e & 15]);
        });
        if constexpr (slot == last_max_slot()) asm volatile("" : "+v"(mx_next));
      }
      static_for<16>([&](auto p_c) {
        if constexpr (pair_slot(decltype(p_c)::value) == slot) softmax_pair(p_c);
      });
      fence_schedule();
    });
    if constexpr (D == 128) __builtin_amdgcn_s_setprio(0);
    if constexpr (HAS_NEXT) {
      prepare(j + 1, s_nxt, mx_next, now1.gone);
      // Direct loads have landed (codes in flight to registers need not have), and
      // every wave is done with the buffers the next step's loads overwrite.
      barrier_after_loads<FP8 ? 63 : 0>();
    }
  };

  if (tile0 < tile_end) {
    // ---- prologue: K_0, K_1 and V_0 into LDS; S_0 -----------------------------
    int e0[4], e1[4], e2[4];
    look_up(tile0, e0);
    look_up(tile0 + 1, e1);
    look_up(tile0 + 2, e2);
    look_up(tile0 + 3, ahead);
    load_q();
    const Pages pg0 = pages_of(e0);
    pg1 = pages_of(e1);
    pg2 = pages_of(e2);
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    if constexpr (FP8) {
      load_k8(tile0, pg0.own);
      load_v8(tile0, pg0.own);
      static_for<LQ>([&](auto i_c) {
        constexpr int i = decltype(i_c)::value;
        static_for<2>([&](auto h_c) {
          store_codes(k_lds0, kr[i], ksr[i], i, decltype(h_c)::value);
          store_codes(v_lds0, vr[i], vsr[i], i, decltype(h_c)::value);
        });
      });
      load_k8(tile0 + 1, pg1.own);
      static_for<LQ>([&](auto i_c) {
        constexpr int i = decltype(i_c)::value;
        static_for<2>([&](auto h_c) { store_codes(k_lds1, kr[i], ksr[i], i, decltype(h_c)::value); });
      });
      load_k8(tile0 + 2, pg2.own);
      load_v8(tile0 + 1, pg1.own);
      fence_schedule();
      sign_q();
      barrier_after_loads<63>();
    } else {
      const __amdgpu_buffer_rsrc_t rk0 = window(kh, a.kp, a.kn, tile0, pg0.own);
      const __amdgpu_buffer_rsrc_t rk1 = window(kh, a.kp, a.kn, tile0 + 1, pg1.own);
      const __amdgpu_buffer_rsrc_t rv0 = window(vh, a.vp, a.vn, tile0, pg0.own);
#pragma unroll
      for (int i = 0; i < SEGQ; ++i) direct_load16(rk0, lds_seg(k_lds0, i), koff[i]);
#pragma unroll
      for (int i = 0; i < SEGQ; ++i) direct_load16(rk1, lds_seg(k_lds1, i), koff[i]);
#pragma unroll
      for (int i = 0; i < SEGQ; ++i) load_v16(rv0, lds_seg(v_lds0, i), voff[i]);
      fence_schedule();
      sign_q();
      barrier_after_loads<2 * SEGQ>();  // S_0 needs K_0 only
    }
    if (qw >= nrows) {
      // A wave without rows (a short block: a single token's heads) brings its share
      // of the tiles and meets the barriers.
      barrier_after_loads<FP8 ? 63 : 0>();
      for (int j = tile0; j + 1 < tile_end; ++j) {
        const Pages now1 = pg1, now2 = pg2;
        pg1 = pg2;
        pg2 = pages_of(ahead);
        look_up(j + 4, ahead);
        const bool odd = (j - tile0) & 1;
        _Float16* const k_dst = odd ? k_lds1 : k_lds0;
        _Float16* const v_dst = odd ? v_lds0 : v_lds1;
        if constexpr (FP8) {
          static_for<LQ>([&](auto i_c) {
            constexpr int i = decltype(i_c)::value;
            static_for<2>([&](auto h_c) {
              store_codes(k_dst, kr[i], ksr[i], i, decltype(h_c)::value);
              store_codes(v_dst, vr[i], vsr[i], i, decltype(h_c)::value);
            });
          });
          load_k8(j + 3, pg2.own);
          load_v8(j + 2, pg1.own);
        } else {
          const __amdgpu_buffer_rsrc_t rk = window(kh, a.kp, a.kn, j + 2, now2.own);
          const __amdgpu_buffer_rsrc_t rv = window(vh, a.vp, a.vn, j + 1, now1.own);
#pragma unroll
          for (int i = 0; i < SEGQ; ++i) direct_load16(rk, lds_seg(k_dst, i), koff[i]);
#pragma unroll
          for (int i = 0; i < SEGQ; ++i) load_v16(rv, lds_seg(v_dst, i), voff[i]);
        }
        barrier_after_loads<FP8 ? 63 : 0>();
      }
    } else {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s_buf[0][t] = (float16v)0.0f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        s_buf[0][t] = E::mfma(read_k(k_lds0, t * KK + kk), qf[kk], s_buf[0][t]);
    }
    float mx = -__builtin_inff();
    static_for<32>([&](auto e_c) {
      constexpr int e = decltype(e_c)::value;
      mx = fmaxf(mx, s_buf[0][e >> 4][e & 15]);
    });
    prepare(tile0, s_buf[0], mx, pg0.gone);
    // Step 0 writes K_2 into K_0's buffer: every wave must be done with it.
    barrier_after_loads<FP8 ? 63 : 0>();
    int j = tile0;
    for (; j + 2 < tile_end; j += 2) {
      step(j, Flag<true>{}, I0{});
      step(j + 1, Flag<true>{}, I1{});
    }
    if (tile_end - j == 1) {
      step(j, Flag<false>{}, I0{});
    } else {
      step(j, Flag<true>{}, I0{});
      step(j + 1, Flag<false>{}, I1{});
    }
    }
  }
  // No direct load may land in LDS after the workgroup, or the segment, ends.
  __builtin_amdgcn_s_waitcnt(0x0F70);

  const float l = halves_sum(l_run);
  const float m2 = m_run == -__builtin_inff() ? m_run : m_run * c2;
  if (row < nrows) {
    if (whole) {
      const PagedRow pr = row_of(row - q0);
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      _Float16* const op = a.o + pr.token * a.ot + pr.head * a.oh + 8 * hi;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int g = 0; g < 4; g += 2)
          store_pair<BF16>(op + 32 * mt + 8 * g,
                           float4v{oacc[mt][4 * g], oacc[mt][4 * g + 1], oacc[mt][4 * g + 2], oacc[mt][4 * g + 3]},
                           float4v{oacc[mt][4 * g + 4], oacc[mt][4 * g + 5], oacc[mt][4 * g + 6],
                                   oacc[mt][4 * g + 7]},
                           inv);
      if (a.lse != nullptr && hi == 0) a.lse[(int64_t)pr.head * a.tokens + pr.token] = natural_lse(m2, l);
    } else {
      // (see ChunkRecord; coherent over the L2s: the merging workgroup may be on
      // another XCD)
      const ChunkRecord<D> rec(a);
      const int record = 2 * (int)blockIdx.x + (first == 0 ? 1 : 0);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          __builtin_amdgcn_raw_buffer_store_b128(
              __builtin_bit_cast(uint4v, float4v{oacc[mt][4 * g], oacc[mt][4 * g + 1], oacc[mt][4 * g + 2],
                                                 oacc[mt][4 * g + 3]}),
              rec.o, rec.o_at(record, wave, 4 * mt + g, lane), 0, kPCoherent);
      if (hi == 0)
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, v2f{m2, l}), rec.ml,
                                              rec.ml_at(record, wave, ql), 0, kPCoherent);
    }
  }
  if constexpr (SPLIT) {
    if (!whole) {
      const PagedPieces pieces(stretch, a.wgs, u0, u1);
      if (pieces.count > chunk_pieces(D)) {
        ask_combine(a);
      } else if (last_to_finish(a, pieces, cls, 2 * (int)blockIdx.x + (first == 0 ? 1 : 0), (int*)k_lds0)) {
        for (int pair = 0; pair < D / 16; pair += 4)
          merge_chunk<D, BF16>(a, pieces, cls, row_of, nrows - q0, pair);
      }
    }
    __syncthreads();  // the next segment's loads go into these tiles
  }
  } while (SPLIT && pos < end);
}

// Merges the partials of units whose last workgroup does not.  The kChunkCombineY
// workgroups of a border between two stretches look at the unit it lies in; all those
// of the unit share its tasks, a pair of groups of one wave's 32 rows each.  Of a task
// the workgroup's waves take every fourth piece, and meet in LDS.
constexpr int kChunkCombineY = 2;
template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads) fa_paged_chunk_combine_kernel(const PagedArgs a) {
  __shared__ float4v xo[kWaves][2][64];
  __shared__ float xml[kWaves][2][64];
  if (!combine_asked(a)) return;
  const int cls = (int)blockIdx.x & (a.classes - 1);
  const int wg = (int)(blockIdx.x >> a.class_shift);
  const PagedLine<kChunkRows, kBlockN, kChunkAhead> line(a, threadIdx.x & 63, true);
  const auto stretch = chunk_stretch<D>(a, line);
  if (wg == 0 || wg >= stretch.active) return;
  int border, end;
  stretch.of(wg, border, end);
  int seq_start;
  const int b = uniform(line.find(border, seq_start));
  const PagedSeq s = line.seq(b);
  const int unit_len = line.unit_of(s);
  const int blocks = paged_blocks<kChunkRows>(a, s);
  if (blocks == 0) return;
  const int unit = line.unit_at(border - seq_start, unit_len, blocks);
  const int u0 = seq_start + unit * unit_len + line.ahead;  // its first tile on the line
  if (border <= u0) return;
  const PagedPieces pieces(stretch, a.wgs, u0, seq_start + (unit + 1) * unit_len);
  if (pieces.count <= chunk_pieces(D)) return;
  const int hc = unit / blocks;
  const int rb = blocks - 1 - (unit - hc * blocks);
  const int rows = s.n * a.group - rb * kChunkRows;
  const PagedRows row_of(a, s, hc * a.classes + cls, rb * kChunkRows);
  const ChunkRecord<D> rec(a);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int hi = lane >> 5, ql = lane & 31;
  const int share = (wg - pieces.first - 1) * kChunkCombineY + (int)blockIdx.y;
  for (int task = share; task < D / 16 * 4; task += (pieces.count - 1) * kChunkCombineY) {
    const int pair = task / 4, rw = task % 4;  // (rows 32 rw ..)
    constexpr int AT = 8;
    float m = -__builtin_inff(), l = 0.0f;
    float4v x[2] = {(float4v)0.0f, (float4v)0.0f};
    for (int i0 = wave; i0 < pieces.count; i0 += AT * kWaves) {
      v2f ml[AT];
      float4v o[AT][2];
      float m_new = m;
#pragma unroll
      for (int u = 0; u < AT; ++u) {
        const int record = pieces.slot(a, cls, min(i0 + u * kWaves, pieces.count - 1));
        ml[u] = __builtin_bit_cast(
            v2f, __builtin_amdgcn_raw_buffer_load_b64(rec.ml, rec.ml_at(record, rw, ql), 0, 0));
#pragma unroll
        for (int e = 0; e < 2; ++e)
          o[u][e] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(
                                                    rec.o, rec.o_at(record, rw, 2 * pair + e, lane), 0, 0));
      }
#pragma unroll
      for (int u = 0; u < AT; ++u) m_new = fmaxf(m_new, ml[u][0]);
      const float f = __builtin_amdgcn_exp2f(m - over_zero(m_new));
      l *= f;
      x[0] *= f;
      x[1] *= f;
#pragma unroll
      for (int u = 0; u < AT; ++u) {
        if (i0 + u * kWaves >= pieces.count) break;  // (the last one again)
        const float w = __builtin_amdgcn_exp2f(ml[u][0] - over_zero(m_new));
        l += w * ml[u][1];
        x[0] += w * o[u][0];
        x[1] += w * o[u][1];
      }
      m = m_new;
    }
    xo[wave][0][lane] = x[0];
    xo[wave][1][lane] = x[1];
    xml[wave][0][lane] = m;
    xml[wave][1][lane] = l;
    __syncthreads();
    const int r = 32 * rw + ql;
    if (wave == 0 && r < rows) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w) m = fmaxf(m, xml[w][0][lane]);
      l = 0.0f;
      x[0] = x[1] = (float4v)0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(xml[w][0][lane] - over_zero(m));
        l += f * xml[w][1][lane];
        x[0] += f * xo[w][0][lane];
        x[1] += f * xo[w][1][lane];
      }
      const PagedRow pr = row_of(r);
      store_pair<BF16>(a.o + pr.token * a.ot + pr.head * a.oh + 16 * pair + 8 * hi, x[0], x[1],
                       l > 0.0f ? 1.0f / l : 0.0f);
      if (a.lse != nullptr && hi == 0 && pair == 0)
        a.lse[(int64_t)pr.head * a.tokens + pr.token] = natural_lse(m, l);
    }
    __syncthreads();
  }
}

}  // namespace

template <int D, bool BF16, bool FP8>
void launch_paged_chunk(const PagedArgs& a, int64_t grid, hipStream_t stream) {
  const dim3 g((unsigned)grid), t(kThreads);
  if (a.split && a.stream_v)
    hipLaunchKernelGGL((fa_paged_chunk_kernel<D, BF16, FP8, true, true>), g, t, 0, stream, a);
  else if (a.split)
    hipLaunchKernelGGL((fa_paged_chunk_kernel<D, BF16, FP8, true, false>), g, t, 0, stream, a);
  else
    hipLaunchKernelGGL((fa_paged_chunk_kernel<D, BF16, FP8, false, false>), g, t, 0, stream, a);
}

}  // namespace fa
