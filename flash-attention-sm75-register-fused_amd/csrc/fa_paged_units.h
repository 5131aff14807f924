// What the two attention kernels over a paged cache (fa_paged_attn.h, fa_paged_chunk.h)
// share: a sequence's rows, wave broadcasts, and merging partial results.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_paged.h"

namespace fa {
namespace {

// Lane `lane`'s value, the same in every lane.
__device__ __forceinline__ int wave_bcast(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

// Inclusive prefix sum over the wave's lanes: within rows of 16, then rows 0 and 2
// into 1 and 3, then the lower half into the upper.
__device__ __forceinline__ int wave_prefix(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// The largest of the lanes' values (all 0 or more), in the same steps.
__device__ __forceinline__ int wave_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return wave_bcast(x, 63);
}

// Blocks of R rows of a sequence: its units for one KV head.
template <int R>
__device__ __forceinline__ int paged_blocks(const PagedArgs& a, const PagedSeq& s) {
  return (int)((unsigned)(s.n * a.group + R - 1) / R);  // (below 2^28)
}

// A sequence's prefix: which, its keys and their tiles (0: none).
struct PagedPre {
  int group, keys, tiles;
};

// The line of a class of KV heads (every classes-th head): the units of its
// sequences (blocks of R rows, for each head) end to end, each as long as its sequence
// has tiles of T keys (one at least, so that the rows of a sequence without keys are
// written too) and, where the sequences' lengths differ, H more in front of them, about
// what it costs a workgroup to begin another unit (where they are equal the borders
// of stretches often meet the units', which H would undo); or with tiles false of
// length one.  Below 2^31 in all (the launcher sees to it; only where cu_seqlens falls
// again and again, so that sequences share rows, may positions wrap round, and then
// units are held to those there are, and pieces to the workgroups).  Called by whole
// waves; the first 64 sequences, one a lane, are looked at once.
template <int R, int T, int H, int STAGE = 0>
struct PagedLine {
  const std::conditional_t<STAGE == kBoth, PagedShared, PagedArgs>& a;
  const int lane;
  const bool by_tiles;
  int ahead;     // H or 0: a unit's first `ahead` are no tiles
  int same;      // every unit's length, 0 where they differ or are not looked at
  PagedSeq own;  // sequence `lane` (kBoth: its keys behind its prefix's tiles)
  int first;     // prefix(0)
  PagedPre pre;  // kBoth: the sequence's prefix

  __device__ __forceinline__ PagedLine(const std::conditional_t<STAGE == kBoth, PagedShared, PagedArgs>& args, int ln,
                                       bool tiles)
      : a(args), lane(ln), by_tiles(tiles) {
    own = look(lane);
    if constexpr (STAGE == kBoth) {
      pre = shared();
      own.keys += T * pre.tiles;
    }
    ahead = 0;
    same = 0;
    if (tiles) {
      const int t = tiles_of(own);
      const uint64_t there = __builtin_amdgcn_ballot_w64(own.n > 0);
      const int t0 = there != 0 ? wave_bcast(t, __builtin_ctzll(there)) : 0;
      if (__builtin_amdgcn_ballot_w64(own.n > 0 && t != t0) != 0) ahead = H;
      else if (a.batch <= 64) same = max(1, t0);
    }
    first = wave_prefix(length_of(own));
  }
  __device__ __forceinline__ PagedSeq look(int b) const {
    PagedSeq s = paged_seq(a, min(b, a.batch - 1), [](const int32_t* p) { return *p; });
    if (b >= a.batch) s.n = 0;
    return s;
  }
  // (kBoth: at most 64 sequences and 63 prefixes)
  __device__ __forceinline__ PagedPre shared() const {
    PagedPre p = {0, 0, 0};
    if (a.groups != nullptr) {  // the last that begins at the sequence or before
      const int begin = a.groups[min(lane, a.prefixes)];
      for (int i = 0; i <= a.prefixes; ++i) p.group += wave_bcast(begin, i) <= lane ? 1 : 0;
      --p.group;
    }
    const bool has = lane < a.batch && p.group >= 0 && p.group < a.prefixes;
    if (!has) p.group = 0;
    const int len = a.pre_lens[p.group];
    p.keys = has ? clamp_int(len, 0, a.pre_pages << a.page_shift) : 0;
    p.tiles = (int)((unsigned)(p.keys + T - 1) / T);
    return p;
  }
  // Sequence b's prefix.
  __device__ __forceinline__ PagedPre pre_of(int b) const {
    if constexpr (STAGE != kBoth) return {0, 0, 0};
    return {wave_bcast(pre.group, b), wave_bcast(pre.keys, b), wave_bcast(pre.tiles, b)};
  }
  static __device__ __forceinline__ int tiles_of(const PagedSeq& s) { return (int)((unsigned)(s.keys + T - 1) / T); }
  // A unit's length on the line.
  __device__ __forceinline__ int unit_of(const PagedSeq& s) const {
    return by_tiles ? ahead + max(1, tiles_of(s)) : 1;
  }
  __device__ __forceinline__ int length_of(const PagedSeq& s) const {
    return a.heads * paged_blocks<R>(a, s) * unit_of(s);
  }
  // Inclusive prefix sum of the lengths of sequences b0 + lane.
  __device__ __forceinline__ int prefix(int b0) const {
    return b0 == 0 ? first : wave_prefix(length_of(look(b0 + lane)));
  }
  __device__ __forceinline__ int total() const {
    int sum = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) sum += wave_bcast(prefix(b0), 63);
    return sum;
  }
  // The longest unit's tiles, 1 at least.
  __device__ __forceinline__ int longest() const {
    int most = 1;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      const PagedSeq s = b0 == 0 ? own : look(b0 + lane);
      most = max(most, wave_max(s.n > 0 ? tiles_of(s) : 0));
    }
    return most;
  }
  __device__ __forceinline__ PagedSeq seq(int b) const {
    if (b >= 64) return scalar_seq(a, b);
    return {wave_bcast(own.t0, b), wave_bcast(own.n, b), wave_bcast(own.len, b), wave_bcast(own.keys, b)};
  }
  // The sequence b that holds position pos (0 <= pos < total), and where it starts.
  __device__ __forceinline__ int find(int pos, int& start) const {
    int before = 0;
    for (int b0 = 0;; b0 += 64) {
      const int x = prefix(b0);
      const uint64_t past = __builtin_amdgcn_ballot_w64(before + x > pos);
      if (past != 0 || b0 + 64 >= a.batch) {
        const int l = past != 0 ? __builtin_ctzll(past) : 63;
        start = l > 0 ? before + wave_bcast(x, l - 1) : before;
        return min(b0 + l, a.batch - 1);
      }
      before += wave_bcast(x, 63);
    }
  }
  // The unit (of sequence s, `blocks` of them for each head) at rel from its start.
  __device__ __forceinline__ int unit_at(int rel, int unit_len, int blocks) const {
    return uniform((int)min((unsigned)rel / (unsigned)unit_len, (unsigned)(a.heads * blocks - 1)));
  }
  // Where sequence b starts.
  __device__ __forceinline__ int start_of(int b) const {
    int before = 0;
    for (int b0 = 0; b0 + 64 <= b; b0 += 64) before += wave_bcast(prefix(b0), 63);
    return b % 64 == 0 ? before : before + wave_bcast(prefix(b / 64 * 64), b % 64 - 1);
  }
};

// The stretches of a class's line, one for each workgroup of it: of the whole line, total /
// active tiles each, or (cut_units) of every unit for itself where all are equally long.
// The first ones of the line, or unit, are a tile longer.  There are at most as many as
// stretches of LEAST tiles would be, rounded up: some may be shorter (nine tiles are two
// stretches), but none is then longer than LEAST, and all of them together are at most LEAST - 1
// short of it.
template <int LEAST>
struct PagedStretch {
  int active;
  int len, cuts;  // what is cut, and into how many
  __device__ __forceinline__ PagedStretch(const PagedArgs& a, int total) {
    active = uniform(min(a.wgs, (total + LEAST - 1) / LEAST));
    len = uniform(total);
    cuts = active;
  }
  // The most pieces a unit of `tiles` tiles is cut into.  Of `count` pieces all but the two
  // ends are whole stretches, of LEAST (count - 2) - (LEAST - 1) tiles in all or more, and
  // the ends have a tile each; of a unit cut for itself there are ceil(tiles / LEAST) at most.
  static __host__ __device__ constexpr int64_t most_pieces(int64_t tiles, int64_t wgs) {
    const int64_t pieces = (tiles + LEAST - 3) / LEAST + 2;
    return pieces < wgs ? pieces : wgs;
  }
  // Units of a line of them that are `same` tiles long (a quotient past 2^21, where this is
  // not exact, is more than there are workgroups).
  __device__ __forceinline__ int units(int same) const {
    return max(1, (int)rintf((float)len * __builtin_amdgcn_rcpf((float)same)));
  }
  // Every unit into q stretches.
  __device__ __forceinline__ void cut_units(int count, int same, int q) {
    active = uniform(count * q);
    len = uniform(same);
    cuts = uniform(q);
  }
  // x / y, x below 2^21 (x + 0.5 is 0.5 / y at least off a multiple of y).
  static __device__ __forceinline__ int small_quotient(int x, int y) {
    return (int)(((float)x + 0.5f) * __builtin_amdgcn_rcpf((float)y));
  }
  // Workgroup wg's (below active) stretch [pos, end).
  __device__ __forceinline__ void of(int wg, int& pos, int& end) const {
    const int u = wg < cuts ? 0 : small_quotient(wg, cuts), i = wg - u * cuts;
    const int size = (int)((unsigned)len / (unsigned)cuts), longer = len - size * cuts;
    pos = uniform(u * len + i * size + min(i, longer));
    end = uniform(pos + size + (i < longer ? 1 : 0));
  }
  __device__ __forceinline__ int holder(int pos) const {  // the workgroup of a position
    const int u = pos < len ? 0 : (int)((unsigned)pos / (unsigned)len), x = pos - u * len;
    const int size = (int)((unsigned)len / (unsigned)cuts), longer = len - size * cuts;
    const int p = x - longer * (size + 1);
    return u * cuts + (int)(p < 0 ? (unsigned)x / (unsigned)(size + 1) : longer + (unsigned)p / (unsigned)size);
  }
};

// The workgroups a unit whose tiles are [u0, u1) of the line was cut into: from first on, each
// with its record number slot(i) of the workspace.  A stretch starts inside at most one
// unit that it does not start with, and ends inside at most one: two records.
struct PagedPieces {
  int first, count;
  template <int LEAST>
  __device__ __forceinline__ PagedPieces(PagedStretch<LEAST> st, int wgs, int u0, int u1) {
    // (opaque: what its divisions begin with is not to be made ready ahead of each launch)
    asm volatile("" : "+v"(st.len), "+v"(st.cuts));
    first = st.holder(u0);
    count = st.holder(u1 - 1) - first + 1;
    // (no change but on a line past 2^31, see PagedLine)
    first = uniform(clamp_int(first, 0, wgs - 1));
    count = uniform(clamp_int(count, 1, wgs - first));
  }
  __device__ __forceinline__ int slot(const PagedArgs& a, int cls, int i) const {
    return 2 * ((first + i) * a.classes + cls) + (i == 0 ? 1 : 0);
  }
};

// Rows of a block: row r0 + c of a sequence is token r / group of query head
// kv_head * group + r % group.  The quotient of r0 is scalar; that of what is left and a
// lane's c (below 2^22) comes from a product with 1 / group, whose error stays under the
// 0.5 / group by which it is off a whole number.
struct PagedRow {
  int token, head;
};
struct PagedRows {
  int tok0, rem0, head0, group;
  float inv;
  __device__ __forceinline__ PagedRows(const PagedArgs& a, const PagedSeq& s, int hkv, int r0) {
    group = a.group;
    int i = 0;
    if (r0 != 0) {
      int g = group;
      asm volatile("" : "+s"(g));  // (so too)
      i = uniform((int)((unsigned)r0 / (unsigned)g));
    }
    tok0 = s.t0 + i;
    rem0 = r0 - i * group;
    head0 = hkv * group;
    inv = a.inv_group;
  }
  __device__ __forceinline__ PagedRow operator()(int c) const {
    const int x = rem0 + c;
    const int i = (int)(((float)x + 0.5f) * inv);
    return {tok0 + i, head0 + x - i * group};
  }
};

__device__ __forceinline__ float natural_lse(float m2, float l) {
  return ((m2 == -__builtin_inff() ? 0.0f : m2) + __builtin_log2f(l)) * 0.69314718055994530942f;
}

// A merge of partials: the running maximum (log2 units), sum and O.  Where the
// maximum is -inf every partial so far saw no key, with sum and O zero, or only
// NaN scores, with both NaN; relative to 0 the weight of either is 2^-inf = 0, which
// leaves the zeros and keeps the NaN.
__device__ __forceinline__ float over_zero(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// Cache policies of buffer accesses: the sc1 bit, coherent over the device's L2s; and the
// nt bit, for what is read once.
constexpr int kPCoherent = 16, kPStreamed = 2;
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

// Folds up to BATCH partials, step apart from i0 among count, into (m, l, x): all their
// loads are in flight together.  `load` gives a record's (max, sum) and 4 dimensions.
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

// ---- states over shared prefixes ---------------------------------------------------

// Rows of a prefix's unit (fa_paged_chunk.h), and where a record of their states keeps them: in
// the order its waves' registers hold them.  Group 4 mt + g of a wave: dimensions 32 mt + 8 g +
// 4 (lane / 32) .. + 3 of its row lane % 32.
constexpr int kChunkRows = 128;
template <int D>
__device__ __forceinline__ int64_t record_o(int64_t record, int wave, int group, int lane) {  // in floats
  return (((record * 4 + wave) * (D / 8) + group) * 64 + lane) * 4;
}
__device__ __forceinline__ int64_t record_ml(int64_t record, int row) { return (record * kChunkRows + row) * 2; }

// The records of one KV head's rows of a sequence over its prefix: `pieces` of them (0: it has
// none), `step` apart, the first rec0 for the prefix's first block of rows.
struct PagedJoint {
  int pieces, rec0, step, t0, n, head0;
};
__device__ __forceinline__ int joint_of(const PagedArgs&, int, int) { return 0; }  // (no prefixes)
__device__ __forceinline__ PagedJoint joint_of(const PagedShared& a, int b, int hkv) {
  PagedJoint j = {0, 0, 0, 0, 0, 0};
  int g = 0;
  if (a.groups != nullptr) {  // the last that begins at b or before
    const int lane = threadIdx.x & 63;
    for (int g0 = 0; g0 <= a.prefixes; g0 += 64) {
      const bool starts = g0 + lane <= a.prefixes && a.groups[min(g0 + lane, a.prefixes)] <= b;
      g += __builtin_popcountll(__builtin_amdgcn_ballot_w64(starts));
    }
    --g;
  }
  if (g >= 0 && g < a.prefixes) {
    const int32_t* const info = a.joint_info + 4 * g;
    const int start = load_scalar(info);
    j.pieces = load_scalar(info + 1);
    j.t0 = load_scalar(info + 2);
    j.n = load_scalar(info + 3);
    const int blocks = (int)((unsigned)(j.n * a.group + kChunkRows - 1) / kChunkRows);
    j.rec0 = ((start + ((hkv >> a.class_shift) + 1) * blocks - 1) << a.class_shift) + (hkv & (a.classes - 1));
    j.step = (a.heads * blocks) << a.class_shift;
    j.head0 = hkv * a.group;
  }
  return j;
}
// A row's own state (m, l, x) joined with those over its prefix's pieces: with M the largest of
// their maxima l = sum 2^(m_i - M) l_i, x likewise; all in 32 bits, one rounding to the 16-bit type
// behind it.
struct JointRow {
  int pieces;  // 0: none (also of a row that is not the prefix's, where cu_seqlens falls)
  int row;
  int64_t record;
  __device__ __forceinline__ JointRow(const PagedShared& a, const PagedJoint& j, const PagedRow pr) {
    pieces = j.pieces;
    const int i = pr.token - j.t0;
    const int r = i * a.group + pr.head - j.head0;
    row = r & (kChunkRows - 1);
    record = j.rec0 - ((int64_t)(r / kChunkRows) << a.class_shift);  // (blocks go from the last to the first)
    if ((unsigned)i >= (unsigned)j.n || record < 0 || record + (int64_t)(pieces - 1) * j.step >= a.joint_records)
      pieces = 0;
  }
};

// Folds pieces first, first + step, .. of a row's states over its prefix into (m, l, x), 4
// dimensions, BATCH of them asked for at once.
template <int D, int BATCH>
__device__ __forceinline__ void fold_joint(const PagedShared& a, const PagedJoint& joint, const PagedRow pr, int dim,
                                           int first, int step, float& m, float& l, float4v& x) {
  const JointRow j(a, joint, pr);
  const float* const o = a.joint_o + record_o<D>(j.record, j.row >> 5, dim >> 3, (dim & 4) * 8 + (j.row & 31));
  const float* const ml = a.joint_ml + record_ml(j.record, j.row);
  for (int i = first; i < j.pieces; i += BATCH * step)
    fold_partials<BATCH>(
        i, step, j.pieces, m, l, x, [&](int i) { return *(const v2f*)(ml + record_ml((int64_t)i * joint.step, 0)); },
        [&](int i) { return *(const float4v*)(o + record_o<D>((int64_t)i * joint.step, 0, 0, 0)); });
}

// O and LSE of a row from its state, 4 dimensions.
template <bool BF16>
__device__ __forceinline__ void finish_row(const PagedArgs& a, const PagedRow pr, int dim, float m2, float l, float4v x) {
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  half4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = Elem<BF16>::round(x[e] * inv);
  *(half4*)(a.o + pr.token * a.ot + pr.head * a.oh + dim) = y;
  if (a.lse != nullptr && dim == 0) a.lse[(int64_t)pr.head * a.tokens + pr.token] = natural_lse(m2, l);
}
// The same of a row that may have a prefix, whose state this is over its own keys.
template <int D, bool BF16>
__device__ __forceinline__ void store_row(const PagedArgs& a, int, const PagedRow pr, int dim, float m2, float l,
                                          float4v x) {
  finish_row<BF16>(a, pr, dim, m2, l, x);
}
template <int D, bool BF16>
__device__ __forceinline__ void store_row(const PagedShared& a, const PagedJoint& joint, const PagedRow pr, int dim,
                                          float m2, float l, float4v x) {
  if (joint.pieces > 0) fold_joint<D, 8>(a, joint, pr, dim, 0, 1, m2, l, x);
  finish_row<BF16>(a, pr, dim, m2, l, x);
}

// Waits until at most N of the wave's vector loads and stores are in flight (they
// land in order), and keeps the LDS reads that depend on it behind the wait.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
  asm volatile("" ::: "memory");
}

// The word behind the flags: whether some unit's partials are left to the second
// kernel, whose workgroups else end at once.
__device__ __forceinline__ uint64_t* combine_word(const PagedArgs& a) {
  return a.flags + 2 * (int64_t)a.wgs * a.classes;
}
__device__ __forceinline__ void ask_combine(const PagedArgs& a) {
  if (threadIdx.x == 0) *combine_word(a) = a.mark;
}
__device__ __forceinline__ bool combine_asked(const PagedArgs& a) { return *combine_word(a) == a.mark; }

// Sets the flag of a workgroup's record, whose partials its waves have stored
// coherently, and says whether every piece's flag of the unit is set (at most kThreads
// pieces).  `scratch`: kWaves ints of LDS that the workgroup is done with.  A
// workgroup's partials are acknowledged before it sets its flag, and its flag
// before it reads the others': the last flag to be set is set by a workgroup that
// sees them all.  Two that both do store the same values.
__device__ __forceinline__ bool last_to_finish(const PagedArgs& a, const PagedPieces& pieces, int cls,
                                               int record, int* scratch) {
  const __amdgpu_buffer_rsrc_t rf = make_rsrc(a.flags, 2 * (int)gridDim.x * 8);
  wait_loads<0>();
  __syncthreads();
  if (threadIdx.x == 0) {
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, a.mark), rf, record * 8, 0, kPCoherent);
    wait_loads<0>();
  }
  __syncthreads();
  bool set = true;
  if ((int)threadIdx.x < pieces.count)
    set = __builtin_bit_cast(uint64_t, __builtin_amdgcn_raw_buffer_load_b64(
              rf, pieces.slot(a, cls, threadIdx.x) * 8, 0, kPCoherent)) == a.mark;
  // (not __syncthreads_and, whose own LDS two workgroups a CU have no room for)
  const bool all = __builtin_amdgcn_ballot_w64(!set) == 0;
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = all;
  __syncthreads();
  bool last = true;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) last = last && scratch[w] != 0;
  __syncthreads();
  return last;
}

}  // namespace
}  // namespace fa
