// Eviction from a paged cache by accumulated attention weight: of each sequence and KV head,
// which rows stay (select), and their copies to the pages of another table (move).
//
// Of the positions that hold a row (not past the sequence's end, in a page), those of the
// last `recent` stay, and the heaviest others, min(keep, held) in all.  Weights compare as
// 32-bit integers in an order that is theirs (order_key), positions without a row below all
// of them and recent ones above, so what stays is the `target` largest keys, of equal ones
// those at the lowest positions.  Their smallest is found digit by digit from the top (11, 11 and 10
// bits): a histogram of the next digit among the keys that agree so far, and the bin at which the
// count from above reaches the target.  Counts are whole numbers, so no order of
// the additions shows.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "fa_kernel_common.h"
#include "fa_paged_units.h"

namespace fa {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kSelBins = 2048;
constexpr unsigned kRecentKey = 0xffffffffu;

// An integer that orders as the weights do: NaN below all (1; 0 is no row), -0 as 0.
__device__ __forceinline__ unsigned order_key(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);  // (-0 + 0 = 0)
  if (w != w) return 1;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One (sequence, KV head): what it holds and where that goes.
struct SelRow {
  const EvictArgs& e;
  const float* w;
  const int32_t* entries;
  int b, h, keys, recent_from, from_room, room;
  int32_t* kept;
  float* to_w;
  __device__ __forceinline__ SelRow(const EvictArgs& args, int pair) : e(args) {
    const PagedArgs& a = e.p;
    b = (int)((unsigned)pair / (unsigned)a.hkv);
    h = pair - b * a.hkv;
    const int len = max(0, a.lens[b]);
    from_room = a.max_pages << a.page_shift;
    keys = min(len, from_room);
    recent_from = len - min(e.recent, len);
    w = e.weights + b * e.wb + h * e.wh;
    entries = a.table + b * a.table_stride;
    kept = e.kept + (int64_t)pair * e.slots;
    room = e.to_pages << a.page_shift;
    to_w = e.new_weights + (int64_t)pair * room;
  }
};

// KEYS * kSelThreads positions of a row, a wave's KEYS * 64 next to each other, in registers.  (Loads
// do not wait for the sequence's length: the weights have the table's room.)
constexpr int kSelKeys = 8;  // the most
constexpr int kSelBlock = kSelKeys * kSelThreads;
template <int KEYS>
struct SelBlock {
  unsigned k[KEYS];
  float x[KEYS];
  int j0;  // this lane's first; 64 apart
  __device__ __forceinline__ SelBlock(const SelRow& row, int base, int end, int wave, int lane) {
    j0 = base + wave * (64 * KEYS) + lane;
    int page[KEYS];
#pragma unroll
    for (int u = 0; u < KEYS; ++u) {
      const int j = j0 + 64 * u;
      const bool there = j < row.from_room;
      x[u] = there ? row.w[j] : 0.0f;
      page[u] = there ? row.entries[j >> row.e.p.page_shift] : -1;
    }
#pragma unroll
    for (int u = 0; u < KEYS; ++u) {
      const int j = j0 + 64 * u;
      const bool held = j < min(end, row.keys) && page[u] >= 0 && page[u] < row.e.p.num_pages;
      k[u] = !held ? 0 : j >= row.recent_from ? kRecentKey : order_key(x[u]);
    }
  }
};

// The search: keys that stay are above `bound` where they differ from it under `mask`; `need`
// more of those that agree do.
struct Search {
  unsigned bound, mask;
  int need, shift;  // shift: 21, 10, 0
  __device__ __forceinline__ int width() const { return shift == 0 ? 1 << 10 : kSelBins; }
  __device__ __forceinline__ int digit(unsigned k) const { return (k >> shift) & (width() - 1); }
  template <int KEYS>
  __device__ __forceinline__ void count(const SelBlock<KEYS>& x, int* bins) const {
#pragma unroll
    for (int u = 0; u < KEYS; ++u)
      if (x.k[u] != 0 && (x.k[u] & mask) == bound) atomicAdd(&bins[digit(x.k[u])], 1);
  }
};

// What a workgroup shares in the search of one digit.
struct SelShared {
  int waves[kSelWaves];
  int found[2];
};
// The waves' values summed over those before this one, and over all (one barrier; `waves` is not
// written again).
__device__ __forceinline__ int2 across_waves(int x, int wave, int lane, int* waves) {
  if (lane == 0) waves[wave] = x;
  __syncthreads();
  int2 r = {0, 0};
#pragma unroll
  for (int i = 0; i < kSelWaves; ++i) {
    const int y = waves[i];
    r.x += i < wave ? y : 0;
    r.y += y;
  }
  return r;
}

// One digit on, given how many of the agreeing keys have the thread's two digits, hi and
// hi - 1 from the top.  keep: the keys wanted, where this is the first digit.  Returns all that agree.
__device__ __forceinline__ int descend(Search& s, int n1, int n0, int keep, int wave, int lane, SelShared& sh) {
  const int hi = kSelBins - 1 - 2 * (int)threadIdx.x;
  const int upto = wave_prefix(n0 + n1);
  const int2 sum = across_waves(wave_bcast(upto, 63), wave, lane, sh.waves);
  if (s.shift == 21) s.need = min(keep, sum.y);
  const int above = sum.x + upto - n0 - n1;
  if (above < s.need && above + n1 >= s.need) {
    sh.found[0] = hi;
    sh.found[1] = above;
  } else if (above + n1 < s.need && above + n1 + n0 >= s.need) {
    sh.found[0] = hi - 1;
    sh.found[1] = above + n1;
  }
  __syncthreads();
  return sum.y;
}
// (where there is something to search: some but not all stay)
__device__ __forceinline__ void take(Search& s, const SelShared& sh) {
  s.bound |= (unsigned)sh.found[0] << s.shift;
  s.need -= sh.found[1];
  s.mask |= (unsigned)(s.width() - 1) << s.shift;
  s.shift = s.shift > 10 ? s.shift - 11 : s.shift - 10;
}

// Writes which of a block's positions stay: `before` in front of them do, and so many of
// equal keys lie there, of which the first `need` stay.  Returns both for what is behind it.
template <int KEYS>
__device__ __forceinline__ int2 write_kept(const SelRow& row, const SelBlock<KEYS>& x, unsigned bound, int need, int target,
                                           int above, int same, int wave, int lane, int* waves) {
  int n = 0;  // of this wave: above the bound, and equal to it in the upper half
  uint64_t gt[KEYS], eq[KEYS];
#pragma unroll
  for (int u = 0; u < KEYS; ++u) {
    gt[u] = __builtin_amdgcn_ballot_w64(x.k[u] > bound);
    eq[u] = __builtin_amdgcn_ballot_w64(x.k[u] == bound && x.k[u] != 0);
    n += __builtin_popcountll(gt[u]) + (__builtin_popcountll(eq[u]) << 16);
  }
  const int2 sum = across_waves(n, wave, lane, waves);
  int a = above + (sum.x & 0xffff), s = same + (sum.x >> 16);
  const uint64_t lower = ((uint64_t)1 << lane) - 1;
#pragma unroll
  for (int u = 0; u < KEYS; ++u) {
    const int ge = a + __builtin_popcountll(gt[u] & lower), se = s + __builtin_popcountll(eq[u] & lower);
    const bool stays = x.k[u] > bound || (x.k[u] == bound && x.k[u] != 0 && se < need);
    const int to = ge + min(se, need);
    if (stays && to < target) {  // (to < target always, unless the weights change meanwhile)
      row.kept[to] = x.j0 + 64 * u;
      row.to_w[to] = x.x[u];
    }
    a += __builtin_popcountll(gt[u]);
    s += __builtin_popcountll(eq[u]);
  }
  return {above + (sum.y & 0xffff), same + (sum.y >> 16)};
}

// A workgroup for each (sequence, KV head), where the table has room for one block.  The chain of
// its steps bounds it (three digits of three barriers): 5.5 us for two rows of 1025 positions, 12.6 for
// 256 of 4096 .. 8192 (8 MB of weights).  With as few keys a thread as the table has room for: of 2 and 8
// 10.9 and 13.2 us for 8 rows of 1000 positions with the copy, 31.5 and 36.2 for 512.
template <int KEYS>
__global__ void __launch_bounds__(kSelThreads, 8) fa_paged_select_kernel(const EvictArgs e) {
  __shared__ int bins[kSelBins];
  __shared__ SelShared sh[4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  int2* const own = (int2*)bins + (kSelThreads - 1 - threadIdx.x);
  *own = {0, 0};
  const SelRow row(e, (int)blockIdx.x);
  const SelBlock<KEYS> x(row, 0, INT32_MAX, wave, lane);
  __syncthreads();
  Search s = {0, 0, 0, 21};
  int target = 0;
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    s.count(x, bins);
    __syncthreads();
    const int2 n = *own;  // (digits 2 i and 2 i + 1)
    *own = {0, 0};
    const int all = descend(s, n.y, n.x, e.keep, wave, lane, sh[p]);
    if (p == 0) target = s.need;
    if (p == 0 && (target == all || target == 0)) break;  // all that are held stay: those above 0
    take(s, sh[p]);
  }
  if (target > 0) {
    if (s.mask == 0) s.need = 0;
    write_kept(row, x, s.bound, s.need, target, 0, 0, wave, lane, sh[3].waves);
  }
  for (int j = target + (int)threadIdx.x; j < row.room; j += kSelThreads) row.to_w[j] = 0.0f;
  if (row.h == 0 && threadIdx.x == 0) e.new_lens[row.b] = target;
}

// Longer rows where they are many: the same, a block of positions after the other, for each digit anew.
// (Through the kernels below with one chunk a row they were four launches with a histogram of each digit in memory, 24 KB
// a row: with the copy 93.0 us for 78.9 at 256 rows of 20000 positions, 203 for 183 at 512 of 30000.)
__global__ void __launch_bounds__(kSelThreads, 8) fa_paged_select_blocks_kernel(const EvictArgs e) {
  __shared__ int bins[kSelBins];
  __shared__ SelShared sh[4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  int2* const own = (int2*)bins + (kSelThreads - 1 - threadIdx.x);
  *own = {0, 0};
  const SelRow row(e, (int)blockIdx.x);
  const int keys = row.keys;
  __syncthreads();
  Search s = {0, 0, 0, 21};
  int target = 0;
  for (int p = 0; p < 3; ++p) {
    for (int j = 0; j < keys; j += kSelBlock) s.count(SelBlock<kSelKeys>(row, j, keys, wave, lane), bins);
    __syncthreads();
    const int2 n = *own;
    *own = {0, 0};
    const int all = descend(s, n.y, n.x, e.keep, wave, lane, sh[p]);
    if (p == 0) target = s.need;
    if (p == 0 && (target == all || target == 0)) break;
    take(s, sh[p]);
  }
  if (target > 0) {
    if (s.mask == 0) s.need = 0;
    int2 before = {0, 0};
    for (int j = 0; j < keys; j += kSelBlock) {
      before = write_kept(row, SelBlock<kSelKeys>(row, j, keys, wave, lane), s.bound, s.need, target, before.x, before.y, wave,
                          lane, sh[3].waves);
      __syncthreads();
    }
  }
  for (int j = target + (int)threadIdx.x; j < row.room; j += kSelThreads) row.to_w[j] = 0.0f;
  if (row.h == 0 && threadIdx.x == 0) e.new_lens[row.b] = target;
}

// Longer rows, few: `chunks` workgroups each, in four launches.  The first three count a digit each over
// the chunk's keys, into a histogram of its own; the next launch adds those up to find the digit (and
// keeps where the search is), and what of the chunks in front of its own stays by it.  The launches'
// own chains bound them: 5, 8, 8 and 11 us at eight rows of 131072 positions (4 MB of weights, read four
// times), with the move 56 where the caches have them and 66 cold.  The chunk's first keys are loaded under the
// search for the digit (without, 57.0 for 55.6).
struct SelState {  // a row's search behind a digit
  unsigned bound;
  int need, target, search;
};
template <int PHASE>
__global__ void __launch_bounds__(kSelThreads, 8) fa_paged_select_long_kernel(const EvictArgs e) {
  __shared__ int bins[kSelBins];
  __shared__ SelShared sh;
  __shared__ int waves[3][kSelWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int pair = (int)((unsigned)blockIdx.x / (unsigned)e.chunks), chunk = (int)blockIdx.x - pair * e.chunks;
  const int slot = kSelThreads - 1 - (int)threadIdx.x;
  SelState* const states = (SelState*)e.states + (int64_t)pair * 3;
  int* const fronts = e.fronts + (int64_t)pair * 2 * e.chunks;  // above the first two digits
  const SelRow row(e, pair);
  const int part = (int)((unsigned)(row.keys + e.chunks * kSelBlock - 1) / (unsigned)(e.chunks * kSelBlock)) * kSelBlock;
  const int begin = (int)min((int64_t)chunk * part, (int64_t)row.keys), end = min(row.keys, begin + part);
  Search s = {0, 0, 0, 21};
  int target = 0, above = 0, same = 0;
  bool search = true;
  const SelBlock<kSelKeys> first(row, begin, end, wave, lane);  // (loads under the search)
  if constexpr (PHASE > 0) {
    constexpr int p = PHASE - 1;  // the digit that was counted last
    if constexpr (p > 0) {
      const SelState before = states[p - 1];
      s.bound = before.bound;
      s.need = before.need;
      s.shift = p == 1 ? 10 : 0;
      s.mask = p == 1 ? 0xffe00000u : 0xfffffc00u;
      target = before.target;
      search = before.search != 0;
    }
    if (search) {
      const int2* const hist = (const int2*)e.counts + ((int64_t)pair * 3 + p) * e.chunks * kSelThreads + slot;
      int2 all = {0, 0}, front = {0, 0};
      for (int c = 0; c < e.chunks; c += 8) {
        int2 n[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) n[u] = c + u < e.chunks ? hist[(int64_t)(c + u) * kSelThreads] : int2{0, 0};
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          all.x += n[u].x;
          all.y += n[u].y;
          front.x += c + u < chunk ? n[u].x : 0;
          front.y += c + u < chunk ? n[u].y : 0;
        }
      }
      const int total = descend(s, all.y, all.x, e.keep, wave, lane, sh);
      if constexpr (p == 0) {
        target = s.need;
        search = target < total && target > 0;
      }
      const int at = search ? sh.found[0] : -1;
      above = (2 * slot > at ? front.x : 0) + (2 * slot + 1 > at ? front.y : 0);
      if constexpr (p == 2) same = 2 * slot == at ? front.x : 2 * slot + 1 == at ? front.y : 0;
      if (search) take(s, sh);
      above = across_waves(wave_bcast(wave_prefix(above), 63), wave, lane, waves[0]).y;
      if constexpr (p < 2) {
        if (threadIdx.x == 0) {
          fronts[p * e.chunks + chunk] = above;
          if (chunk == 0) states[p] = {s.bound, s.need, target, search};
        }
      }
    } else if constexpr (p == 1) {
      if (threadIdx.x == 0 && chunk == 0) states[1] = states[0];
    }
  }
  if constexpr (PHASE < 3) {
    if (!search) return;  // (all the workgroups of the row; the histograms are not asked for)
    int2* const own = (int2*)bins + slot;
    *own = {0, 0};
    __syncthreads();
    if (begin < end) s.count(first, bins);
    for (int j = begin + kSelBlock; j < end; j += kSelBlock) s.count(SelBlock<kSelKeys>(row, j, end, wave, lane), bins);
    __syncthreads();
    ((int2*)e.counts)[(((int64_t)pair * 3 + PHASE) * e.chunks + chunk) * kSelThreads + slot] = *own;
  } else {
    // What stays in front of the chunk: above the bound, and equal to it.  (Where nothing is searched
    // for, all that the first digit counted.)
    int2 before = {fronts[chunk], 0};
    if (search) {
      before.x += fronts[e.chunks + chunk] + above;
      before.y = across_waves(wave_bcast(wave_prefix(same), 63), wave, lane, waves[1]).y;
    } else {
      s.bound = 0;
      s.need = 0;
    }
    if (target > 0) {
      if (begin < end) {
        before = write_kept(row, first, s.bound, s.need, target, before.x, before.y, wave, lane, waves[2]);
        __syncthreads();
      }
      for (int j = begin + kSelBlock; j < end; j += kSelBlock) {
        before = write_kept(row, SelBlock<kSelKeys>(row, j, end, wave, lane), s.bound, s.need, target, before.x, before.y, wave,
                            lane, waves[2]);
        __syncthreads();
      }
    }
    for (int64_t j = target + (int64_t)chunk * kSelThreads + threadIdx.x; j < row.room; j += e.chunks * kSelThreads)
      row.to_w[j] = 0.0f;
    if (row.h == 0 && chunk == 0 && threadIdx.x == 0) e.new_lens[row.b] = target;
  }
}

// Copies the rows that stay, 16 bytes a lane, kMoveRows rows of K and V at once.  Bound: memory; 256 MB
// read and written, rows of 256 bytes where they lie, take 113 us (4.7 TB/s, a large copy's rate).
constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 4;
template <int BYTES>  // of a row
__global__ void __launch_bounds__(kMoveThreads) fa_paged_move_kernel(const EvictArgs e) {
  constexpr int LANES = BYTES / 16;
  constexpr int AT = kMoveThreads / LANES;  // rows next to each other
  const PagedArgs& a = e.p;
  const unsigned pairs = (unsigned)a.batch * a.hkv;
  const int chunk = (int)(blockIdx.x / pairs);
  const int pair = (int)(blockIdx.x - chunk * pairs);
  const int b = (int)((unsigned)pair / (unsigned)a.hkv), h = pair - b * a.hkv;
  const int n = e.new_lens[b];
  const int part = (int)threadIdx.x % LANES;
  const int r0 = chunk * AT * kMoveRows + (int)threadIdx.x / LANES;
  if (chunk * AT * kMoveRows >= n) return;
  const int32_t* const kept = e.kept + (int64_t)pair * e.slots;
  const int32_t* const from = a.table + b * a.table_stride;
  const int32_t* const to = e.to_table + b * e.to_stride;
  const int in_page = (1 << a.page_shift) - 1;
  int src[kMoveRows], dst[kMoveRows], off[kMoveRows];
#pragma unroll
  for (int u = 0; u < kMoveRows; ++u) {
    const int r = min(r0 + u * AT, n - 1);
    const int j = kept[r];
    off[u] = j & in_page;
    src[u] = from[clamp_int(j >> a.page_shift, 0, a.max_pages - 1)];
    dst[u] = to[r >> a.page_shift];
    // (a row that stays is in a page, unless the table changes meanwhile)
    if (r0 + u * AT >= n || dst[u] >= a.num_pages || src[u] < 0 || src[u] >= a.num_pages) dst[u] = -1;
    src[u] = clamp_int(src[u], 0, a.num_pages - 1);
  }
  uint4v x[kMoveRows][2];
  uint8_t s[kMoveRows][2];
#pragma unroll
  for (int u = 0; u < kMoveRows; ++u) {
    x[u][0] = *(const uint4v*)(a.k + src[u] * a.kp + h * a.kh + off[u] * a.kn + 16 * part);
    x[u][1] = *(const uint4v*)(a.v + src[u] * a.vp + h * a.vh + off[u] * a.vn + 16 * part);
    if (a.ks != nullptr) {
      s[u][0] = a.ks[src[u] * a.ksp + h * a.ksh + off[u] * a.ksn];
      s[u][1] = a.vs[src[u] * a.vsp + h * a.vsh + off[u] * a.vsn];
    }
  }
#pragma unroll
  for (int u = 0; u < kMoveRows; ++u) {
    if (dst[u] < 0) continue;
    const int row = (r0 + u * AT) & in_page;
    *(uint4v*)(a.k + dst[u] * a.kp + h * a.kh + row * a.kn + 16 * part) = x[u][0];
    *(uint4v*)(a.v + dst[u] * a.vp + h * a.vh + row * a.vn + 16 * part) = x[u][1];
    if (a.ks != nullptr && part == 0) {
      a.ks[dst[u] * a.ksp + h * a.ksh + row * a.ksn] = s[u][0];
      a.vs[dst[u] * a.vsp + h * a.vsh + row * a.vsn] = s[u][1];
    }
  }
}

}  // namespace

// Workgroups of a long row: one for each block of positions, up to 64 (each adds up the histograms of
// all), and 256 in all; 1: one takes block after block; 0: one has them in its registers.  (us with 256, 512 and 4096 in all, 1024
// rows kept: 64 rows of 60000 51.5 / 59 / 59, 128 of 60000 83 / 83 / 105, of 130000 125 / 117 / 173, 256 of
// 20000 79 / 104 / 104, 512 of 30000 183 / 204 / 238.  Blocks of 2, 4 and 16 keys a thread in place of 8: 8
// rows of 131072 93, 58 and 71 for 56.)
static int evict_chunks(const EvictArgs& e) {
  const int64_t room = (int64_t)e.p.max_pages << e.p.page_shift, pairs = (int64_t)e.p.batch * e.p.hkv;
  if (room <= kSelBlock) return 0;
  return (int)std::max<int64_t>(1, std::min<int64_t>({64, (room + kSelBlock - 1) / kSelBlock, 256 / pairs}));
}
static int64_t kept_bytes(const EvictArgs& e) {
  return ((int64_t)e.p.batch * e.p.hkv * e.slots * (int64_t)sizeof(int32_t) + 15) & ~(int64_t)15;
}

int64_t evict_workspace_bytes(const EvictArgs& e) {
  const int64_t pairs = (int64_t)e.p.batch * e.p.hkv, chunks = evict_chunks(e);
  if (chunks <= 1) return kept_bytes(e);
  const int64_t row = 3 * chunks * kSelBins * (int64_t)sizeof(int) + 3 * (int64_t)sizeof(SelState) + 2 * chunks * (int64_t)sizeof(int);
  return (kept_bytes(e) + pairs * row + 15) & ~(int64_t)15;
}

int launch_evict(const EvictArgs& args, int head_dim, void* workspace, hipStream_t stream) {
  EvictArgs e = args;
  e.chunks = evict_chunks(e);
  e.kept = static_cast<int32_t*>(workspace);
  e.counts = reinterpret_cast<int*>(static_cast<char*>(workspace) + kept_bytes(e));
  e.states = e.counts + (int64_t)e.p.batch * e.p.hkv * 3 * e.chunks * kSelBins;
  e.fronts = e.states + (int64_t)e.p.batch * e.p.hkv * 3 * (int64_t)(sizeof(SelState) / sizeof(int));
  const int64_t pairs = (int64_t)e.p.batch * e.p.hkv;
  const dim3 threads(kSelThreads);
  if (e.chunks == 0) {
    const int64_t room = (int64_t)e.p.max_pages << e.p.page_shift;
    const dim3 rows((unsigned)pairs);
    if (room <= 2 * kSelThreads) hipLaunchKernelGGL(fa_paged_select_kernel<2>, rows, threads, 0, stream, e);
    else if (room <= 4 * kSelThreads) hipLaunchKernelGGL(fa_paged_select_kernel<4>, rows, threads, 0, stream, e);
    else hipLaunchKernelGGL(fa_paged_select_kernel<kSelKeys>, rows, threads, 0, stream, e);
  } else if (e.chunks == 1) {
    hipLaunchKernelGGL(fa_paged_select_blocks_kernel, dim3((unsigned)pairs), threads, 0, stream, e);
  } else {
    const dim3 rows((unsigned)(pairs * e.chunks));
    hipLaunchKernelGGL(fa_paged_select_long_kernel<0>, rows, threads, 0, stream, e);
    hipLaunchKernelGGL(fa_paged_select_long_kernel<1>, rows, threads, 0, stream, e);
    hipLaunchKernelGGL(fa_paged_select_long_kernel<2>, rows, threads, 0, stream, e);
    hipLaunchKernelGGL(fa_paged_select_long_kernel<3>, rows, threads, 0, stream, e);
  }
  if (e.slots == 0 || e.p.num_pages == 0) return 0;
  const int bytes = head_dim * (e.p.ks != nullptr ? 1 : 2);
  const int per = kMoveThreads / (bytes / 16) * kMoveRows;
  const dim3 grid((unsigned)((e.slots + per - 1) / per * pairs));
#define FA_MOVE(B) hipLaunchKernelGGL(fa_paged_move_kernel<B>, grid, dim3(kMoveThreads), 0, stream, e)
  if (bytes == 64) FA_MOVE(64);
  else if (bytes == 128) FA_MOVE(128);
  else FA_MOVE(256);
#undef FA_MOVE
  return 0;
}

}  // namespace fa
