// Attention over a paged cache: the plan, the launches, and the kernel that merges
// the partials of cut units (fa_paged_attn.h).
#include <algorithm>
#include <numeric>

#include "fa_internal.h"
#include "fa_paged_attn.h"
#include "fa_paged_chunk.h"

namespace fa {

// The instances of fa_paged_d*.hip.
#define FA_PAGED_EXTERN(D, BF, F8)                                                                     \
  extern template void launch_paged_attn<D, BF, F8, 0>(const PagedArgs&, int, int64_t, hipStream_t);      \
  extern template void launch_paged_attn<D, BF, F8, kOwn>(const PagedShared&, int, int64_t, hipStream_t); \
  extern template void launch_paged_attn<D, BF, F8, kBoth>(const PagedShared&, int, int64_t, hipStream_t); \
  extern template void launch_paged_chunk<D, BF, F8, 0>(const PagedArgs&, int64_t, hipStream_t);          \
  extern template void launch_paged_chunk<D, BF, F8, kPrefix>(const PagedShared&, int64_t, hipStream_t);  \
  extern template void launch_paged_chunk<D, BF, F8, kOwn>(const PagedShared&, int64_t, hipStream_t);
FA_PAGED_EXTERN(64, false, false) FA_PAGED_EXTERN(64, true, false)
FA_PAGED_EXTERN(64, false, true) FA_PAGED_EXTERN(64, true, true)
FA_PAGED_EXTERN(128, false, false) FA_PAGED_EXTERN(128, true, false)
FA_PAGED_EXTERN(128, false, true) FA_PAGED_EXTERN(128, true, true)
#undef FA_PAGED_EXTERN

namespace {
int64_t partial_bytes(int rows, int head_dim) {  // of one workgroup: two records and their flags
  return 2 * (rows * (head_dim + 2ll) * (int64_t)sizeof(float) + (int64_t)sizeof(uint64_t));
}
constexpr int64_t kLastCacheBytes = 256 << 20;
constexpr int kOwnShort = 640, kOwnShare = 1024;
constexpr int64_t kJoinBytes = 128 << 20, kJoinAgain = 96 << 20;
constexpr int64_t kCombineWord = 16;  // behind them, to keep workspaces whole 16 bytes
}  // namespace

// Whether a line of `units` units stays below 2^31 tiles.
static bool fits_line(const PagedArgs& a, int64_t units, int tile, int ahead) {
  const int64_t tiles = (((int64_t)a.max_pages << a.page_shift) + tile - 1) / tile;
  return units * (ahead + std::max<int64_t>(1, tiles)) <= INT32_MAX - 64;  // (room to round up)
}

// V non-temporally, where one block of a sequence reads it and the tables have room for
// more than stays in the 256 MB cache behind the L2s from one step to the next (us without
// and with: 16 tokens each of 16 sequences of 4096 to 8192 keys, 32 over 8 heads d128, 400
// MB 99.9 / 81.2, of 32 in 8 bits 118.7 / 108.8, 10 of 48 of 8192 to 16384 d64, 302 MB 68.2 /
// 63.8; in the cache: 16 of those 33.0 / 35.4, 16 in 8 bits d128 72.5 / 73.7).
static bool streams_v(const PagedArgs& a, int head_dim, int64_t max_query_len) {
  const int64_t room = ((int64_t)a.max_pages << a.page_shift) * a.batch * a.hkv;
  return max_query_len * a.group <= kChunkRows &&
         room > kLastCacheBytes / (2 * head_dim * (a.ks != nullptr ? 1 : 2));
}

// Units of 128 rows, cut into pieces where they may be fewer than the GPU runs at once.
static PagedPlan plan_chunks(const PagedArgs& a, int head_dim, int64_t max_query_len,
                             int64_t workspace_bytes) {
  PagedPlan p{};
  p.chunk = true;
  p.rows = kChunkRows;
  p.classes = std::gcd(a.hkv, kNumXcds);
  // A class's units, the last block of each sequence not full: at least and at most.
  const int64_t heads = a.hkv / p.classes, rows = (int64_t)a.tokens * a.group;
  const int64_t least = heads * ((rows + p.rows - 1) / p.rows);
  p.units = (int)(heads * ((rows + (p.rows - 1ll) * std::min(a.batch, a.tokens)) / p.rows));
  const int64_t record = partial_bytes(p.rows, head_dim) * p.classes;
  const int64_t wgs = std::min<int64_t>(p.resident = resident_fused_workgroups() / p.classes,
                                        (workspace_bytes - kCombineWord) / record);
  p.split = least < wgs && fits_line(a, p.units, kBlockN, kChunkAhead);
  // (us with the second kernel and without: 512 tokens of one sequence among 15 single
  // ones d128 60.9 / 59.1, one prompt of 700 tokens 21.8 / 20.3, three of 777 tokens d64 8 bits 50.7 / 47.5)
  const bool few = least * (chunk_pieces(head_dim) - 1) < wgs;
  p.combine = p.split && few;
  p.stream_v = streams_v(a, head_dim, max_query_len);
  p.pieces = few ? 0 : chunk_pieces(head_dim);
  p.wgs = p.split ? (int)wgs : p.units;
  p.workspace_bytes = p.split ? p.wgs * record + kCombineWord : 0;
  return p;
}

PagedPlan plan_paged(const PagedArgs& a, int head_dim, int64_t max_query_len,
                     int64_t workspace_bytes, int stage) {
  if (max_query_len * a.group > 32) return plan_chunks(a, head_dim, max_query_len, workspace_bytes);
  PagedPlan p{};
  p.rows = max_query_len * a.group <= 16 ? 16 : 32;
  p.classes = std::gcd(a.hkv, kNumXcds);
  // Two workgroups a CU.  Head_dim 64 and 8-bit instances have room for three or four;
  // with those a launch took longer (us, two against three: 32 sequences to 8192 keys d128
  // 8 bits 68.3 / 70.7, 4 rows over 131072 keys 49.3 / 51.6, 16 to 32768 keys d64 39.6 /
  // 41.0, 8 bits 32.1 / 32.4; 8 to 8192 keys without grouping d128 8 bits 29.3 / 33.5):
  // stretches are shorter and more of them end inside a unit.
  const int64_t resident = resident_fused_workgroups();
  const int64_t room = (workspace_bytes - kCombineWord) / (partial_bytes(p.rows, head_dim) * p.classes);
  p.wgs = (int)std::min(resident / p.classes, room);
  // Units of a class: blocks of rows, the last of each sequence not full.
  const int64_t blocks =
      a.cu == nullptr ? (int64_t)a.batch * ((a.group + p.rows - 1) / p.rows)
                      : (int64_t)a.tokens * a.group / p.rows + std::min(a.batch, a.tokens);
  p.units = (int)(a.hkv / p.classes * blocks);
  // (Of very many units a workgroup each is balanced enough.)
  p.split = p.wgs > 0 && p.units <= 16 * resident / p.classes && fits_line(a, p.units, kPTile, kPAhead);
  // Behind a shared prefix the own keys are often few, and cutting them (a plan by tiles, records, a merge: about 8
  // us) costs more than it balances: up to 640 keys whatever the units, and more keys the more of the GPU the
  // units fill, twice as many more where a row is half as wide.  us of both launches, units whole and cut, of
  // sequences of a tenth to all of the keys (and of as many each), caches cold:
  //   32 over 8 heads d128, 16 bits   512 keys     1024        1536        2048         border
  //     2 sequences                   22.9 / 24.0  27.8 / 22.0 32.8 / 22.5 37.5 / 22.8   672
  //     (each as long)                23.0 / 22.6  27.9 / 22.6 32.9 / 22.9
  //     16                            23.4 / 28.2  28.7 / 31.2 35.5 / 33.1 41.6 / 36.2   896
  //     (each as long)                23.8 / 25.0  31.6 / 32.4 38.1 / 37.2 44.7 / 42.3
  //     32                            25.6 / 31.5  34.0 / 37.3 40.6 / 42.8 48.5 / 48.1  1152
  //     64                            35.7 / 44.6  50.6 / 53.5 63.8 / 66.1 79.7 / 75.9  1664
  //     96                            47.8 / 49.0  67.3 / 65.8 88.8 / 83.4              1664
  //   8 bits
  //     16                            25.6 / 30.2  30.7 / 32.1 35.6 / 37.0 40.8 / 34.7  1152
  //     48                            31.3 / 37.1  37.7 / 40.2 44.2 / 47.6 48.5 / 54.0  2176 (4096: 74.6 / 69.0)
  //     64                            31.6 / 41.6  39.7 / 48.4 47.6 / 55.4 55.9 / 60.2  2688 (4096: 82.9 / 79.5)
  //   14 over 2 heads d64, 16 bits
  //     4                             17.4 / 26.1  19.8 / 23.9 22.6 / 24.3 25.0 / 22.6   672
  //     (each as long)                17.8 / 19.2  20.4 / 19.3 22.9 / 19.1 25.4 / 19.4
  //     128                           20.1 / 30.1  23.3 / 31.7 27.3 / 34.5 31.7 / 36.6  1664 (4096: 45.3 / 47.1)
  if (stage == kOwn && p.split) {
    const int64_t longest = (int64_t)a.max_pages << a.page_shift;
    const int share = head_dim == 128 && a.ks == nullptr ? kOwnShare : 2 * kOwnShare;
    if (longest <= kOwnShort + (int64_t)share * std::min(p.units, p.wgs) / p.wgs) p.split = false;
  }
  if (!p.split) p.wgs = p.units;
  p.workspace_bytes =
      p.split ? (int64_t)p.wgs * p.classes * partial_bytes(p.rows, head_dim) + kCombineWord : 0;
  // What the longest unit the tables have room for may be cut into.
  const int64_t tiles = (((int64_t)a.max_pages << a.page_shift) + kPTile - 1) / kPTile;
  const int64_t pieces = PagedStretch<kPMinTiles>::most_pieces(tiles, p.wgs);
  p.y = (int)std::min<int64_t>(p.rows, max_query_len * a.group);
  // (max_query_len may be wrong: rows are then up to p.rows)
  p.combine = p.split && !paged_merges_itself((int)pieces, a.cu == nullptr ? p.y : p.rows, head_dim);
  return p;
}

// Up to 32 rows of a KV head, where every sequence reads its prefix itself: what is read again comes mostly from the
// caches, at 12 TB/s, which while the tables have room for no more than 128 MB so read, 96 MB of it again, costs
// less than a launch over the prefixes, their records and what joins them; up to 128 MB again where a second launch would cut
// its own keys, whose plan and merge one launch has anyway.  One launch's time over that of two, caches cold, at
// 1634 sizes (2 to 64 sequences of 100 to 1800 own keys, 1 or 4 prefixes of 128 to 16000, nine layouts; least, median, most):
//   MB read again           up to 16     16 .. 48     48 .. 80     80 .. 100    100 .. 130   130 .. 200
//     own keys whole        .49 .81 1.30 .57 .87 1.14 .64 .95 1.20 .81 .96 1.19 .80 1.03 1.32 .88 1.15 1.41
//     cut                   .38 .57 .84  .57 .67 .83  .60 .75 .88  .68 .82 .99  .70 .87 .93   .89 1.02 1.09
// (The rule's choice is 0.8% slower than the better of the two on average; at the most 34.7 us where two launches take 26.7, with 8
// tokens each of 24 sequences of 100 to 300 keys behind 4 prefixes of 128.)
bool joins_prefixes(const PagedShared& own, int head_dim, int64_t max_query_len) {
  if (max_query_len * own.group > 32 || own.batch > 64 || own.prefixes > 63) return false;
  const int64_t bytes = ((int64_t)own.pre_pages << own.page_shift) * own.hkv * 2 * head_dim * (own.ks != nullptr ? 1 : 2);
  return bytes * own.batch <= kJoinBytes &&
         (bytes * (own.batch - own.prefixes) <= kJoinAgain ||
          plan_paged(own, head_dim, max_query_len, INT64_MAX, kOwn).split);
}

PagedPlan plan_joined(const PagedShared& own, int head_dim, int64_t max_query_len, int64_t workspace_bytes) {
  PagedArgs a = own;  // as wide as both tables (and a tile that the prefix's last leaves open)
  a.max_pages += own.pre_pages + (kPTile >> std::min(a.page_shift, 5));
  return plan_paged(a, head_dim, max_query_len, workspace_bytes);
}

PagedPlan plan_prefix(const PagedShared& a, int head_dim, int64_t max_queries) {
  PagedPlan p{};
  p.chunk = p.split = true;
  p.rows = kChunkRows;
  p.classes = std::gcd(a.hkv, kNumXcds);
  const int64_t rows = (int64_t)a.tokens * a.group;
  p.units = (int)(a.hkv / p.classes * ((rows + (p.rows - 1ll) * std::min(a.batch, a.tokens)) / p.rows));
  // A workgroup for each unit, or, while they are fewer than run at once, for each piece.
  const int64_t tiles = (((int64_t)a.max_pages << a.page_shift) + kBlockN - 1) / kBlockN;
  const int64_t pieces = std::max<int64_t>(1, (tiles + kPrefixMinTiles - 1) / kPrefixMinTiles);
  const int64_t resident = resident_fused_workgroups() / p.classes;
  p.wgs = (int)std::max<int64_t>(p.units, std::min<int64_t>(resident, p.units * pieces));
  p.stream_v = streams_v(a, head_dim, max_queries);
  p.workspace_bytes = (int64_t)p.wgs * p.classes * p.rows * (head_dim + 2) * (int64_t)sizeof(float) + 16ll * a.batch;
  return p;
}

template <int D, bool BF16, int STAGE>
void launch_paged_combine(const StageArgs<STAGE>& a, int rows, int y, hipStream_t stream) {
  if (STAGE != kBoth && rows == kChunkRows) {
    hipLaunchKernelGGL((fa_paged_chunk_combine_kernel<D, BF16, STAGE>),
                       dim3((unsigned)(a.wgs * a.classes), kChunkCombineY), dim3(kThreads), 0, stream, a);
    return;
  }
  const dim3 g((unsigned)(a.units * a.classes), (unsigned)y);
  if (rows == 16)
    hipLaunchKernelGGL((fa_paged_combine_kernel<D, BF16, 1, STAGE>), g, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((fa_paged_combine_kernel<D, BF16, 2, STAGE>), g, dim3(kThreads), 0, stream, a);
}

template <int D, bool BF16, bool FP8, int STAGE>
static void launch_planned(const StageArgs<STAGE>& a, const PagedPlan& plan, hipStream_t stream) {
  const int64_t grid = (int64_t)plan.wgs * plan.classes;
  if constexpr (STAGE == kPrefix) {
    launch_paged_chunk<D, BF16, FP8, STAGE>(a, grid, stream);
    return;
  } else if constexpr (STAGE == kBoth) {
    launch_paged_attn<D, BF16, FP8, STAGE>(a, plan.rows, grid, stream);
  } else if (plan.chunk) {
    launch_paged_chunk<D, BF16, FP8, STAGE>(a, grid, stream);
  } else {
    launch_paged_attn<D, BF16, FP8, STAGE>(a, plan.rows, grid, stream);
  }
  if (plan.combine) launch_paged_combine<D, BF16, STAGE>(a, plan.rows, plan.y, stream);
}
template <int D, int STAGE>
static void launch_typed(const StageArgs<STAGE>& a, const PagedPlan& plan, hipStream_t stream) {
  if (a.ks != nullptr) {
    if (a.bf16) launch_planned<D, true, true, STAGE>(a, plan, stream);
    else launch_planned<D, false, true, STAGE>(a, plan, stream);
  } else {
    if (a.bf16) launch_planned<D, true, false, STAGE>(a, plan, stream);
    else launch_planned<D, false, false, STAGE>(a, plan, stream);
  }
}

// A plan's fields, and what follows from the sizes.
static void set_plan(PagedArgs& a, const PagedPlan& plan) {
  a.classes = plan.classes;  // (divides kNumXcds, a power of two)
  a.class_shift = __builtin_ctz(plan.classes);
  a.heads = a.hkv / a.classes;
  a.inv_group = 1.0f / (float)a.group;
  a.rescale = kRescaleLog2 / a.c;
  a.wgs = plan.wgs;
  a.units = plan.units;
  a.resident = plan.resident;
  a.pieces = plan.pieces;
  a.stream_v = plan.stream_v ? 1 : 0;
  a.split = plan.split ? 1 : 0;
}

template <int STAGE>
static void launch_sized(const StageArgs<STAGE>& a, const PagedPlan& plan, int head_dim, hipStream_t stream) {
  if (head_dim == 64) launch_typed<64, STAGE>(a, plan, stream);
  else launch_typed<128, STAGE>(a, plan, stream);
}

int launch_paged_prefix(PagedShared& prefix, PagedShared& own, const PagedPlan& plan, int head_dim, void* workspace,
                        hipStream_t stream) {
  set_plan(prefix, plan);
  const int64_t records = (int64_t)plan.wgs * plan.classes;
  prefix.joint_records = own.joint_records = (int)records;
  prefix.joint_info = own.joint_info = static_cast<int32_t*>(workspace);
  prefix.joint_o = own.joint_o = reinterpret_cast<float*>(prefix.joint_info + 4ll * prefix.batch);
  prefix.joint_ml = own.joint_ml = prefix.joint_o + records * plan.rows * head_dim;
  launch_sized<kPrefix>(prefix, plan, head_dim, stream);
  return 0;
}

template <int STAGE>
static void launch_attention(const StageArgs<STAGE>& args, const PagedPlan& plan, int head_dim, void* workspace,
                             hipStream_t stream) {
  StageArgs<STAGE> a = args;
  set_plan(a, plan);
  const int64_t grid = (int64_t)plan.wgs * plan.classes;
  if (plan.split) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + 2 * grid * plan.rows * head_dim;
    a.flags = reinterpret_cast<uint64_t*>(a.part_ml + 2 * grid * plan.rows * 2);
    a.mark = merge_mark(a.flags, 2 * grid + 1, stream);
  }
  launch_sized<STAGE>(a, plan, head_dim, stream);
}

int launch_paged_attention(const PagedArgs& a, const PagedPlan& plan, int head_dim,
                           void* workspace, hipStream_t stream) {
  launch_attention<0>(a, plan, head_dim, workspace, stream);
  return 0;
}
int launch_paged_attention(const PagedShared& own, const PagedPlan& plan, int head_dim,
                           void* workspace, hipStream_t stream) {
  launch_attention<kOwn>(own, plan, head_dim, workspace, stream);
  return 0;
}
int launch_paged_joined(const PagedShared& own, const PagedPlan& plan, int head_dim, void* workspace,
                        hipStream_t stream) {
  launch_attention<kBoth>(own, plan, head_dim, workspace, stream);
  return 0;
}

}  // namespace fa
