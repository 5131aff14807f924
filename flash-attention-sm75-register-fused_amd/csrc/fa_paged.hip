// Attention over a paged cache: the plan, the launches, and the kernel that merges
// the partials of cut units (fa_paged_attn.h).
#include <algorithm>
#include <numeric>

#include "fa_internal.h"
#include "fa_paged_attn.h"
#include "fa_paged_chunk.h"

namespace fa {

// The instances of fa_paged_d*.hip.
#define FA_PAGED_EXTERN(D, BF, F8) \
  extern template void launch_paged_attn<D, BF, F8>(const PagedArgs&, int, int64_t, hipStream_t); \
  extern template void launch_paged_chunk<D, BF, F8>(const PagedArgs&, int64_t, hipStream_t);
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
constexpr int64_t kCombineWord = 16;  // behind them, to keep workspaces whole 16 bytes
}  // namespace

// Whether a line of `units` units stays below 2^31 tiles.
static bool fits_line(const PagedArgs& a, int64_t units, int tile, int ahead) {
  const int64_t tiles = (((int64_t)a.max_pages << a.page_shift) + tile - 1) / tile;
  return units * (ahead + std::max<int64_t>(1, tiles)) <= INT32_MAX - 64;  // (room to round up)
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
  // V non-temporally, where one block of a sequence reads it and the tables have room for
  // more than stays in the 256 MB cache behind the L2s from one step to the next (us without
  // and with: 16 tokens each of 16 sequences of 4096 to 8192 keys, 32 over 8 heads d128, 400
  // MB 99.9 / 81.2, of 32 in 8 bits 118.7 / 108.8, 10 of 48 of 8192 to 16384 d64, 302 MB 68.2 /
  // 63.8; in the cache: 16 of those 33.0 / 35.4, 16 in 8 bits d128 72.5 / 73.7).
  const int64_t room = ((int64_t)a.max_pages << a.page_shift) * a.batch * a.hkv;
  p.stream_v = max_query_len * a.group <= kChunkRows &&
               room > kLastCacheBytes / (2 * head_dim * (a.ks != nullptr ? 1 : 2));
  p.pieces = few ? 0 : chunk_pieces(head_dim);
  p.wgs = p.split ? (int)wgs : p.units;
  p.workspace_bytes = p.split ? p.wgs * record + kCombineWord : 0;
  return p;
}

PagedPlan plan_paged(const PagedArgs& a, int head_dim, int64_t max_query_len,
                     int64_t workspace_bytes) {
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

template <int D, bool BF16>
void launch_paged_combine(const PagedArgs& a, int rows, int y, hipStream_t stream) {
  if (rows == kChunkRows) {
    hipLaunchKernelGGL((fa_paged_chunk_combine_kernel<D, BF16>),
                       dim3((unsigned)(a.wgs * a.classes), kChunkCombineY), dim3(kThreads), 0, stream, a);
    return;
  }
  const dim3 g((unsigned)(a.units * a.classes), (unsigned)y);
  if (rows == 16)
    hipLaunchKernelGGL((fa_paged_combine_kernel<D, BF16, 1>), g, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((fa_paged_combine_kernel<D, BF16, 2>), g, dim3(kThreads), 0, stream, a);
}

int launch_paged_attention(const PagedArgs& args, const PagedPlan& plan, int head_dim,
                           void* workspace, hipStream_t stream) {
  PagedArgs a = args;
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
  const int64_t grid = (int64_t)plan.wgs * plan.classes;
  if (plan.split) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + 2 * grid * plan.rows * head_dim;
    a.flags = reinterpret_cast<uint64_t*>(a.part_ml + 2 * grid * plan.rows * 2);
    a.mark = merge_mark(a.flags, 2 * grid + 1, stream);
  }
  const bool fp8 = a.ks != nullptr;
#define FA_PAGED(D)                                                                     \
  if (plan.chunk) {                                                                     \
    if (fp8) {                                                                          \
      if (a.bf16) launch_paged_chunk<D, true, true>(a, grid, stream);                   \
      else launch_paged_chunk<D, false, true>(a, grid, stream);                         \
    } else {                                                                            \
      if (a.bf16) launch_paged_chunk<D, true, false>(a, grid, stream);                  \
      else launch_paged_chunk<D, false, false>(a, grid, stream);                        \
    }                                                                                   \
  } else if (fp8) {                                                                     \
    if (a.bf16) launch_paged_attn<D, true, true>(a, plan.rows, grid, stream);           \
    else launch_paged_attn<D, false, true>(a, plan.rows, grid, stream);                 \
  } else {                                                                              \
    if (a.bf16) launch_paged_attn<D, true, false>(a, plan.rows, grid, stream);          \
    else launch_paged_attn<D, false, false>(a, plan.rows, grid, stream);                \
  }                                                                                     \
  if (plan.combine) {                                                                   \
    if (a.bf16) launch_paged_combine<D, true>(a, plan.rows, plan.y, stream);            \
    else launch_paged_combine<D, false>(a, plan.rows, plan.y, stream);                  \
  }
  if (head_dim == 64) { FA_PAGED(64) } else { FA_PAGED(128) }
#undef FA_PAGED
  return 0;
}

}  // namespace fa
