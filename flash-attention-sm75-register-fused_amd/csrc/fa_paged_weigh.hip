// The weights attention gave a paged cache's rows: the plan and the launches (fa_paged_weigh.h).
#include <algorithm>

#include "fa_internal.h"
#include "fa_paged_weigh.h"

namespace fa {

#define FA_WEIGH_EXTERN(D, BF, F8) \
  extern template void launch_weigh_few<D, BF, F8>(const WeighArgs&, int, int64_t, hipStream_t); \
  extern template void launch_weigh_chunk<D, BF, F8>(const WeighArgs&, int64_t, hipStream_t);
FA_WEIGH_EXTERN(64, false, false) FA_WEIGH_EXTERN(64, true, false)
FA_WEIGH_EXTERN(64, false, true) FA_WEIGH_EXTERN(64, true, true)
FA_WEIGH_EXTERN(128, false, false) FA_WEIGH_EXTERN(128, true, false)
FA_WEIGH_EXTERN(128, false, true) FA_WEIGH_EXTERN(128, true, true)
#undef FA_WEIGH_EXTERN

WeighPlan plan_weigh(const WeighArgs& a, int64_t max_query_len, int64_t workspace_bytes) {
  WeighPlan p{};
  const int64_t pairs = (int64_t)a.p.batch * a.p.hkv;
  if (max_query_len * a.p.group > 32) {
    // A workgroup for each block of keys there is room for, and as many as run at once for those that
    // are cut (fewer units than that, of at most 2^27 rows in all: tiles on the line have 31 bits).
    const int wgs = resident_fused_workgroups();
    const int64_t bytes = (3ll * kWBlock * 4 + 2 * 8) * wgs;
    p.wgs = workspace_bytes >= bytes ? wgs : 0;
    p.workspace_bytes = p.wgs > 0 ? bytes : 0;
    p.grid = ((int64_t)a.max_len + kWBlock - 1) / kWBlock * pairs + p.wgs;
    return p;
  }
  p.rows = max_query_len * a.p.group <= 16 ? 16 : 32;
  // Waves: four a SIMD, of 32 rows three, or one for each tile there is room for; and those that
  // clear what is behind the keys.
  const int64_t tiles = ((int64_t)a.max_len + kWTile - 1) / kWTile * pairs;
  const int64_t blocks = ((int64_t)a.max_len + kWBlock - 1) / kWBlock * pairs;
  p.waves = (int)std::min<int64_t>(tiles, (int64_t)resident_fused_workgroups() * (p.rows == 16 ? 8 : 6));
  p.grid = (p.waves + (a.add ? 0 : blocks) + kWaves - 1) / kWaves;
  return p;
}

template <int D, bool BF16, bool FP8>
static void launch_planned(const WeighArgs& a, const WeighPlan& plan, hipStream_t stream) {
  if (plan.rows == 0) launch_weigh_chunk<D, BF16, FP8>(a, plan.grid, stream);
  else launch_weigh_few<D, BF16, FP8>(a, plan.rows, plan.grid, stream);
}
template <int D>
static void launch_typed(const WeighArgs& a, const WeighPlan& plan, hipStream_t stream) {
  if (a.p.ks != nullptr) {
    if (a.p.bf16) launch_planned<D, true, true>(a, plan, stream);
    else launch_planned<D, false, true>(a, plan, stream);
  } else {
    if (a.p.bf16) launch_planned<D, true, false>(a, plan, stream);
    else launch_planned<D, false, false>(a, plan, stream);
  }
}

int launch_weigh(const WeighArgs& args, const WeighPlan& plan, int head_dim, void* workspace, hipStream_t stream) {
  WeighArgs a = args;
  a.waves = plan.waves;
  a.wgs = plan.wgs;
  a.p.inv_group = 1.0f / (float)a.p.group;
  if (plan.wgs > 0) {
    a.partial = static_cast<float*>(workspace);
    a.flags = reinterpret_cast<uint64_t*>(a.partial + 3ll * plan.wgs * kWBlock);
    a.mark = merge_mark(a.flags, 2 * plan.wgs, stream);
  }
  if (head_dim == 64) launch_typed<64>(a, plan, stream);
  else launch_typed<128>(a, plan, stream);
  return 0;
}

}  // namespace fa
