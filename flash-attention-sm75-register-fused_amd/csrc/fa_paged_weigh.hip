// The weights attention gave a paged cache's rows: the plan and the launches (fa_paged_weigh.h).
#include <algorithm>

#include "fa_internal.h"
#include "fa_paged_weigh.h"

namespace fa {

#define FA_WEIGH_EXTERN(D, BF, F8) \
  extern template void launch_weigh_few<D, BF, F8>(const WeighArgs&, int, int64_t, hipStream_t);
FA_WEIGH_EXTERN(64, false, false) FA_WEIGH_EXTERN(64, true, false)
FA_WEIGH_EXTERN(64, false, true) FA_WEIGH_EXTERN(64, true, true)
FA_WEIGH_EXTERN(128, false, false) FA_WEIGH_EXTERN(128, true, false)
FA_WEIGH_EXTERN(128, false, true) FA_WEIGH_EXTERN(128, true, true)
#undef FA_WEIGH_EXTERN

WeighPlan plan_weigh(const WeighArgs& a, int head_dim, int64_t max_query_len) {
  (void)head_dim;
  WeighPlan p{};
  p.rows = max_query_len * a.p.group <= 16 ? 16 : 32;
  const int64_t pairs = (int64_t)a.p.batch * a.p.hkv;
  const int64_t tiles = ((int64_t)a.max_len + kWTile - 1) / kWTile;
  // Tiles of a wave: one where there are few, at most eight.
  const int64_t waves = (int64_t)resident_fused_workgroups() * 8;
  p.run = (int)std::max<int64_t>(1, std::min<int64_t>(8, tiles * pairs / waves));
  p.grid = ((tiles + p.run - 1) / p.run * pairs + kWaves - 1) / kWaves;
  return p;
}

int launch_weigh(const WeighArgs& args, const WeighPlan& plan, int head_dim, hipStream_t stream) {
  WeighArgs a = args;
  a.run = plan.run;
  a.p.inv_group = 1.0f / (float)a.p.group;
  const bool fp8 = a.p.ks != nullptr;
#define FA_WEIGH(D)                                                             \
  if (fp8) {                                                                    \
    if (a.p.bf16) launch_weigh_few<D, true, true>(a, plan.rows, plan.grid, stream);   \
    else launch_weigh_few<D, false, true>(a, plan.rows, plan.grid, stream);     \
  } else {                                                                      \
    if (a.p.bf16) launch_weigh_few<D, true, false>(a, plan.rows, plan.grid, stream);  \
    else launch_weigh_few<D, false, false>(a, plan.rows, plan.grid, stream);    \
  }
  if (head_dim == 64) { FA_WEIGH(64) } else { FA_WEIGH(128) }
#undef FA_WEIGH
  return 0;
}

}  // namespace fa
