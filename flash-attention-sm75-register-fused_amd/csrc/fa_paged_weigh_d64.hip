// The weights attention gave a paged cache's rows, head_dim 64, 16-bit rows (see fa_paged_weigh.h).
#include "fa_paged_weigh.h"

namespace fa {
template void launch_weigh_few<64, false, false>(const WeighArgs&, int, int64_t, hipStream_t);
template void launch_weigh_few<64, true, false>(const WeighArgs&, int, int64_t, hipStream_t);
template void launch_weigh_chunk<64, false, false>(const WeighArgs&, int64_t, hipStream_t);
template void launch_weigh_chunk<64, true, false>(const WeighArgs&, int64_t, hipStream_t);
}  // namespace fa
