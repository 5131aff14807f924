// The weights attention gave a paged cache's rows, head_dim 128, 16-bit rows (see fa_paged_weigh.h).
#include "fa_paged_weigh.h"

namespace fa {
template void launch_weigh_few<128, false, false>(const WeighArgs&, int, int64_t, hipStream_t);
template void launch_weigh_few<128, true, false>(const WeighArgs&, int, int64_t, hipStream_t);
template void launch_weigh_chunk<128, false, false>(const WeighArgs&, int64_t, hipStream_t);
template void launch_weigh_chunk<128, true, false>(const WeighArgs&, int64_t, hipStream_t);
}  // namespace fa
