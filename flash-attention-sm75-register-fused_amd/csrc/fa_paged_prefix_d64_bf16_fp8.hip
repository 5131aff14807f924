// Attention behind shared prefixes of a paged cache, head_dim 64, bfloat16, e4m3 rows (see fa_paged_attn.h, fa_paged_chunk.h).
#include "fa_paged_attn.h"
#include "fa_paged_chunk.h"

namespace fa {
template void launch_paged_attn<64, true, true, kOwn>(const PagedShared&, int, int64_t, hipStream_t);
template void launch_paged_attn<64, true, true, kBoth>(const PagedShared&, int, int64_t, hipStream_t);
template void launch_paged_chunk<64, true, true, kPrefix>(const PagedShared&, int64_t, hipStream_t);
template void launch_paged_chunk<64, true, true, kOwn>(const PagedShared&, int64_t, hipStream_t);
}  // namespace fa
