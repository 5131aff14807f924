// Attention over a paged cache, head_dim 128, binary16, 16-bit rows (see fa_paged_attn.h, fa_paged_chunk.h).
#include "fa_paged_attn.h"
#include "fa_paged_chunk.h"

namespace fa {
template void launch_paged_attn<128, false, false>(const PagedArgs&, int, int64_t, hipStream_t);
template void launch_paged_chunk<128, false, false>(const PagedArgs&, int64_t, hipStream_t);
}  // namespace fa
