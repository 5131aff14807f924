// The plan of attention over a paged cache, for tests/test_paged_plan.py (its host half)
// and tests/test_gpu_paged_merge.py (what a workgroup makes of the lengths on the device).
#include "fa_paged_attn.h"
#include "fa_paged_chunk.h"

namespace fa {
namespace {

// Into out[i], i < count: the number of pieces that unit i of a class is cut into (units in
// the order of its line).  One wave.
template <int R, int T, int H, class Cut>
__device__ void pieces_of_units(const PagedArgs& a, int* out, int count, Cut cut) {
  const int lane = threadIdx.x & 63;
  const PagedLine<R, T, H> line(a, lane, true);
  const auto stretch = cut(line);
  int i = 0;
  for (int b = 0; b < a.batch; ++b) {
    const PagedSeq s = line.seq(b);
    const int start = line.start_of(b), len = line.unit_of(s);
    for (int u = 0; u < a.heads * paged_blocks<R>(a, s); ++u, ++i) {
      const PagedPieces pieces(stretch, a.wgs, start + u * len + line.ahead, start + (u + 1) * len);
      if (lane == 0 && i < count) out[i] = pieces.count;
    }
  }
}

template <int D>
__global__ void __launch_bounds__(64) probe_kernel(const PagedArgs a, int rows, int* out, int count) {
  auto few = [&](const auto& line) { return paged_stretch(a, line); };
  auto chunk = [&](const auto& line) { return chunk_stretch<D>(a, line); };
  if (rows == 16) pieces_of_units<16, kPTile, kPAhead>(a, out, count, few);
  else if (rows == 32) pieces_of_units<32, kPTile, kPAhead>(a, out, count, few);
  else pieces_of_units<kChunkRows, kBlockN, kChunkAhead>(a, out, count, chunk);
}

PagedArgs sizes(int hkv, int group, int batch, int tokens, int page_shift, int max_pages) {
  PagedArgs a{};
  a.hkv = hkv;
  a.hq = hkv * group;
  a.group = group;
  a.batch = batch;
  a.tokens = tokens;
  a.page_shift = page_shift;
  a.max_pages = max_pages;
  return a;
}

}  // namespace
}  // namespace fa

// The host's plan of a call.  out: classes, workgroups of a class, rows of a unit, split,
// merge kernel, chunk kernel, the chunk kernel's most pieces of a unit (0: any number).
extern "C" void fa_probe_paged_plan(int hkv, int group, int batch, int tokens, int head_dim, int page_shift,
                                    int max_pages, int has_cu, int fp8, int64_t max_query_len,
                                    int64_t workspace_bytes, int* out) {
  static const int32_t index = 0;
  static uint8_t scale = 0;
  fa::PagedArgs a = fa::sizes(hkv, group, batch, tokens, page_shift, max_pages);
  a.cu = has_cu ? &index : nullptr;
  a.ks = a.vs = fp8 ? &scale : nullptr;
  const fa::PagedPlan p = fa::plan_paged(a, head_dim, max_query_len, workspace_bytes);
  const int got[7] = {p.classes, p.wgs, p.rows, p.split, p.combine, p.chunk, p.pieces};
  for (int i = 0; i < 7; ++i) out[i] = got[i];
}

// What the device makes of it (a call that splits): lens, cu and out are device memory,
// plan what the host planned.
extern "C" int fa_probe_paged_pieces(int hkv, int group, int batch, int tokens, int head_dim, int page_shift,
                                     int max_pages, const int32_t* lens, const int32_t* cu, const int* plan,
                                     int* out, int count) {
  fa::PagedArgs a = fa::sizes(hkv, group, batch, tokens, page_shift, max_pages);
  a.lens = lens;
  a.cu = cu;
  a.classes = plan[0];
  a.heads = hkv / plan[0];
  a.wgs = plan[1];
  a.pieces = plan[6];
  a.split = 1;
  const auto kernel = head_dim == 64 ? fa::probe_kernel<64> : fa::probe_kernel<128>;
  hipLaunchKernelGGL(kernel, dim3(1), dim3(64), 0, nullptr, a, plan[2], out, count);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? (int)e : (int)hipDeviceSynchronize();
}
