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
#include "fa_paged.h"

namespace fa {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kSelBins = 2048;
// Keys held in LDS (128 KB); those of later positions are made again from the weights.
constexpr int kSelHeld = 32768;
constexpr unsigned kRecentKey = 0xffffffffu;

// An integer that orders as the weights do: NaN below all (1; 0 is no row), -0 as 0.
__device__ __forceinline__ unsigned order_key(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);  // (-0 + 0 = 0)
  if (w != w) return 1;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of the waves' values before this one's, and of all; `scratch` is free again behind it.
struct Before {
  int before, all;
};
__device__ __forceinline__ Before across_waves(int x, int wave, int* scratch) {
  if ((threadIdx.x & 63) == 0) scratch[wave] = x;
  __syncthreads();
  Before r = {0, 0};
#pragma unroll
  for (int i = 0; i < kSelWaves; ++i) {
    const int y = scratch[i];
    r.before += i < wave ? y : 0;
    r.all += y;
  }
  __syncthreads();
  return r;
}

__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) x += __shfl_xor(x, m);
  return x;
}

// A workgroup for each (sequence, KV head); a wave has one stretch of its positions.
__global__ void __launch_bounds__(kSelThreads) fa_paged_select_kernel(const EvictArgs e) {
  __shared__ unsigned keys_lds[kSelHeld];
  __shared__ int bins[kSelBins];
  __shared__ int scratch[kSelWaves];
  __shared__ int found[2];
  const PagedArgs& a = e.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int b = (int)((unsigned)blockIdx.x / (unsigned)a.hkv), h = (int)blockIdx.x - b * a.hkv;
  const int len = max(0, a.lens[b]);
  const int keys = min(len, a.max_pages << a.page_shift);
  const int recent_from = len - min(e.recent, len);
  const float* const w = e.weights + b * e.wb + h * e.wh;
  const int32_t* const entries = a.table + b * a.table_stride;
  const int64_t pair = (int64_t)b * a.hkv + h;
  int32_t* const kept = e.kept + pair * e.slots;
  const int room = e.to_pages << a.page_shift;
  float* const to_w = e.new_weights + pair * room;

  auto make_key = [&](int j) -> unsigned {
    const int page = entries[j >> a.page_shift];
    const float x = w[j];
    if (page < 0 || page >= a.num_pages) return 0;
    return j >= recent_from ? kRecentKey : order_key(x);
  };
  const int part = ((keys + kSelThreads - 1) / kSelThreads) * 64;  // positions of a wave
  const int j0 = min(keys, wave * part), j1 = min(keys, j0 + part);
  int held = 0;
  for (int j = j0 + lane; j < j1; j += 64) {
    const unsigned k = make_key(j);
    if (j < kSelHeld) keys_lds[j] = k;
    held += k != 0;
  }
  auto key_at = [&](int j) -> unsigned { return j < kSelHeld ? keys_lds[j] : make_key(j); };
  const int all = across_waves(wave_sum(held), wave, scratch).all;
  const int target = min(e.keep, all);

  // The smallest key that stays, and how many of those equal to it do.
  unsigned bound = 0;  // (all that are held: those above 0)
  int equal = 0;
  if (target < all && target > 0) {
    int need = target;  // of the keys that agree with `bound` above `shift`
    unsigned mask = 0;
    for (int shift = 21; shift >= 0; shift = shift > 10 ? shift - 11 : shift - 10) {
      const int digits = shift == 0 ? 1 << 10 : kSelBins;
      for (int i = threadIdx.x; i < kSelBins; i += kSelThreads) bins[i] = 0;
      __syncthreads();
      for (int j = j0 + lane; j < j1; j += 64) {
        const unsigned k = key_at(j);
        if ((k & mask) == bound) atomicAdd(&bins[(k >> shift) & (digits - 1)], 1);
      }
      __syncthreads();
      // Thread t: the two bins t from the top.
      const int hi = kSelBins - 1 - 2 * (int)threadIdx.x;
      const int n1 = bins[hi], n0 = bins[hi - 1];
      int upto = n0 + n1;  // inclusive, over the wave's lanes
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        const int y = __shfl_up(upto, m);
        if (lane >= m) upto += y;
      }
      const int above = across_waves(__shfl(upto, 63), wave, scratch).before + upto - n0 - n1;
      if (above < need && above + n1 >= need) {
        found[0] = hi;
        found[1] = above;
      } else if (above + n1 < need && above + n1 + n0 >= need) {
        found[0] = hi - 1;
        found[1] = above + n1;
      }
      __syncthreads();
      bound |= (unsigned)found[0] << shift;
      need -= found[1];
      mask |= (unsigned)(digits - 1) << shift;
      __syncthreads();
      if (shift == 0) break;
    }
    equal = need;
  }

  // The positions that stay, in order.
  int above = 0, same = 0;
  for (int j = j0 + lane; j < j1; j += 64) {
    const unsigned k = key_at(j);
    above += k > bound;
    same += k == bound && k != 0;
  }
  const int above_before = across_waves(wave_sum(above), wave, scratch).before;
  int same_before = across_waves(wave_sum(same), wave, scratch).before;
  int r = above_before + min(same_before, equal);
  if (target > 0) {
    for (int j = j0 + lane; j - lane < j1; j += 64) {
      const unsigned k = j < j1 ? key_at(j) : 0;
      const bool eq = k == bound && k != 0;
      const uint64_t eqs = __builtin_amdgcn_ballot_w64(eq);
      const uint64_t lower = ((uint64_t)1 << lane) - 1;
      const bool stays = k > bound || (eq && same_before + __builtin_popcountll(eqs & lower) < equal);
      const uint64_t all_stay = __builtin_amdgcn_ballot_w64(stays);
      if (stays) {
        const int to = r + __builtin_popcountll(all_stay & lower);
        if (to < target) {  // (always, unless the weights change meanwhile)
          kept[to] = j;
          to_w[to] = w[j];
        }
      }
      r += __builtin_popcountll(all_stay);
      same_before += __builtin_popcountll(eqs);
    }
  }
  for (int j = target + (int)threadIdx.x; j < room; j += kSelThreads) to_w[j] = 0.0f;
  if (h == 0 && threadIdx.x == 0) e.new_lens[b] = target;
}

// Copies the rows that stay, 16 bytes a lane, kMoveRows rows of K and V at once.
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

int64_t evict_workspace_bytes(const EvictArgs& a) {
  return ((int64_t)a.p.batch * a.p.hkv * a.slots * (int64_t)sizeof(int32_t) + 15) & ~(int64_t)15;
}

int launch_evict(const EvictArgs& e, int head_dim, hipStream_t stream) {
  const int64_t pairs = (int64_t)e.p.batch * e.p.hkv;
  hipLaunchKernelGGL(fa_paged_select_kernel, dim3((unsigned)pairs), dim3(kSelThreads), 0, stream, e);
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
