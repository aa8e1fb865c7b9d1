// The attention kernel of hybrid batches: one launch whose work items are the tiles of the chunks and
// those of the decode tokens, in turn.  Chunks are bound by the matrix cores and decodes by memory, so
// some compute units stream keys and values while the others multiply.  Both kinds of item take half
// a compute unit: four waves, one per SIMD, and 66 KiB of LDS (heads above 128: a whole one, 130 KiB).
#pragma once

#include "launch.h"
#include "paged_attn_few.h"
#include "paged_attn_launch.h"
#include "paged_attn_tile.h"

namespace sarathi_hip {

template <int DT, int DP, int RT, bool PAD, bool PAGE16>
__global__ __launch_bounds__(64 * kAttnWaves) __attribute__((amdgpu_waves_per_eu(DP <= 128 ? 2 : 1, DP <= 128 ? 2 : 1)))
void paged_attn_mixed_kernel(PagedAttnArgs a) {
  extern __shared__ u32x4 mixed_lds[];
  const uint32_t h = blockIdx.x % (uint32_t)a.kv_heads;
  const AttnItem it = attn_item(a, blockIdx.x / (uint32_t)a.kv_heads, blockIdx.x == 0);
  if (it.r < 0) return attn_fill(a);
  if (it.tiled) tile_item<DT, DP, PAD, PAGE16>(a, it, h, (lds_char*)mixed_lds);
  else few_item<DT, DP, RT, PAD, PAGE16>(a, it, h, (lds_char*)mixed_lds);
}

template <int DT, int DP, int RT, bool PAD, bool PAGE16>
static int launch_mixed_form(const PagedAttnArgs& a, int64_t groups, hipStream_t st) {
  constexpr int few = few_lds_bytes<DP, RT>(), tile = TileShape<DP>::kBytes;
  constexpr int bytes = few > tile ? few : tile;
  if (!allow_lds<paged_attn_mixed_kernel<DT, DP, RT, PAD, PAGE16>>(bytes)) return SARATHI_ERR_LAUNCH;
  hipLaunchKernelGGL((paged_attn_mixed_kernel<DT, DP, RT, PAD, PAGE16>), dim3((unsigned)groups),
                     dim3(64 * kAttnWaves), bytes, st, a);
  return launch_status();
}
template <int DT, int DP, int RT>
static int launch_mixed_rows(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st) {
  if (a.head_size < DP)
    return page16 ? launch_mixed_form<DT, DP, RT, true, true>(a, groups, st)
                  : launch_mixed_form<DT, DP, RT, true, false>(a, groups, st);
  return page16 ? launch_mixed_form<DT, DP, RT, false, true>(a, groups, st)
                : launch_mixed_form<DT, DP, RT, false, false>(a, groups, st);
}
template <int DT, int DP>
static int launch_mixed(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st) {
  return a.few.rows_log2 == 5 ? launch_mixed_rows<DT, DP, 2>(a, page16, groups, st)
                              : launch_mixed_rows<DT, DP, 1>(a, page16, groups, st);
}

}  // namespace sarathi_hip
