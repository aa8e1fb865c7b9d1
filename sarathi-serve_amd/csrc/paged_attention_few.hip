// The attention kernel of batches without chunks: every work item is a tile of few rows
// (paged_attn_few.h).  Four waves and 66 KiB of LDS per workgroup, so that two share a compute unit
// and one's start and end run beside the other's stream (heads above 128: 130 KiB, one to a unit).
#include "launch.h"
#include "paged_attn_few.h"
#include "paged_attn_launch.h"

namespace sarathi_hip {

template <int DT, int DP, int RT, bool PAD, bool PAGE16>
__global__ __launch_bounds__(64 * kAttnWaves) void paged_attn_few_kernel(PagedAttnArgs a) {
  extern __shared__ u32x4 few_lds[];
  const uint32_t h = blockIdx.x % (uint32_t)a.kv_heads;
  const AttnItem it = attn_item(a, blockIdx.x / (uint32_t)a.kv_heads, blockIdx.x == 0);
  if (it.r < 0) return attn_fill(a);
  few_item<DT, DP, RT, PAD, PAGE16>(a, it, h, (lds_char*)few_lds);
}

template <int DT, int DP, int RT, bool PAD, bool PAGE16>
static int launch_few(const PagedAttnArgs& a, int64_t groups, hipStream_t st) {
  constexpr int bytes = few_lds_bytes<DP, RT>();
  if (!allow_lds<paged_attn_few_kernel<DT, DP, RT, PAD, PAGE16>>(bytes)) return SARATHI_ERR_LAUNCH;
  hipLaunchKernelGGL((paged_attn_few_kernel<DT, DP, RT, PAD, PAGE16>), dim3((unsigned)groups),
                     dim3(64 * kAttnWaves), bytes, st, a);
  return launch_status();
}
// the exact head size and pages of a multiple of 16 keys have kernels of their own
template <int DT, int DP, int RT>
static int launch_few_form(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st) {
  if (a.head_size < DP)
    return page16 ? launch_few<DT, DP, RT, true, true>(a, groups, st)
                  : launch_few<DT, DP, RT, true, false>(a, groups, st);
  return page16 ? launch_few<DT, DP, RT, false, true>(a, groups, st)
                : launch_few<DT, DP, RT, false, false>(a, groups, st);
}
template <int DT, int DP>
static int launch_few_rows(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st) {
  if (a.few.rows_log2 == 4) return launch_few_form<DT, DP, 1>(a, page16, groups, st);
  if constexpr (DP <= 128)
    if (a.few.rows_log2 == 6) return launch_few_form<DT, DP, 4>(a, page16, groups, st);
  return launch_few_form<DT, DP, 2>(a, page16, groups, st);
}
template <int DT>
static int launch_few_heads(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st) {
  if (a.head_size <= 64) return launch_few_rows<DT, 64>(a, page16, groups, st);
  if (a.head_size <= 128) return launch_few_rows<DT, 128>(a, page16, groups, st);
  return launch_few_rows<DT, 256>(a, page16, groups, st);
}

int launch_attn_few(const PagedAttnArgs& a, int dtype, bool page16, int64_t groups, hipStream_t st) {
  return dtype == kBF16 ? launch_few_heads<kBF16>(a, page16, groups, st)
                        : launch_few_heads<kF16>(a, page16, groups, st);
}

}  // namespace sarathi_hip
