// Hybrid-batch attention kernels (paged_attn_mixed.h): bfloat16, heads of up to 256.
#include "paged_attn_mixed.h"

namespace sarathi_hip {

int launch_attn_mixed_bf16_256(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st) {
  return launch_mixed<kBF16, 256>(a, page16, groups, st);
}

}  // namespace sarathi_hip
