// Host entries of the matrix-core attention kernels: `groups` workgroups, key head by key head of
// the work items.  Heads of multiples of 8 elements, 16-byte aligned rows.
#pragma once

#include <hip/hip_runtime.h>

#include "paged_attn.h"

namespace sarathi_hip {

// tiles of few rows only, heads of up to 256
int launch_attn_few(const PagedAttnArgs& a, int dtype, bool page16, int64_t groups, hipStream_t st);
// tiles of chunks and of few rows in one launch, heads of up to 64, 128, 256
int launch_attn_mixed_bf16_64(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st);
int launch_attn_mixed_bf16_128(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st);
int launch_attn_mixed_bf16_256(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st);
int launch_attn_mixed_f16_64(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st);
int launch_attn_mixed_f16_128(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st);
int launch_attn_mixed_f16_256(const PagedAttnArgs& a, bool page16, int64_t groups, hipStream_t st);

}  // namespace sarathi_hip
