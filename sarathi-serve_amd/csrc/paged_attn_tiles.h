// Host entry of the tile kernel (paged_attention_tiles.hip), heads of up to 128: `rows` 128 or 256.
#pragma once

#include <hip/hip_runtime.h>

#include "paged_attn.h"

namespace sarathi_hip {

int launch_attn_tiles(const PagedAttnArgs& a, int dtype, int rows, int64_t groups, hipStream_t st);

}  // namespace sarathi_hip
