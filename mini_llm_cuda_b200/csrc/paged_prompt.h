// Host entry of the paged attention for sequences that bring many rows (paged_prompt.cu): bf16 rows, bf16 or 4-bit pages.
#pragma once
#include <cuda_runtime.h>

namespace mlb {
struct AttnPagedParams;
cudaError_t attn_prompt_launch(const AttnPagedParams& p, int dtype, int head_dim, cudaStream_t st);
}  // namespace mlb
