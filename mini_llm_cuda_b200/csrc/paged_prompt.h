// Host entry of the paged attention for sequences that bring many rows (paged_prompt.cu): bf16 rows, bf16 or 4-bit pages.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace mlb {
struct AttnPagedParams;
// Tensor maps of the pools (bf16 pages; else left empty). Made before a call's first launch, so that a call that fails has written nothing.
struct alignas(64) PromptMaps {
    CUtensorMap k, v;
};
cudaError_t attn_prompt_maps(const AttnPagedParams& p, int dtype, int head_dim, PromptMaps* maps);
cudaError_t attn_prompt_launch(const AttnPagedParams& p, int dtype, int head_dim, const PromptMaps& maps, cudaStream_t st);
}  // namespace mlb
