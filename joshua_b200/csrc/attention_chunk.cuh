// The two kernels of the attention of chunks.
#pragma once

#include "attention_paged.cuh"

namespace jq {

constexpr uint32_t CHUNK_TILE_ROWS = 128;

// attention_chunk_tiles.cu: the sequences of more than a.span.few rows, heads of 64 and 128.  a.part: [grid][2][CHUNK_TILE_ROWS (hd + 2)].
cudaError_t launch_attention_chunk_tiles(const PagedArgs& a, uint32_t grid, int* error_flag, cudaStream_t s);

}  // namespace jq
