// Interface between paged_chunk.cu and paged_chunk_tc.cu (caches of 16 bits).
#pragma once
#include "packed.h"

cudaError_t launch_paged_chunk_tc(const ChunkArgs& a, int n_sm, cudaStream_t s);
constexpr int TC_BK = 128;  // keys of a block
cudaError_t launch_chunk_join_tc(const ChunkArgs& a, cudaStream_t s);   // paged_chunk.cu
