// Rows of a packed step as single tokens (paged_attn.cuh), apart from paged.cu so that the two compile side by side.
#include "paged_attn.cuh"

cudaError_t launch_paged_attention_step(const PagedAttnArgs& a, int n_sm, cudaStream_t s, int& launches) { return launch_attention<true>(a, n_sm, s, launches); }
