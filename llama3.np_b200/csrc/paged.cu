// Attention of one new token per sequence over a cache in pages (paged_attn.cuh).
#include "paged_attn.cuh"

size_t paged_attn_workspace(int H, int G, int HD, int n_sm) {
  const size_t W = (size_t)n_sm * MOST_WARPS;
  return W * sizeof(int4) + 2 * W * (H / G < HEADS ? H / G : HEADS) * ((size_t)HD + 2) * sizeof(float);
}
bool paged_attn_fits(PagedAttnArgs a) { return set_units(a); }
cudaError_t launch_paged_attention(const PagedAttnArgs& a, int n_sm, cudaStream_t s, int* count) {
  int none, &launches = count ? *count : none;
  return a.starts ? launch_paged_attention_step(a, n_sm, s, launches) : launch_attention<false>(a, n_sm, s, launches);
}
