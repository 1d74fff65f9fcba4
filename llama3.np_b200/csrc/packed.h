// A packed step over a cache in pages: interface of packed_step.cu (bookkeeping, rotary positions), paged_chunk.cu (attention) and
// logprobs.cu (log probabilities of tokens).
#pragma once
#include "paged.h"

struct PagedExtendArgs {
  int* table;                        // [B, max_pages], row stride table_stride
  long long table_stride;
  int max_pages, log_page, B, T, n_free;
  const int *lengths, *counts, *free_pages;
  int *out_lengths, *out_starts, *out_positions;
  long long* out_slots;
  int* out_used;
};
cudaError_t launch_paged_extend(const PagedExtendArgs& a, int n_sm, cudaStream_t s);

struct RotaryArgs {
  const int* positions;              // [B * L]
  const double* freqs;               // [dims / 2], radians a position
  float amplitude;                   // of cosines and sines
  bool inverse;
  const void* x;                     // [B, L, H, D], strides in elements
  long long x_sb, x_st, x_sh;
  void* out;
  long long o_sb, o_st, o_sh;
  const void *k, *v;                 // [L, G, D]
  long long k_st, k_sh, v_st, v_sh;
  const long long* slots;            // [L]
  PagedPool kp, vp;                  // strides in elements
  int n_pages, log_page;
  int B, L, H, G, D, dims, layout, dtype;
};
cudaError_t launch_rotary(const RotaryArgs& a, int n_sm, cudaStream_t s);

struct ChunkArgs {
  const void* q;                     // [T, H, HD], strides in elements
  long long q_st, q_sh;
  PagedPool k, v;                    // strides in elements
  int n_pages, log_page;
  const int* table;                  // [B, max_pages], row stride table_stride
  long long table_stride;
  int max_pages;
  const int *lengths, *starts;       // [B], [B + 1]
  int B, T, H, G, R, HD, dtype;      // R: query heads of a kv head
  float scale;
  void* out;                         // [T, H, HD]
  float* lse;                        // [T, H] or null
  int clear_rest;                    // rows of no request: 0 as they are, 1: 0 (lse -infinity), 2: lse alone
  void* ws;                          // paged_chunk_workspace bytes, 16-byte aligned
  // set by the launcher
  int n_cta, tile_rows;              // CTAs, flat rows of an item
  float* part_o;                     // [n_cta][2][rows of a tile][HD]
  float2* part_ml;                   // [n_cta][2][rows of a tile]
  void* left;                        // [n_cta] chunk::Left
};
size_t paged_chunk_workspace(int H, int G, int HD, int dtype, int n_sm);
cudaError_t launch_paged_chunk(ChunkArgs a, int n_sm, cudaStream_t s);

struct LogprobsArgs {
  const void* logits;                // [R, V], row stride in elements
  long long stride;
  int dtype, R, V, n;                // n: how many of the most likely tokens
  const int* tokens;
  float *out_logprobs, *out_entropy, *out_top;
  int* out_top_tokens;
};
constexpr int LOGPROBS_MAX_TOP = 64;
cudaError_t launch_token_logprobs(const LogprobsArgs& a, int n_sm, cudaStream_t s);
