// A key / value cache in pages: interface of paged.cu (attention of single tokens) and paged_rows.cu (writing, copying, reordering).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

// How a pool is addressed: element (page, kv head, token of the page, dimension) is at page * sp + head * sh + token * st + dimension.
struct PagedPool {
  void* p;
  long long sp, sh, st;
};
struct PagedAttnArgs {
  const void* q;                     // [B, H, HD], strides q_sb, q_sh in elements
  long long q_sb, q_sh;
  int q_dtype;                       // L3_DTYPE_*: the cache's own, or fp32
  PagedPool k, v;
  int kv_dtype, n_pages, log_page;   // a page holds 1 << log_page tokens
  const void *k_new, *v_new;         // null, or [B, G, HD] of the cache's type: the token at length - 1, written to its page
  long long kn_sb, kn_sh, vn_sb, vn_sh;
  const int* table;                  // [B, max_pages], row stride table_stride
  long long table_stride;
  int max_pages;
  const int* lengths;                // [B], or null: *pos_ptr + 1 tokens for every sequence
  const int* pos_ptr;
  int B, H, G, HD;
  float scale;
  void* out;                         // [B, H, HD]
  int out_dtype;
  float* out_lo;                     // with fp32 `out`: that gets the TF32 high part, out_lo the rest (may be null)
  float* lse;                        // [B, H] or null
  void* ws;                          // paged_attn_workspace bytes, 16-byte aligned
  // set by the launcher
  int unit;                          // bytes; the pools' strides below are in units of it
  uint32_t ku_page, ku_head, ku_token, vu_page, vu_head, vu_token;
  bool q_vec;                        // every query row begins on 16 bytes
  int nrep, heads_blk, blocks;       // query heads of a kv head, of a work item, items per kv head
  float *part_o, *part_ml;
  int4* info;
  int n_info;
  bool by_item;
};
size_t paged_attn_workspace(int H, int G, int HD, int n_sm);
bool paged_attn_fits(PagedAttnArgs a);  // the pools' offsets fit 32 bits of the largest unit that divides their strides
cudaError_t launch_paged_attention(PagedAttnArgs a, int n_sm, cudaStream_t s, int* launches = nullptr);  // launches: how many it made, 1 or 2

struct PagedWriteArgs {
  const void *k, *v;                 // [B, L, G, HD]; strides in bytes
  long long k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  PagedPool kp, vp;                  // strides in bytes
  int n_pages, log_page;
  const int* table;
  long long table_stride;
  int max_pages;
  const int *start, *count;          // [B]; count null: L tokens of every sequence
  int B, L, G, pieces;               // 16-byte pieces of a head's row
};
cudaError_t launch_paged_write(const PagedWriteArgs& a, cudaStream_t s);

// One tensor of rows (pages of a pool, beams of a state): row r is `outer` runs of `run` bytes, `outer_stride` apart.
struct RowsDesc {
  char* base;
  long long row_stride, outer_stride;
  unsigned outer, run;               // run: in pieces of the launch's size
};
constexpr int ROWS_MAX = 64;         // tensors of one launch
constexpr int ROWS_BEAMS = 256;      // most beams that reordering takes
struct RowsList { RowsDesc t[ROWS_MAX]; };
// row dst[i] <- row src[i] of every tensor, for entries in [0, rows); piece: bytes that every address and run is a multiple of (1 - 16)
cudaError_t launch_copy_rows(const RowsList& l, int n_tensors, const int* src, const int* dst, int n, int rows, int piece, cudaStream_t s);
// row b K + j <- row b K + parents[b][j] of every tensor, in place
cudaError_t launch_reorder_rows(const RowsList& l, int n_tensors, const int* parents, int B, int K, int piece, cudaStream_t s);

struct BeamSelectArgs {
  const void* logits;                // [B, K, V], strides in elements
  long long sb, sk;
  int dtype;                         // L3_DTYPE_*
  const float* scores;               // [B, K]
  const unsigned char* done;         // [B, K] or null
  int eos, B, K, V, n;
  float* out_scores;                 // [B, n]
  int *out_tokens, *out_parents;
  unsigned char* out_done;
  void* ws;                          // beam_select_workspace bytes, 16-byte aligned
};
constexpr int BEAM_MAX_K = 256, BEAM_MAX_N = 64;
size_t beam_select_workspace(int B, int K, int V, int n, int n_sm);
cudaError_t launch_beam_select(const BeamSelectArgs& a, int n_sm, cudaStream_t s);

// Beam search over a model's own caches (l3_generate_beam): rows of B prompts' K beams, tokens in pages of one.  Slot r's row of a cache holds
// the tokens that row r wrote; table [rows, M] names, for every row and position, the token it descends from (slot * stride + position).
struct BeamState {
  int *table, *tokens, *parents, *hist_tokens, *hist_parents;  // [rows, M], [rows], [rows], [M, rows] twice
  float *scores, *new_scores;                                   // [rows]
  unsigned char *done, *new_done;
  int* scal;                                                    // the handle's step scalars: [0] position [1] step [2] position of step 0
  int rows, K, M, stride;                                       // stride: tokens of a slot in a pool, kv heads * M
};
cudaError_t launch_beam_prompts(const BeamState& b, int L, cudaStream_t s);  // every beam descends from its prompt; scores and flags start at 0
cudaError_t launch_beam_begin(const BeamState& b, cudaStream_t s);           // the next step's position, its token the row's own
cudaError_t launch_beam_commit(const BeamState& b, cudaStream_t s);          // the selection becomes the state, and goes into the history
