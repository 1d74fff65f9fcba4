// C-ABI of the operators on device buffers (include/llama3_b200.h): checks of their arguments, then their launches.
#include <stdint.h>

#include "../../include/llama3_b200.h"
#include "internal.h"
#include "paged.h"

#define CKD(call) CK(((L3Model*)nullptr), call)
#define REQ(cond, ...) REQUIRE(((L3Model*)nullptr), cond, __VA_ARGS__)

namespace {
struct OnDevice {  // the calling thread's current device, set for as long as this lives
  int before = -1;
  cudaError_t e;
  explicit OnDevice(int device) {
    e = cudaGetDevice(&before);
    if (e == cudaSuccess && before != device) e = cudaSetDevice(device);
    else if (e == cudaSuccess) before = -1;
  }
  ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};
cudaError_t sm_count(int device, int* n) { return cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, device); }
int size_of(int dtype) { return dtype == L3_DTYPE_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == L3_DTYPE_F32 || dtype == L3_DTYPE_BF16 || dtype == L3_DTYPE_F16; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool strides16(int size, std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if (s * size % 16) return false;
  return true;
}
int log2_of(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}
int check_pool(const L3PagePool& p, int size, const char* name) {
  REQ(p.data != nullptr, "%s: no data", name);
  REQ(aligned16(p.data) && strides16(size, {p.page_stride, p.head_stride, p.token_stride}), "%s: addresses must be multiples of 16 bytes", name);
  return L3_OK;
}
int check_pages(int pages, int page_size, int max_pages) {
  REQ(pages >= 1 && max_pages >= 0, "bad number of pages");
  REQ(page_size >= 1 && page_size <= 65536 && (page_size & (page_size - 1)) == 0, "page_size %d is not a power of two up to 65536", page_size);
  REQ((int64_t)max_pages * page_size < ((int64_t)1 << 31) - 65536, "a sequence of %d pages of %d tokens is too long", max_pages, page_size);
  return L3_OK;
}
PagedPool pool_of(const L3PagePool& p, int scale) { return PagedPool{p.data, p.page_stride * scale, p.head_stride * scale, p.token_stride * scale}; }

// The largest piece that divides every address, stride and run of a tensor.
int piece_of(const L3Rows& t) {
  const uint64_t bits = (uint64_t)(uintptr_t)t.base | (uint64_t)t.run | (t.rows > 1 ? (uint64_t)t.row_stride : 0) | (t.outer > 1 ? (uint64_t)t.outer_stride : 0);
  int piece = 16;
  while (bits & (uint64_t)(piece - 1)) piece /= 2;
  return piece;
}
bool empty(const L3Rows& t) { return t.rows == 0 || t.outer == 0 || t.run == 0; }
// The tensors in launches of up to ROWS_MAX, all checks ahead of the first.  `moved`: rows of a tensor that a launch moves.  Tensors of one piece go
// together, so that one of odd bytes does not cut the others into bytes, too - but all of them in pieces of the smallest where those are few, since a
// launch costs as much as a million pieces.  us, one launch : one for each size, a tensor of 16-byte pieces beside bytes: 0.5 MB 3.7 : 5.4, 1 MB 5.6 :
// 5.3, 4 MB 11.7 : 5.9, 17 MB 40 : 7.9; beside 4-byte pieces, both together 0.5 MB 2.9 : 5.4, 8 MB 7.2 : 7.6, 34 MB 18.0 : 15.6; copied pages beside
// bytes 0.4 MB 3.5 : 5.4, 1.6 MB 6.6 : 5.2, 13 MB 40 : 7.4.
template <typename F> int by_pieces(int device, const L3Rows* t, int n, int64_t rows_of_call, int64_t moved, F launch) {
  REQ(t != nullptr && n >= 1, "no tensors");
  int least = 16;
  double bytes = 0;
  for (int i = 0; i < n; ++i) {
    REQ(t[i].outer >= 0 && t[i].run >= 0 && t[i].rows >= 0, "tensor %d: bad sizes", i);
    REQ(rows_of_call < 0 || t[i].rows == rows_of_call, "tensor %d has %lld rows where %lld are meant", i, (long long)t[i].rows, (long long)rows_of_call);
    REQ(t[i].rows == t[0].rows && t[i].rows < ((int64_t)1 << 31), "tensor %d has %lld rows, the first %lld", i, (long long)t[i].rows, (long long)t[0].rows);
    REQ(t[i].base || empty(t[i]), "tensor %d: no data", i);
    if (empty(t[i])) continue;
    // counted in 32 bits, and divided by a multiplication that takes numbers below 2^31
    const int piece = piece_of(t[i]);
    REQ(t[i].outer < ((int64_t)1 << 30) && t[i].run / piece < ((int64_t)1 << 30) && t[i].outer * (t[i].run / piece) < ((int64_t)1 << 30),
        "tensor %d: a row of %lld x %lld bytes is too long", i, (long long)t[i].outer, (long long)t[i].run);
    REQ((double)t[i].outer * (t[i].run / piece) * moved < 0x1p41, "tensor %d: %lld rows of %lld x %lld bytes are too many", i, (long long)moved,
        (long long)t[i].outer, (long long)t[i].run);  // of 2^11 pieces a block
    if (piece < least) least = piece;
    bytes += (double)t[i].outer * t[i].run * moved;
  }
  if (moved == 0) return L3_OK;
  OnDevice on(device);
  CKD(on.e);
  const bool together = bytes <= (double)least * (1 << 20);
  for (int piece = together ? least : 16; piece >= least; piece /= 2) {
    RowsList l;  // the first m entries count
    int m = 0;
    for (int i = 0; i < n; ++i) {
      if (empty(t[i]) || (!together && piece_of(t[i]) != piece)) continue;
      l.t[m++] = RowsDesc{(char*)t[i].base, t[i].row_stride, t[i].outer_stride, (unsigned)t[i].outer, (unsigned)(t[i].run / piece)};
      if (m < ROWS_MAX) continue;
      CKD(launch(l, m, piece));
      m = 0;
    }
    if (m) CKD(launch(l, m, piece));
  }
  return L3_OK;
}
}  // namespace

extern "C" int l3_paged_attention_workspace(int device, int heads, int kv_heads, int head_dim, int64_t* bytes) {
  REQ(bytes && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, "heads %d not a multiple of kv_heads %d", heads, kv_heads);
  REQ(attn_head_dim_supported(head_dim), "head_dim %d unsupported (16,32,48,64,96,128)", head_dim);
  int n_sm = 0;
  CKD(sm_count(device, &n_sm));
  *bytes = (int64_t)paged_attn_workspace(heads, kv_heads, head_dim, n_sm);
  return L3_OK;
}

extern "C" int l3_paged_attention(const L3PagedAttention* a) {
  REQ(a != nullptr, "no arguments");
  REQ(a->batch >= 0 && a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0, "heads %d not a multiple of kv_heads %d", a->heads, a->kv_heads);
  REQ(attn_head_dim_supported(a->head_dim), "head_dim %d unsupported (16,32,48,64,96,128)", a->head_dim);
  REQ(known(a->kv_dtype) && (a->q_dtype == a->kv_dtype || a->q_dtype == L3_DTYPE_F32) && a->out_dtype == a->q_dtype,
      "types: q must have the cache's type or fp32, out q's");
  int rc;
  if ((rc = check_pages(a->pages, a->page_size, a->max_pages)) != L3_OK) return rc;
  const int size = size_of(a->kv_dtype);
  if (a->batch == 0) return L3_OK;
  if ((rc = check_pool(a->k, size, "k")) != L3_OK || (rc = check_pool(a->v, size, "v")) != L3_OK) return rc;
  REQ(a->q && a->out && a->lengths && (a->table || a->max_pages == 0), "q, out, lengths or table missing");
  REQ((int64_t)a->batch * a->kv_heads * ((a->heads / a->kv_heads + 3) / 4) < ((int64_t)1 << 31), "batch %d is too large", a->batch);
  REQ(((uintptr_t)a->out & 7) == 0 && (!a->lse || ((uintptr_t)a->lse & 3) == 0), "out must be aligned to 8 bytes");
  REQ((a->k_new == nullptr) == (a->v_new == nullptr), "k_new and v_new go together");
  if (a->k_new)
    REQ(aligned16(a->k_new) && aligned16(a->v_new) &&
            strides16(size, {a->k_new_batch_stride, a->k_new_head_stride, a->v_new_batch_stride, a->v_new_head_stride}),
        "k_new, v_new: addresses must be multiples of 16 bytes");
  OnDevice on(a->device);
  CKD(on.e);
  int n_sm = 0;
  CKD(sm_count(a->device, &n_sm));
  const size_t need = paged_attn_workspace(a->heads, a->kv_heads, a->head_dim, n_sm);
  REQ(a->workspace && aligned16(a->workspace) && a->workspace_bytes >= (int64_t)need, "the workspace must be %zu bytes, aligned to 16", need);
  PagedAttnArgs p{};
  p.q = a->q; p.q_sb = a->q_batch_stride; p.q_sh = a->q_head_stride; p.q_dtype = a->q_dtype;
  p.k = pool_of(a->k, 1); p.v = pool_of(a->v, 1);
  p.kv_dtype = a->kv_dtype; p.n_pages = a->pages; p.log_page = log2_of(a->page_size);
  p.k_new = a->k_new; p.v_new = a->v_new;
  p.kn_sb = a->k_new_batch_stride; p.kn_sh = a->k_new_head_stride; p.vn_sb = a->v_new_batch_stride; p.vn_sh = a->v_new_head_stride;
  p.table = a->table; p.table_stride = a->table_stride; p.max_pages = a->max_pages; p.lengths = a->lengths;
  p.B = a->batch; p.H = a->heads; p.G = a->kv_heads; p.HD = a->head_dim;
  p.scale = a->scale; p.out = a->out; p.out_dtype = a->out_dtype; p.lse = a->lse; p.ws = a->workspace;
  REQ(paged_attn_fits(p), "a pool of %d pages spans more than 2^32 of its strides' common unit", a->pages);
  CKD(launch_paged_attention(p, n_sm, (cudaStream_t)a->stream));
  return L3_OK;
}

extern "C" int l3_paged_write(const L3PagedWrite* a) {
  REQ(a != nullptr, "no arguments");
  REQ(a->batch >= 0 && a->batch <= 65535 && a->tokens >= 0 && a->kv_heads >= 1 && a->head_dim >= 1, "bad sizes");
  REQ(known(a->dtype), "bad dtype");
  const int size = size_of(a->dtype);
  REQ((int64_t)a->head_dim * size % 16 == 0 && (int64_t)a->kv_heads * a->head_dim < (1 << 28), "head_dim %d: a head's row must be a multiple of 16 bytes", a->head_dim);
  int rc;
  if ((rc = check_pages(a->pages, a->page_size, a->max_pages)) != L3_OK) return rc;
  if (a->batch == 0 || a->tokens == 0) return L3_OK;
  if ((rc = check_pool(a->k_pool, size, "k_pool")) != L3_OK || (rc = check_pool(a->v_pool, size, "v_pool")) != L3_OK) return rc;
  REQ(a->k && a->v && a->start && (a->table || a->max_pages == 0), "k, v, start or table missing");
  REQ(aligned16(a->k) && aligned16(a->v) &&
          strides16(size, {a->k_batch_stride, a->k_token_stride, a->k_head_stride, a->v_batch_stride, a->v_token_stride, a->v_head_stride}),
      "k, v: addresses must be multiples of 16 bytes");
  OnDevice on(a->device);
  CKD(on.e);
  PagedWriteArgs p{};
  p.k = a->k; p.v = a->v;
  p.k_sb = a->k_batch_stride * size; p.k_st = a->k_token_stride * size; p.k_sh = a->k_head_stride * size;
  p.v_sb = a->v_batch_stride * size; p.v_st = a->v_token_stride * size; p.v_sh = a->v_head_stride * size;
  p.kp = pool_of(a->k_pool, size); p.vp = pool_of(a->v_pool, size);
  p.n_pages = a->pages; p.log_page = log2_of(a->page_size);
  p.table = a->table; p.table_stride = a->table_stride; p.max_pages = a->max_pages; p.start = a->start; p.count = a->count;
  p.B = a->batch; p.L = a->tokens; p.G = a->kv_heads; p.pieces = a->head_dim * size / 16;
  CKD(launch_paged_write(p, (cudaStream_t)a->stream));
  return L3_OK;
}

extern "C" int l3_copy_rows(int device, void* stream, const L3Rows* tensors, int n_tensors, const int32_t* src, const int32_t* dst, int n) {
  REQ(n >= 0, "bad number of pairs");
  REQ(n == 0 || (src && dst), "src or dst missing");
  return by_pieces(device, tensors, n_tensors, -1, n, [&](const RowsList& l, int m, int piece) {
    return launch_copy_rows(l, m, src, dst, n, (int)tensors[0].rows, piece, (cudaStream_t)stream);
  });
}

extern "C" int l3_beam_reorder(int device, void* stream, const L3Rows* tensors, int n_tensors, const int32_t* parents, int batch, int beams) {
  REQ(batch >= 0 && batch <= 65535 && beams >= 1 && beams <= ROWS_BEAMS, "batch %d (at most 65535) or beams %d (at most %d)", batch, beams, ROWS_BEAMS);
  REQ(batch == 0 || parents, "parents missing");
  // in place, and all tensors at once: one that is there twice would be read while it is written
  for (int i = 0; tensors && i < n_tensors; ++i)
    for (int j = 0; j < i; ++j)
      REQ(tensors[i].base != tensors[j].base || empty(tensors[i]) || empty(tensors[j]), "tensors %d and %d are the same memory", j, i);
  return by_pieces(device, tensors, n_tensors, (int64_t)batch * beams, (int64_t)batch * beams, [&](const RowsList& l, int m, int piece) {
    return launch_reorder_rows(l, m, parents, batch, beams, piece, (cudaStream_t)stream);
  });
}

static int check_select(int batch, int beams, int vocab, int best) {
  REQ(batch >= 0 && beams >= 1 && beams <= BEAM_MAX_K && best >= 1 && best <= BEAM_MAX_N, "beams %d (1 - %d) or best %d (1 - %d)", beams, BEAM_MAX_K, best,
      BEAM_MAX_N);
  REQ(vocab >= 1 && vocab < (1 << 24) && (int64_t)batch * beams <= 65535, "vocab %d or batch %d is too large", vocab, batch);
  REQ((int64_t)beams * vocab < ((int64_t)1 << 31), "%d beams of %d tokens are too many", beams, vocab);
  return L3_OK;
}
extern "C" int l3_beam_select_workspace(int device, int batch, int beams, int vocab, int best, int64_t* bytes) {
  REQ(bytes != nullptr, "no place for the answer");
  int rc = check_select(batch, beams, vocab, best), n_sm = 0;
  if (rc != L3_OK) return rc;
  CKD(sm_count(device, &n_sm));
  *bytes = batch ? (int64_t)beam_select_workspace(batch, beams, vocab, best, n_sm) : 0;
  return L3_OK;
}
extern "C" int l3_beam_select(const L3BeamSelect* a) {
  REQ(a != nullptr, "no arguments");
  int rc = check_select(a->batch, a->beams, a->vocab, a->best);
  if (rc != L3_OK) return rc;
  REQ(known(a->dtype), "bad dtype");
  REQ(a->eos >= -1 && a->eos < a->vocab && (!a->done || a->eos >= 0), "eos %d: finished beams need an end token below vocab", a->eos);
  if (a->batch == 0) return L3_OK;
  REQ(a->logits && a->scores && a->out_scores && a->out_tokens && a->out_parents && a->out_done, "a buffer is missing");
  OnDevice on(a->device);
  CKD(on.e);
  int n_sm = 0;
  CKD(sm_count(a->device, &n_sm));
  const size_t need = beam_select_workspace(a->batch, a->beams, a->vocab, a->best, n_sm);
  REQ(a->workspace && aligned16(a->workspace) && a->workspace_bytes >= (int64_t)need, "the workspace must be %zu bytes, aligned to 16", need);
  BeamSelectArgs s{};
  s.logits = a->logits; s.sb = a->batch_stride; s.sk = a->beam_stride; s.dtype = a->dtype;
  s.scores = a->scores; s.done = a->done; s.eos = a->eos; s.B = a->batch; s.K = a->beams; s.V = a->vocab; s.n = a->best;
  s.out_scores = a->out_scores; s.out_tokens = a->out_tokens; s.out_parents = a->out_parents; s.out_done = a->out_done; s.ws = a->workspace;
  CKD(launch_beam_select(s, n_sm, (cudaStream_t)a->stream));
  return L3_OK;
}
