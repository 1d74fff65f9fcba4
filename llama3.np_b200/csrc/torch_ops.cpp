// The operators on device buffers as Python calls on torch tensors: checks of shapes, types, strides and devices, outputs and workspaces
// from torch's allocator, and one call of the C-ABI (include/llama3_b200.h), whose entries _cabi.py hands over (`bind`).  In Python the checks
// and the filling of the C structs took 10 - 20 us a call, several times as long as a small call's kernels.
#define PY_SSIZE_T_CLEAN
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/llama3_b200.h"

namespace {
struct Entries {
  decltype(&l3_paged_attention_workspace) attention_workspace;
  decltype(&l3_paged_attention) attention;
  decltype(&l3_paged_write) write;
  decltype(&l3_copy_rows) copy;
  decltype(&l3_beam_reorder) reorder;
  decltype(&l3_beam_select_workspace) select_workspace;
  decltype(&l3_beam_select) select;
  decltype(&l3_last_error) last_error;
  decltype(&l3_paged_extend) extend;
  decltype(&l3_rotary) rotary;
  decltype(&l3_paged_chunk_workspace) chunk_workspace;
  decltype(&l3_paged_chunk_attention) chunk;
  decltype(&l3_token_logprobs) logprobs;
} entry{};

using at::Tensor;
#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

void done(int rc) {
  if (rc == L3_OK) return;
  const std::string text = entry.last_error(nullptr);
  if (rc == L3_EINVAL) NEED(false, text);
  TORCH_CHECK(false, "llama3_b200 error ", rc, ": ", text);
}
const Tensor& tensor(PyObject* x, const char* name) {
  NEED(THPVariable_Check(x), name, " must be a tensor");
  const Tensor& t = THPVariable_Unpack(x);
  NEED(t.layout() == at::kStrided, name, " must be a strided tensor");
  NEED(!t.is_neg(), name, " is a negated view: resolve_neg() it first");
  NEED(!t.requires_grad() || !c10::GradMode::is_enabled(), name, " requires a gradient, and this has no backward pass: call it under torch.no_grad()");
  NEED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(/*level=*/0).defined(), name,
       " has a forward-mode gradient, which this would drop: unpack the dual tensor first");
  return t;
}
// what a call writes is new to autograd: a backward pass that saved the old values raises
void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
const Tensor& tensor(PyObject* x, const char* name, int64_t dims) {
  const Tensor& t = tensor(x, name);
  NEED(t.dim() == dims, name, " must have ", dims, " dimensions, got ", t.sizes());
  return t;
}
int kind(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return L3_DTYPE_F32;
    case at::kBFloat16: return L3_DTYPE_BF16;
    case at::kHalf: return L3_DTYPE_F16;
    default: NEED(false, name, ": type ", t.scalar_type(), " is not one of float32, bfloat16, float16"); return 0;
  }
}
void typed(const Tensor& t, const char* name, at::ScalarType type) { NEED(t.scalar_type() == type, name, ": type ", t.scalar_type(), " where ", type, " is meant"); }
int64_t step_of(const Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }  // of one entry it may be anything
const int32_t* ints(const Tensor& t, const char* name, int64_t n) {
  typed(t, name, at::kInt);
  NEED(t.dim() == 1 && t.size(0) == n, name, " must be [", n, "], got ", t.sizes());
  NEED(t.is_contiguous(), name, " must be contiguous");
  return t.const_data_ptr<int32_t>();
}
void last_is_dense(const Tensor& t, const char* name) { NEED(t.size(-1) <= 1 || t.stride(-1) == 1, name, ": the last dimension must be contiguous"); }
void fits16(const Tensor& t, const char* name) {
  bool ok = (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && (t.size(d) <= 1 || t.stride(d) * t.element_size() % 16 == 0);
  NEED(ok, name, ": addresses must be multiples of 16 bytes");
}
struct OneDevice {  // every tensor of a call is on the same one
  int index = -1;
  void add(const Tensor& t, const char* name) {
    NEED(t.is_cuda(), name, " must be on a CUDA device");
    const int i = t.get_device();
    NEED(index < 0 || i == index, name, " is on device ", i, ", the others on ", index);
    index = i;
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(index).stream(); }
};
const Tensor& table_of(PyObject* x, int64_t batch) {
  const Tensor& t = tensor(x, "page_table", 2);
  typed(t, "page_table", at::kInt);
  NEED(t.size(0) == batch, "page_table has ", t.size(0), " rows for ", batch, " sequences");
  NEED(t.size(1) <= 1 || t.stride(1) == 1, "page_table: a row must be contiguous");
  return t;
}
void own_places(const Tensor& t, const char* name) {
  for (int64_t d = 0; d < 3; ++d) NEED(t.size(d) <= 1 || t.stride(d) != 0, name, " is expanded, and would be written");
}
int pools_of(const Tensor& k, const Tensor& v) {
  const int type = kind(k, "k_pages");
  typed(v, "v_pages", k.scalar_type());
  NEED(k.sizes() == v.sizes(), "k_pages and v_pages differ: ", k.sizes(), " and ", v.sizes());
  const int64_t page = k.size(2);
  NEED(k.size(0) >= 1 && page >= 1 && page <= 65536 && (page & (page - 1)) == 0, "page size ", page, " is not a power of two up to 65536");
  last_is_dense(k, "k_pages");
  last_is_dense(v, "v_pages");
  fits16(k, "k_pages");
  fits16(v, "v_pages");
  return type;
}
L3PagePool pool(const Tensor& t) { return L3PagePool{t.data_ptr(), step_of(t, 0), step_of(t, 1), step_of(t, 2)}; }
int size32(int64_t n, const char* what) {
  NEED(n < ((int64_t)1 << 31), what, " ", n, " is too large");
  return (int)n;
}
void args(Py_ssize_t n, Py_ssize_t want) { NEED(n == want, "takes ", want, " arguments, got ", n); }
bool given(PyObject* x) { return x != Py_None; }
int64_t integer(PyObject* x) {
  const long long v = PyLong_AsLongLong(x);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double real(PyObject* x) {
  const double v = PyFloat_AsDouble(x);
  if (v == -1. && PyErr_Occurred()) throw python_error();
  return v;
}

// paged_attention(q, k_pages, v_pages, page_table, lengths, k_new, v_new, scale, return_lse, out)
PyObject* paged_attention(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 10);
  const Tensor &q = tensor(x[0], "q", 3), &k = tensor(x[1], "k_pages", 4), &v = tensor(x[2], "v_pages", 4);
  L3PagedAttention a{};
  a.kv_dtype = pools_of(k, v);
  a.q_dtype = a.out_dtype = kind(q, "q");
  const int64_t batch = q.size(0), heads = q.size(1), dim = q.size(2), G = k.size(1);
  NEED(a.q_dtype == a.kv_dtype || a.q_dtype == L3_DTYPE_F32, "q must have the cache's type or fp32, got ", q.scalar_type(), " over ", k.scalar_type());
  NEED(k.size(3) == dim && (dim == 16 || dim == 32 || dim == 48 || dim == 64 || dim == 96 || dim == 128), "head size ", dim, " (cache: ", k.size(3),
       ") is not one of 16, 32, 48, 64, 96, 128");
  NEED(G >= 1 && heads >= 1 && heads % G == 0, heads, " heads over ", G, " kv heads");
  last_is_dense(q, "q");
  const Tensor& table = table_of(x[3], batch);
  const Tensor& lengths = tensor(x[4], "lengths", 1);
  a.lengths = ints(lengths, "lengths", batch);
  NEED(given(x[5]) == given(x[6]), "k_new and v_new go together");
  OneDevice on;
  if (given(x[5])) {
    own_places(k, "k_pages");
    own_places(v, "v_pages");
    const Tensor *fresh[2] = {&tensor(x[5], "k_new", 3), &tensor(x[6], "v_new", 3)};
    for (int i = 0; i < 2; ++i) {
      const char* name = i ? "v_new" : "k_new";
      const Tensor& t = *fresh[i];
      typed(t, name, k.scalar_type());
      NEED(t.size(0) == batch && t.size(1) == G && t.size(2) == dim, name, " must be [", batch, ", ", G, ", ", dim, "], got ", t.sizes());
      last_is_dense(t, name);
      fits16(t, name);
    }
    a.k_new = fresh[0]->const_data_ptr(); a.v_new = fresh[1]->const_data_ptr();
    a.k_new_batch_stride = step_of(*fresh[0], 0); a.k_new_head_stride = step_of(*fresh[0], 1);
    a.v_new_batch_stride = step_of(*fresh[1], 0); a.v_new_head_stride = step_of(*fresh[1], 1);
  }
  if (given(x[9])) {
    const Tensor& out = tensor(x[9], "out", 3);
    typed(out, "out", q.scalar_type());
    NEED(out.sizes() == q.sizes() && out.is_contiguous() && (reinterpret_cast<uintptr_t>(out.const_data_ptr()) & 15) == 0,
         "out must be contiguous, of q's shape");
  }
  on.add(q, "q"); on.add(k, "k_pages"); on.add(v, "v_pages"); on.add(table, "page_table"); on.add(lengths, "lengths");
  if (given(x[5])) {
    on.add(THPVariable_Unpack(x[5]), "k_new");
    on.add(THPVariable_Unpack(x[6]), "v_new");
  }
  if (given(x[9])) on.add(THPVariable_Unpack(x[9]), "out");
  const bool want_lse = x[8] == Py_True;
  const Tensor out = given(x[9]) ? THPVariable_Unpack(x[9]) : at::empty({batch, heads, dim}, q.options());
  Tensor lse, room;
  if (want_lse) lse = at::empty({batch, heads}, q.options().dtype(at::kFloat));
  if (batch) {
    a.device = on.index; a.batch = size32(batch, "batch"); a.heads = size32(heads, "heads"); a.kv_heads = (int)G; a.head_dim = (int)dim;
    a.pages = size32(k.size(0), "pages"); a.page_size = (int)k.size(2); a.max_pages = size32(table.size(1), "page_table");
    a.scale = given(x[7]) ? (float)real(x[7]) : (float)(1.0 / std::sqrt((double)dim));
    a.stream = on.stream();
    a.q = q.const_data_ptr(); a.q_batch_stride = step_of(q, 0); a.q_head_stride = step_of(q, 1);
    a.k = pool(k); a.v = pool(v);
    a.table = table.const_data_ptr<int32_t>(); a.table_stride = step_of(table, 0);
    a.out = out.data_ptr();
    a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
    done(entry.attention_workspace(on.index, a.heads, a.kv_heads, a.head_dim, &a.workspace_bytes));
    room = at::empty({a.workspace_bytes}, q.options().dtype(at::kByte));  // of this call: a captured graph has one of its own
    a.workspace = room.data_ptr();
    done(entry.attention(&a));
    if (given(x[5])) {
      changed(k);
      changed(v);
    }
  }
  if (given(x[9])) changed(out);
  if (!want_lse) return THPVariable_Wrap(out);
  PyObject* both = PyTuple_New(2);
  if (!both) throw python_error();
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(out));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(lse));
  return both;
  END_HANDLE_TH_ERRORS
}

// paged_write(k, v, k_pages, v_pages, page_table, start, count)
PyObject* paged_write(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 7);
  const Tensor &k = tensor(x[0], "k", 4), &v = tensor(x[1], "v", 4), &kp = tensor(x[2], "k_pages", 4), &vp = tensor(x[3], "v_pages", 4);
  L3PagedWrite a{};
  a.dtype = pools_of(kp, vp);
  const int64_t batch = k.size(0), tokens = k.size(1), G = kp.size(1), dim = kp.size(3);
  for (const Tensor* t : {&k, &v}) {
    const char* name = t == &k ? "k" : "v";
    typed(*t, name, kp.scalar_type());
    NEED(t->sizes() == k.sizes() && t->size(2) == G && t->size(3) == dim, name, " must be [batch, tokens, ", G, ", ", dim, "], got ", t->sizes());
    last_is_dense(*t, name);
    fits16(*t, name);
  }
  NEED(dim * k.element_size() % 16 == 0, "head size ", dim, ": a head's row must be a multiple of 16 bytes");
  NEED(batch <= 65535, "at most 65535 sequences a call");
  own_places(kp, "k_pages");
  own_places(vp, "v_pages");
  const Tensor& table = table_of(x[4], batch);
  const Tensor& start = tensor(x[5], "start", 1);
  a.start = ints(start, "start", batch);
  if (given(x[6])) a.count = ints(tensor(x[6], "count", 1), "count", batch);
  OneDevice on;
  on.add(k, "k"); on.add(v, "v"); on.add(kp, "k_pages"); on.add(vp, "v_pages"); on.add(table, "page_table"); on.add(start, "start");
  if (given(x[6])) on.add(THPVariable_Unpack(x[6]), "count");
  if (batch && tokens) {
    a.device = on.index; a.batch = (int)batch; a.tokens = size32(tokens, "tokens"); a.kv_heads = size32(G, "kv heads"); a.head_dim = size32(dim, "head size");
    a.pages = size32(kp.size(0), "pages"); a.page_size = (int)kp.size(2); a.max_pages = size32(table.size(1), "page_table");
    a.stream = on.stream();
    a.k = k.const_data_ptr(); a.v = v.const_data_ptr();
    a.k_batch_stride = step_of(k, 0); a.k_token_stride = step_of(k, 1); a.k_head_stride = step_of(k, 2);
    a.v_batch_stride = step_of(v, 0); a.v_token_stride = step_of(v, 1); a.v_head_stride = step_of(v, 2);
    a.k_pool = pool(kp); a.v_pool = pool(vp);
    a.table = table.const_data_ptr<int32_t>(); a.table_stride = step_of(table, 0);
    done(entry.write(&a));
    changed(kp);
    changed(vp);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// A tensor's rows (first dimension) as runs of bytes: one, or equal ones at equal distances.
L3Rows rows_of(const Tensor& t, const char* what, int64_t i) {
  NEED(t.dim() >= 1, what, " ", i, " has no rows");
  const int64_t size = t.element_size();
  int64_t run = 1, outer = 1, outer_stride = 0, d = t.dim() - 1;
  for (; d > 0 && (t.size(d) <= 1 || t.stride(d) == run); --d) run *= t.size(d);
  if (run && d > 0) {
    bool none = false;
    for (int64_t e = d; e > 0; --e) none = none || t.size(e) == 0;
    if (none) run = d = 0;
  } else d = 0;
  if (d > 0) {
    outer = t.size(d);
    outer_stride = t.stride(d);
    for (--d; d > 0 && (t.size(d) == 1 || t.stride(d) == outer * outer_stride); --d) outer *= t.size(d);
  }
  NEED(d == 0, what, " ", i, ": a row of shape ", t.sizes().slice(1), " and strides ", t.strides().slice(1),
       " is not a run, or equal runs at equal distances");
  const int64_t row = t.stride(0), span = run && outer ? (outer - 1) * outer_stride + run : 0;
  NEED(outer <= 1 || outer_stride >= run, what, " ", i, " overlaps itself");
  // rows apart, or between one another's runs, as in a cache kept [heads, sequences, ...]
  NEED(t.size(0) <= 1 || row >= span || (run <= row && row * t.size(0) <= outer_stride), what, " ", i, ": rows overlap");
  return L3Rows{t.data_ptr(), t.size(0), row * size, outer, outer_stride * size, run * size};
}
struct Listed {  // a tensor, or any iterable of them, which is walked once: it may be a generator that alone holds them
  std::vector<Tensor> tensors;
  std::vector<L3Rows> rows;
  Listed(PyObject* x, const char* what) {
    if (THPVariable_Check(x)) {
      add(x, what);
      return;
    }
    PyObject* seq = PySequence_Fast(x, "a tensor or a list of tensors is needed");
    if (!seq) throw python_error();
    struct Drop {
      PyObject* p;
      ~Drop() { Py_DECREF(p); }
    } drop{seq};
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    NEED(n >= 1, "no ", what);
    tensors.reserve(n);
    rows.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) add(PySequence_Fast_GET_ITEM(seq, i), what);
  }
  void add(PyObject* x, const char* what) {
    tensors.push_back(tensor(x, what));
    rows.push_back(rows_of(tensors.back(), what, (int64_t)rows.size()));
  }
};

// copy_pages(pools, src, dst)
PyObject* copy_pages(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 3);
  OneDevice on;
  const Listed pools(x[0], "pools");
  for (const L3Rows& r : pools.rows) NEED(r.rows == pools.rows[0].rows, "pools have ", pools.rows[0].rows, " and ", r.rows, " pages");
  const Tensor &src = tensor(x[1], "src", 1), &dst = tensor(x[2], "dst", 1);
  const int pairs = size32(src.size(0), "src");
  const int32_t *from = ints(src, "src", pairs), *to = ints(dst, "dst", pairs);
  for (const Tensor& t : pools.tensors) on.add(t, "pools");
  on.add(src, "src"); on.add(dst, "dst");
  if (pairs) {
    done(entry.copy(on.index, on.stream(), pools.rows.data(), size32(pools.rows.size(), "pools"), from, to, pairs));
    for (const Tensor& t : pools.tensors) changed(t);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// beam_reorder(states, parents)
PyObject* beam_reorder(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 2);
  const Tensor& parents = tensor(x[1], "parents", 2);
  typed(parents, "parents", at::kInt);
  NEED(parents.is_contiguous(), "parents must be contiguous");
  const int64_t batch = parents.size(0), beams = parents.size(1);
  NEED(beams >= 1 && beams <= 256 && batch <= 65535, "parents of shape ", parents.sizes(), ": 1 to 256 beams of up to 65535 sequences are supported");
  OneDevice on;
  const Listed states(x[0], "states");
  for (const L3Rows& r : states.rows) NEED(r.rows == batch * beams, "a state has ", r.rows, " rows for ", batch, " x ", beams, " beams");
  for (const Tensor& t : states.tensors) on.add(t, "states");
  on.add(parents, "parents");
  if (batch) {
    done(entry.reorder(on.index, on.stream(), states.rows.data(), size32(states.rows.size(), "states"), parents.const_data_ptr<int32_t>(), (int)batch,
                       (int)beams));
    for (const Tensor& t : states.tensors) changed(t);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// beam_select(logits, scores, best, done, eos_id)
PyObject* beam_select(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 5);
  const Tensor &logits = tensor(x[0], "logits", 3), &scores = tensor(x[1], "scores", 2);
  L3BeamSelect a{};
  a.dtype = kind(logits, "logits");
  const int64_t batch = logits.size(0), beams = logits.size(1), vocab = logits.size(2), best = given(x[2]) ? integer(x[2]) : beams;
  NEED(beams >= 1 && beams <= 256, beams, " beams: 1 to 256 are supported");
  NEED(best >= 1 && best <= 64, "best ", best, ": 1 to 64 are supported");
  NEED(vocab >= 1 && vocab < (1 << 24) && batch * beams <= 65535, "logits of shape ", logits.sizes(), " are too large");
  last_is_dense(logits, "logits");
  typed(scores, "scores", at::kFloat);
  NEED(scores.size(0) == batch && scores.size(1) == beams && scores.is_contiguous(), "scores must be contiguous, [", batch, ", ", beams, "], got ",
       scores.sizes());
  const int64_t eos = given(x[4]) ? integer(x[4]) : -1;
  NEED(eos < vocab && (eos >= 0 || !given(x[4])), "eos_id ", eos, " is not in the vocabulary of ", vocab);
  OneDevice on;
  if (given(x[3])) {
    const Tensor& d = tensor(x[3], "done", 2);
    NEED(d.scalar_type() == at::kBool || d.scalar_type() == at::kByte, "done: type ", d.scalar_type(), " is not bool");
    NEED(d.size(0) == batch && d.size(1) == beams && d.is_contiguous(), "done must be contiguous, [", batch, ", ", beams, "], got ", d.sizes());
    NEED(eos >= 0, "finished beams need an eos_id");
    a.done = static_cast<const uint8_t*>(d.const_data_ptr());
  }
  on.add(logits, "logits"); on.add(scores, "scores");
  if (given(x[3])) on.add(THPVariable_Unpack(x[3]), "done");
  const auto like = scores.options();
  const Tensor out[4] = {at::empty({batch, best}, like), at::empty({batch, best}, like.dtype(at::kInt)), at::empty({batch, best}, like.dtype(at::kInt)),
                         at::empty({batch, best}, like.dtype(at::kBool))};
  if (batch) {
    a.device = on.index; a.batch = (int)batch; a.beams = (int)beams; a.vocab = (int)vocab; a.best = (int)best; a.eos = (int)eos;
    a.stream = on.stream();
    a.logits = logits.const_data_ptr(); a.batch_stride = step_of(logits, 0); a.beam_stride = step_of(logits, 1);
    a.scores = scores.const_data_ptr<float>();
    a.out_scores = out[0].data_ptr<float>(); a.out_tokens = out[1].data_ptr<int32_t>(); a.out_parents = out[2].data_ptr<int32_t>();
    a.out_done = static_cast<uint8_t*>(out[3].data_ptr());
    done(entry.select_workspace(on.index, a.batch, a.beams, a.vocab, a.best, &a.workspace_bytes));
    const Tensor room = at::empty({a.workspace_bytes}, like.dtype(at::kByte));  // of this call: a captured graph has one of its own
    a.workspace = room.data_ptr();
    done(entry.select(&a));
  }
  PyObject* all = PyTuple_New(4);
  if (!all) throw python_error();
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(all, i, THPVariable_Wrap(out[i]));
  return all;
  END_HANDLE_TH_ERRORS
}

// A tuple of what a call returns; an undefined tensor is None.
PyObject* tuple_of(std::initializer_list<Tensor> list) {
  PyObject* all = PyTuple_New((Py_ssize_t)list.size());
  if (!all) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor& t : list) {
    PyObject* x = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    PyTuple_SET_ITEM(all, i++, x);
  }
  return all;
}
// Several small results in one piece of memory: an allocation costs a microsecond of the call.
struct Together {
  Tensor all;
  int64_t used = 0;
  static int64_t room(int64_t n, at::ScalarType type) { return (n * (int64_t)c10::elementSize(type) + 255) / 256 * 256; }
  Together(int64_t bytes, const at::TensorOptions& like) : all(at::empty({bytes}, like.dtype(at::kByte))) {}
  Tensor take(at::IntArrayRef sizes, at::ScalarType type) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(type));
    impl->set_storage_offset(used / (int64_t)c10::elementSize(type));
    impl->set_sizes_contiguous(sizes);
    used += room(impl->numel(), type);
    return Tensor(std::move(impl));
  }
};
void no_overlap(const Tensor& t, const char* name) {
  for (int64_t d = 0; d < t.dim(); ++d) NEED(t.size(d) <= 1 || t.stride(d) != 0, name, " is expanded, and would be written");
}
// whether the stretches of memory from the first entry to the last meet
bool meets(const Tensor& a, const Tensor& b) {
  auto end = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return (uintptr_t)t.const_data_ptr() + (last + 1) * t.element_size();
  };
  return a.numel() && b.numel() && (uintptr_t)a.const_data_ptr() < end(b) && (uintptr_t)b.const_data_ptr() < end(a);
}
int page_of(int64_t page) {
  NEED(page >= 1 && page <= 65536 && (page & (page - 1)) == 0, "page size ", page, " is not a power of two up to 65536");
  return (int)page;
}

// paged_extend(page_table, lengths, counts, free_pages, page_size, tokens)
PyObject* paged_extend(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 6);
  const Tensor& lengths = tensor(x[1], "lengths", 1);
  const int64_t batch = lengths.size(0);
  const Tensor& table = table_of(x[0], batch);
  const Tensor &counts = tensor(x[2], "counts", 1), &pages = tensor(x[3], "free_pages", 1);
  L3PagedExtend a{};
  a.batch = size32(batch, "batch");
  a.lengths = ints(lengths, "lengths", batch);
  a.counts = ints(counts, "counts", batch);
  a.n_free = size32(pages.size(0), "free_pages");
  a.free_pages = ints(pages, "free_pages", a.n_free);
  a.page_size = page_of(integer(x[4]));
  const int64_t tokens = integer(x[5]);
  NEED(tokens >= 0, "tokens ", tokens);
  a.tokens = size32(tokens, "tokens");
  a.max_pages = size32(table.size(1), "page_table");
  NEED(batch <= 1 || table.size(1) == 0 || table.stride(0) >= table.size(1), "page_table is expanded, and would be written");
  for (const Tensor* t : {&lengths, &counts, &pages}) NEED(!meets(table, *t), "page_table shares memory with lengths, counts or free_pages");
  OneDevice on;
  on.add(table, "page_table"); on.add(lengths, "lengths"); on.add(counts, "counts"); on.add(pages, "free_pages");
  const auto like = lengths.options();
  Together made(3 * 256 + Together::room(batch, at::kInt) * 2 + Together::room(tokens, at::kInt) + Together::room(tokens, at::kLong), like);
  const Tensor len = made.take({batch}, at::kInt), starts = made.take({batch + 1}, at::kInt), positions = made.take({tokens}, at::kInt),
               slots = made.take({tokens}, at::kLong), used = made.take({1}, at::kInt);
  a.device = on.index;
  a.stream = on.stream();
  a.table = table.data_ptr<int32_t>(); a.table_stride = step_of(table, 0);
  a.out_lengths = len.data_ptr<int32_t>(); a.out_starts = starts.data_ptr<int32_t>(); a.out_positions = positions.data_ptr<int32_t>();
  a.out_slots = slots.data_ptr<int64_t>(); a.out_used = used.data_ptr<int32_t>();
  done(entry.extend(&a));
  if (batch && tokens) changed(table);
  return tuple_of({len, starts, positions, slots, used});
  END_HANDLE_TH_ERRORS
}

// what every rotary call has: positions of `rows`, frequencies, layout, amplitude, inverse
void turn_of(L3Rotary& a, const Tensor& positions, PyObject* frequencies, PyObject* layout, PyObject* amplitude, PyObject* inverse) {
  typed(positions, "positions", at::kInt);
  NEED(positions.is_contiguous(), "positions must be contiguous");
  const Tensor& f = tensor(frequencies, "frequencies", 1);
  typed(f, "frequencies", at::kDouble);
  NEED(f.is_contiguous(), "frequencies must be contiguous");
  NEED(a.head_dim <= 1024, "head size ", a.head_dim, ": up to 1024 are supported");
  NEED(2 * f.size(0) <= a.head_dim, f.size(0), " frequencies for heads of ", a.head_dim);
  a.dims = 2 * (int)f.size(0);
  const char* name = PyUnicode_Check(layout) ? PyUnicode_AsUTF8(layout) : nullptr;
  NEED(name && (std::string(name) == "pairs" || std::string(name) == "halves"), "layout must be \"pairs\" or \"halves\"");
  a.layout = std::string(name) == "halves";
  a.amplitude = (float)real(amplitude);
  a.inverse = inverse == Py_True;
  a.positions = positions.const_data_ptr<int32_t>();
  a.frequencies = f.const_data_ptr<double>();
}
bool same_place(const Tensor& a, const Tensor& b) { return a.const_data_ptr() == b.const_data_ptr() && a.strides() == b.strides(); }

// rotary(x, positions, frequencies, layout, amplitude, inverse, out)
PyObject* rotary(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 7);
  const Tensor& t = tensor(x[0], "x");
  NEED(t.dim() == 3 || t.dim() == 4, "x must be [tokens, heads, size] or [batch, tokens, heads, size], got ", t.sizes());
  const int64_t d = t.dim() - 3;
  L3Rotary a{};
  a.dtype = kind(t, "x");
  last_is_dense(t, "x");
  const Tensor& positions = tensor(x[1], "positions");
  NEED(positions.sizes() == t.sizes().slice(0, d + 1), "positions must be ", t.sizes().slice(0, d + 1), ", got ", positions.sizes());
  a.batch = d ? size32(t.size(0), "batch") : 1;
  a.tokens = size32(t.size(d), "tokens"); a.heads = size32(t.size(d + 1), "heads"); a.head_dim = size32(t.size(d + 2), "head size");
  turn_of(a, positions, x[2], x[3], x[4], x[5]);
  if (given(x[6])) {
    const Tensor& o = tensor(x[6], "out");
    typed(o, "out", t.scalar_type());
    NEED(o.sizes() == t.sizes(), "out must be ", t.sizes(), ", got ", o.sizes());
    last_is_dense(o, "out");
    no_overlap(o, "out");
    NEED(!meets(o, t) || same_place(o, t), "out shares memory with x and is not x itself");
  }
  OneDevice on;
  on.add(t, "x"); on.add(positions, "positions"); on.add(THPVariable_Unpack(x[2]), "frequencies");
  if (given(x[6])) on.add(THPVariable_Unpack(x[6]), "out");
  const Tensor out = given(x[6]) ? THPVariable_Unpack(x[6]) : at::empty(t.sizes(), t.options());
  a.device = on.index;
  a.stream = on.stream();
  a.x = t.const_data_ptr();
  a.x_batch_stride = d ? step_of(t, 0) : 0; a.x_token_stride = step_of(t, d); a.x_head_stride = step_of(t, d + 1);
  a.out = out.data_ptr();
  a.out_batch_stride = d ? step_of(out, 0) : 0; a.out_token_stride = step_of(out, d); a.out_head_stride = step_of(out, d + 1);
  if (t.numel()) {
    done(entry.rotary(&a));
    if (given(x[6])) changed(out);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// paged_rotary_write(q, k, v, positions, slots, k_pages, v_pages, frequencies, layout, amplitude, out)
PyObject* paged_rotary_write(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 11);
  const Tensor &q = tensor(x[0], "q", 3), &k = tensor(x[1], "k", 3), &v = tensor(x[2], "v", 3), &kp = tensor(x[5], "k_pages", 4),
               &vp = tensor(x[6], "v_pages", 4);
  L3Rotary a{};
  a.dtype = pools_of(kp, vp);
  const int64_t tokens = q.size(0), G = kp.size(1), dim = kp.size(3);
  typed(q, "q", kp.scalar_type());
  NEED(q.size(2) == dim, "q must be [", tokens, ", heads, ", dim, "], got ", q.sizes());
  last_is_dense(q, "q");
  for (const Tensor* t : {&k, &v}) {
    const char* name = t == &k ? "k" : "v";
    typed(*t, name, kp.scalar_type());
    NEED(t->size(0) == tokens && t->size(1) == G && t->size(2) == dim, name, " must be [", tokens, ", ", G, ", ", dim, "], got ", t->sizes());
    last_is_dense(*t, name);
  }
  own_places(kp, "k_pages");
  own_places(vp, "v_pages");
  const Tensor &positions = tensor(x[3], "positions", 1), &slots = tensor(x[4], "slots", 1);
  NEED(positions.size(0) == tokens, "positions must be [", tokens, "], got ", positions.sizes());
  typed(slots, "slots", at::kLong);
  NEED(slots.size(0) == tokens && slots.is_contiguous(), "slots must be contiguous, [", tokens, "], got ", slots.sizes());
  a.batch = 1;
  a.tokens = size32(tokens, "tokens"); a.heads = size32(q.size(1), "heads"); a.head_dim = size32(dim, "head size"); a.kv_heads = size32(G, "kv heads");
  a.pages = size32(kp.size(0), "pages"); a.page_size = (int)kp.size(2);
  turn_of(a, positions, x[7], x[8], x[9], Py_False);
  if (given(x[10])) {
    const Tensor& o = tensor(x[10], "out", 3);
    typed(o, "out", q.scalar_type());
    NEED(o.sizes() == q.sizes(), "out must be ", q.sizes(), ", got ", o.sizes());
    last_is_dense(o, "out");
    no_overlap(o, "out");
    NEED(same_place(o, q) || !(meets(o, q) || meets(o, k) || meets(o, v)), "out shares memory with q, k or v and is not q itself");
    NEED(!meets(o, kp) && !meets(o, vp), "out shares memory with the pools");
  }
  OneDevice on;
  on.add(q, "q"); on.add(k, "k"); on.add(v, "v"); on.add(positions, "positions"); on.add(slots, "slots"); on.add(kp, "k_pages"); on.add(vp, "v_pages");
  on.add(THPVariable_Unpack(x[7]), "frequencies");
  if (given(x[10])) on.add(THPVariable_Unpack(x[10]), "out");
  const Tensor out = given(x[10]) ? THPVariable_Unpack(x[10]) : at::empty(q.sizes(), q.options());
  if (tokens) {
    a.device = on.index;
    a.stream = on.stream();
    a.x = q.const_data_ptr(); a.x_token_stride = step_of(q, 0); a.x_head_stride = step_of(q, 1);
    a.out = out.data_ptr(); a.out_token_stride = step_of(out, 0); a.out_head_stride = step_of(out, 1);
    a.k = k.const_data_ptr(); a.k_token_stride = step_of(k, 0); a.k_head_stride = step_of(k, 1);
    a.v = v.const_data_ptr(); a.v_token_stride = step_of(v, 0); a.v_head_stride = step_of(v, 1);
    a.slots = slots.const_data_ptr<int64_t>();
    a.k_pool = pool(kp); a.v_pool = pool(vp);
    done(entry.rotary(&a));
    changed(kp);
    changed(vp);
    if (given(x[10])) changed(out);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// paged_chunk_attention(q, k_pages, v_pages, page_table, lengths, starts, scale, return_lse, out)
PyObject* paged_chunk_attention(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 9);
  const Tensor &q = tensor(x[0], "q", 3), &k = tensor(x[1], "k_pages", 4), &v = tensor(x[2], "v_pages", 4), &lengths = tensor(x[4], "lengths", 1),
               &starts = tensor(x[5], "starts", 1);
  L3PagedChunk a{};
  a.dtype = pools_of(k, v);
  const int64_t batch = lengths.size(0), tokens = q.size(0), heads = q.size(1), dim = q.size(2), G = k.size(1);
  typed(q, "q", k.scalar_type());
  NEED(k.size(3) == dim && (dim == 16 || dim == 32 || dim == 48 || dim == 64 || dim == 96 || dim == 128), "head size ", dim, " (cache: ", k.size(3),
       ") is not one of 16, 32, 48, 64, 96, 128");
  NEED(G >= 1 && heads >= 1 && heads % G == 0, heads, " heads over ", G, " kv heads");
  last_is_dense(q, "q");
  fits16(q, "q");
  const Tensor& table = table_of(x[3], batch);
  a.lengths = ints(lengths, "lengths", batch);
  a.starts = ints(starts, "starts", batch + 1);
  if (given(x[8])) {
    const Tensor& out = tensor(x[8], "out", 3);
    typed(out, "out", q.scalar_type());
    NEED(out.sizes() == q.sizes() && out.is_contiguous() && (reinterpret_cast<uintptr_t>(out.const_data_ptr()) & 15) == 0,
         "out must be contiguous, of q's shape");
    for (const Tensor* t : {&q, &k, &v, &table, &lengths, &starts}) NEED(!meets(out, *t), "out shares memory with what is read");
  }
  OneDevice on;
  on.add(q, "q"); on.add(k, "k_pages"); on.add(v, "v_pages"); on.add(table, "page_table"); on.add(lengths, "lengths"); on.add(starts, "starts");
  if (given(x[8])) on.add(THPVariable_Unpack(x[8]), "out");
  const bool want_lse = x[7] == Py_True;
  const Tensor out = given(x[8]) ? THPVariable_Unpack(x[8]) : at::empty({tokens, heads, dim}, q.options());
  Tensor lse, room;
  if (want_lse) lse = at::empty({tokens, heads}, q.options().dtype(at::kFloat));
  if (tokens) {
    a.device = on.index; a.batch = size32(batch, "batch"); a.tokens = size32(tokens, "tokens"); a.heads = size32(heads, "heads"); a.kv_heads = size32(G, "kv heads");
    a.head_dim = (int)dim; a.pages = size32(k.size(0), "pages"); a.page_size = (int)k.size(2); a.max_pages = size32(table.size(1), "page_table");
    a.clear_rest = given(x[8]) ? 2 : 1;  // lse is made here
    a.scale = given(x[6]) ? (float)real(x[6]) : (float)(1.0 / std::sqrt((double)dim));
    a.stream = on.stream();
    a.q = q.const_data_ptr(); a.q_token_stride = step_of(q, 0); a.q_head_stride = step_of(q, 1);
    a.k = pool(k); a.v = pool(v);
    a.table = table.const_data_ptr<int32_t>(); a.table_stride = step_of(table, 0);
    a.out = out.data_ptr();
    a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
    done(entry.chunk_workspace(on.index, a.tokens, a.heads, a.kv_heads, a.head_dim, a.dtype, &a.workspace_bytes));
    room = at::empty({a.workspace_bytes}, q.options().dtype(at::kByte));  // of this call: a captured graph has one of its own
    a.workspace = room.data_ptr();
    done(entry.chunk(&a));
  }
  if (given(x[8])) changed(out);
  if (!want_lse) return THPVariable_Wrap(out);
  return tuple_of({out, lse});
  END_HANDLE_TH_ERRORS
}

// token_logprobs(logits, tokens, top, entropy)
PyObject* token_logprobs(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 4);
  const Tensor &logits = tensor(x[0], "logits", 2), &tokens = tensor(x[1], "tokens", 1);
  L3TokenLogprobs a{};
  a.dtype = kind(logits, "logits");
  const int64_t rows = logits.size(0), vocab = logits.size(1), top = integer(x[2]);
  NEED(vocab >= 1 && vocab < (1 << 24), "logits of shape ", logits.sizes(), ": 1 to 2^24 - 1 tokens are supported");
  NEED(top >= 0 && top <= 64 && top <= vocab, "top ", top, ": 0 to 64, and no more than the vocabulary's ", vocab, " are supported");
  last_is_dense(logits, "logits");
  a.tokens = ints(tokens, "tokens", rows);
  OneDevice on;
  on.add(logits, "logits"); on.add(tokens, "tokens");
  const auto like = logits.options().dtype(at::kFloat);
  Together made(Together::room(rows, at::kFloat) * 2 + Together::room(rows * top, at::kFloat) * 2, like);
  const Tensor lp = made.take({rows}, at::kFloat);
  Tensor entropy, best, best_tokens;
  if (x[3] == Py_True) entropy = made.take({rows}, at::kFloat);
  if (top) {
    best = made.take({rows, top}, at::kFloat);
    best_tokens = made.take({rows, top}, at::kInt);
  }
  if (rows) {
    a.device = on.index; a.rows = size32(rows, "rows"); a.vocab = (int)vocab; a.top = (int)top;
    a.stream = on.stream();
    a.logits = logits.const_data_ptr(); a.row_stride = step_of(logits, 0);
    a.out_logprobs = lp.data_ptr<float>();
    a.out_entropy = entropy.defined() ? entropy.data_ptr<float>() : nullptr;
    a.out_top_logprobs = top ? best.data_ptr<float>() : nullptr;
    a.out_top_tokens = top ? best_tokens.data_ptr<int32_t>() : nullptr;
    done(entry.logprobs(&a));
  }
  return tuple_of({lp, entropy, best, best_tokens});
  END_HANDLE_TH_ERRORS
}

// rows(tensor): how copy_pages and beam_reorder take a tensor (rows, row stride, runs of a row, their distance, their bytes)
PyObject* rows(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  args(n, 1);
  const L3Rows r = rows_of(tensor(x[0], "states"), "states", 0);
  return Py_BuildValue("LLLLL", (long long)r.rows, (long long)r.row_stride, (long long)r.outer, (long long)r.outer_stride, (long long)r.run);
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the C-ABI's entries, in Entries' order)
PyObject* bind(PyObject*, PyObject* const* x, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  constexpr int N = sizeof(Entries) / sizeof(void*);
  args(n, N);
  void* p[N];
  for (int i = 0; i < N; ++i) p[i] = reinterpret_cast<void*>(integer(x[i]));
  static_assert(sizeof(entry) == sizeof p, "");
  std::copy(p, p + N, reinterpret_cast<void**>(&entry));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"paged_attention", (PyCFunction)(void (*)())paged_attention, METH_FASTCALL, nullptr},
                         {"paged_write", (PyCFunction)(void (*)())paged_write, METH_FASTCALL, nullptr},
                         {"copy_pages", (PyCFunction)(void (*)())copy_pages, METH_FASTCALL, nullptr},
                         {"beam_reorder", (PyCFunction)(void (*)())beam_reorder, METH_FASTCALL, nullptr},
                         {"beam_select", (PyCFunction)(void (*)())beam_select, METH_FASTCALL, nullptr},
                         {"paged_extend", (PyCFunction)(void (*)())paged_extend, METH_FASTCALL, nullptr},
                         {"rotary", (PyCFunction)(void (*)())rotary, METH_FASTCALL, nullptr},
                         {"paged_rotary_write", (PyCFunction)(void (*)())paged_rotary_write, METH_FASTCALL, nullptr},
                         {"paged_chunk_attention", (PyCFunction)(void (*)())paged_chunk_attention, METH_FASTCALL, nullptr},
                         {"token_logprobs", (PyCFunction)(void (*)())token_logprobs, METH_FASTCALL, nullptr},
                         {"rows", (PyCFunction)(void (*)())rows, METH_FASTCALL, nullptr},
                         {"bind", (PyCFunction)(void (*)())bind, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }
