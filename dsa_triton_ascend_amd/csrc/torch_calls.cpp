// Short way from torch tensors into the C-ABI entry points of the paged
// decoding operators.  A decoding step makes several such calls per layer,
// and at its sizes the kernels take 5 us where the checks and conversions of
// a call in Python take 10.
//
// Each function checks that its call is an ordinary one (plain tensors of the
// documented shapes and types on the current GPU, nothing to convert) and makes it; for anything else, an entry point that
// refuses included, it returns None and the Python function goes its own way,
// which converts what may be converted and raises the errors.  An error of the
// HIP runtime is raised here: the kernels may have run by then (an error that
// another call left behind is reported by the next launch), and a rotation in
// place must not be made twice.
#include <torch/csrc/autograd/python_variable.h>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/Allocator.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <climits>
#include <stdexcept>
#include <utility>
#include <vector>

#include "../../include/dsa_capi.h"

namespace {

struct Entries {
  decltype(&dsa_rope) rope;
  decltype(&dsa_paged_cache_write) write;
  decltype(&dsa_paged_cache_fork_workspace_size) fork_bytes;
  decltype(&dsa_paged_cache_fork) fork;
  decltype(&dsa_paged_cache_compact_workspace_size) compact_bytes;
  decltype(&dsa_paged_cache_compact) compact;
  decltype(&dsa_paged_attn_workspace_size) attn_bytes;
  decltype(&dsa_paged_attn) attn;
  decltype(&dsa_last_error) error;
} entry;

// the HIP runtime reported an error at or before a launch
struct HipError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

// Whether an entry point made its launches; other Python threads run
// meanwhile, since a launch may wait for room in its queue.
template <typename F, typename... Args>
bool launched(F f, Args... args) {
  int status;
  if (!PyGILState_Check()) {  // (a thread of the autograd engine)
    status = f(args...);
  } else {
    PyThreadState* state = PyEval_SaveThread();
    status = f(args...);
    PyEval_RestoreThread(state);
  }
  if (status == DSA_ERR_HIP) throw HipError(entry.error());
  return status == DSA_OK;
}

constexpr int64_t kMaxCaches = 512;

// A plain tensor of the GPU of the call (the first tensor's; index -1 before
// it), else null.
const at::Tensor* tensor(PyObject* o, int* index) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_conj() || t.is_neg()) return nullptr;
  if (*index < 0) *index = (int)t.get_device();
  return t.get_device() == *index ? &t : nullptr;
}

// the tangent of a dual tensor (forward-mode derivatives), else undefined
const at::Tensor& tangent(const at::Tensor& t) { return t._fw_grad(/*level=*/0); }

// whether a derivative would be lost in an operator that has none
bool differentiable(const at::Tensor& t) {
  return (t.requires_grad() && c10::GradMode::is_enabled()) || tangent(t).defined();
}

const at::Tensor* ints(PyObject* o, int* index, int64_t dim) {
  const at::Tensor* t = tensor(o, index);
  return t && t->scalar_type() == at::kInt && t->dim() == dim && t->numel() > 0 && t->is_contiguous() ? t : nullptr;
}

bool integer(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow;
}

bool number(PyObject* o, double* v) {
  if (PyFloat_CheckExact(o)) *v = PyFloat_AS_DOUBLE(o);
  else if (PyLong_CheckExact(o)) *v = PyLong_AsDouble(o);
  else return false;
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool flag(PyObject* o, bool* v) {
  *v = o == Py_True;
  return PyBool_Check(o);
}

// "BSND" 0, "TND" 1, else -1
int layout(PyObject* o) {
  if (!PyUnicode_CheckExact(o)) return -1;
  if (PyUnicode_CompareWithASCIIString(o, "BSND") == 0) return 0;
  return PyUnicode_CompareWithASCIIString(o, "TND") == 0 ? 1 : -1;
}

// items of a tensor, list or tuple
bool items(PyObject* o, PyObject*** first, PyObject** self, int64_t* n) {
  if (PyList_CheckExact(o) || PyTuple_CheckExact(o)) {
    *n = PySequence_Fast_GET_SIZE(o);
    *first = PySequence_Fast_ITEMS(o);
    return *n <= kMaxCaches;
  }
  *self = o;
  *first = self;
  *n = 1;
  return true;
}

struct Caches {
  std::vector<const at::Tensor*> t;
  std::vector<void*> at;
  std::vector<int64_t> row_bytes;
  int64_t pages = 0, page = 0;

  bool read(PyObject* o, int* index) {
    PyObject **list, *self;
    int64_t n;
    if (!items(o, &list, &self, &n)) return false;
    t.reserve(n), at.reserve(n), row_bytes.reserve(n);
    for (int64_t i = 0; i < n; ++i) {
      const at::Tensor* c = tensor(list[i], index);
      if (!c || c->dim() < 3 || !c->is_contiguous() || c->numel() == 0) return false;
      if (i == 0) pages = c->size(0), page = c->size(1);
      if (c->size(0) != pages || c->size(1) != page || differentiable(*c)) return false;
      t.push_back(c);
      at.push_back(c->data_ptr());
      row_bytes.push_back(c->numel() / (pages * page) * (int64_t)c->element_size());
    }
    std::vector<int64_t> order(n);
    for (int64_t i = 0; i < n; ++i) order[i] = i;
    std::sort(order.begin(), order.end(), [&](int64_t a, int64_t b) { return at[a] < at[b]; });
    for (int64_t i = 1; i < n; ++i)
      if ((char*)at[order[i - 1]] + row_bytes[order[i - 1]] * pages * page > (char*)at[order[i]]) return false;
    return true;
  }
};

// Tells autograd that a tensor was changed in place: a backward that saved it
// raises instead of using the new values.  (Inference tensors are not saved.)
// Before the call: while it runs, another thread may drop the caller's tensors.
void changed(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void changed(const Caches& c) {
  for (const at::Tensor* t : c.t) changed(*t);
}

bool current(int index) { return index >= 0 && c10::hip::current_device() == index; }
void* stream_of(int index) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)index).stream(); }
const int32_t* data(const at::Tensor* t) { return t ? (const int32_t*)t->data_ptr() : nullptr; }

// (caches, rows, block_table, seq_lengths, row_lengths, layout) -> True
PyObject* write(PyObject* const* a) {
  const int tnd = layout(a[5]);
  int index = -1;
  Caches c;
  if (tnd < 0 || !c.read(a[0], &index) || c.t.empty()) return nullptr;
  const at::Tensor *table = ints(a[2], &index, 2), *lens = ints(a[3], &index, 1), *counts = nullptr;
  if (!table || !lens || !current(index)) return nullptr;
  const int64_t batch = table->size(0);
  if (a[4] != Py_None && (!(counts = ints(a[4], &index, 1)) || counts->size(0) != batch)) return nullptr;
  if (lens->size(0) != batch || (tnd && !counts)) return nullptr;
  PyObject **list, *self;
  int64_t n;
  if (!items(a[1], &list, &self, &n) || n != (int64_t)c.t.size()) return nullptr;
  const int64_t lead = tnd ? 1 : 2;
  std::vector<const void*> src(n);
  std::vector<int64_t> sb(n), st(n);
  int64_t t0 = 0, t1 = 0;
  for (int64_t i = 0; i < n; ++i) {
    const at::Tensor* r = tensor(list[i], &index);
    const at::Tensor& k = *c.t[i];
    if (!r || r->dim() != lead + k.dim() - 2 || r->scalar_type() != k.scalar_type() || differentiable(*r)) return nullptr;
    if (i == 0) t0 = r->size(0), t1 = tnd ? 1 : r->size(1);
    if (r->size(0) != t0 || (!tnd && (r->size(1) != t1 || t0 != batch))) return nullptr;
    int64_t step = 1;
    for (int64_t d = r->dim() - 1; d >= lead; --d) {
      if (r->size(d) != k.size(d - lead + 2) || (r->stride(d) != step && r->size(d) != 1)) return nullptr;
      step *= r->size(d);
    }
    const int64_t es = (int64_t)r->element_size();
    src[i] = r->data_ptr();
    sb[i] = tnd ? 0 : r->stride(0) * es;
    st[i] = r->stride(lead - 1) * es;
  }
  if (t0 * t1 == 0) return nullptr;
  changed(c);
  if (!launched(entry.write, n, src.data(), c.at.data(), c.row_bytes.data(), sb.data(), st.data(), data(table), data(lens),
                  data(counts), batch, tnd ? 0 : t1, t0 * t1, table->size(1), c.pages, c.page,
                  tnd ? DSA_LAYOUT_TND : DSA_LAYOUT_BSND, stream_of(index)))
    return nullptr;
  Py_RETURN_TRUE;
}

PyObject* triple(at::Tensor x, at::Tensor y, at::Tensor z) {
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(x)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(y)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(z)));
  return r;
}

// a new contiguous tensor beside t (what at::empty comes down to)
at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor& t, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, t.device(), std::nullopt));
}
at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor& t) { return fresh(sizes, t, t.scalar_type()); }

// memory of torch's allocator for a workspace: returned to it with the value,
// in the order of the current stream
c10::DataPtr workspace(size_t n) { return c10::GetAllocator(c10::kCUDA)->allocate(std::max<size_t>(n, 1)); }

// (caches, block_table, seq_lengths, page_refs, parents, new_tokens, page_size) -> triple
PyObject* fork(PyObject* const* a) {
  int index = -1;
  Caches c;
  int64_t more, page;
  if (!c.read(a[0], &index) || c.t.empty() || !integer(a[5], &more) || more < 0 || more > INT_MAX) return nullptr;
  if (a[6] != Py_None && (!integer(a[6], &page) || page != c.page)) return nullptr;
  const at::Tensor *table = ints(a[1], &index, 2), *lens = ints(a[2], &index, 1), *refs = ints(a[3], &index, 1);
  const at::Tensor* parents = nullptr;
  if (!table || !lens || !refs || !current(index)) return nullptr;
  if (a[4] != Py_None && !(parents = ints(a[4], &index, 1))) return nullptr;
  const int64_t rows = table->size(0), wide = table->size(1), children = parents ? parents->size(0) : rows;
  if (lens->size(0) != rows || refs->size(0) != c.pages) return nullptr;
  at::Tensor new_table = fresh({children, wide}, *table), new_lens = fresh({children}, *table);
  at::Tensor new_refs = fresh({c.pages}, *table);
  const size_t bytes = entry.fork_bytes(rows, children, c.pages);
  c10::DataPtr ws = workspace(bytes);
  changed(c);
  if (!launched(entry.fork, (int64_t)c.t.size(), c.at.data(), c.row_bytes.data(), data(table), data(lens), data(refs),
                 data(parents), (int32_t*)new_table.data_ptr(), (int32_t*)new_lens.data_ptr(),
                 (int32_t*)new_refs.data_ptr(), rows, children, wide, wide, c.pages, c.page, more, ws.get(),
                 bytes, stream_of(index)))
    return nullptr;
  return triple(std::move(new_table), std::move(new_lens), std::move(new_refs));
}

// (caches, block_table, page_refs, page_size) -> triple
PyObject* compact(PyObject* const* a) {
  int index = -1;
  Caches c;
  int64_t page;
  if (!c.read(a[0], &index) || c.t.empty()) return nullptr;
  if (a[3] != Py_None && (!integer(a[3], &page) || page != c.page)) return nullptr;
  const at::Tensor *table = ints(a[1], &index, 2), *refs = ints(a[2], &index, 1);
  if (!table || !refs || !current(index) || refs->size(0) != c.pages) return nullptr;
  at::Tensor new_table = fresh(table->sizes(), *table), new_refs = fresh({c.pages}, *table);
  at::Tensor map = fresh({c.pages}, *table);
  const size_t bytes = entry.compact_bytes(c.pages);
  c10::DataPtr ws = workspace(bytes);
  changed(c);
  if (!launched(entry.compact, (int64_t)c.t.size(), c.at.data(), c.row_bytes.data(), data(table), data(refs),
                    (int32_t*)new_table.data_ptr(), (int32_t*)new_refs.data_ptr(), (int32_t*)map.data_ptr(),
                    table->size(0), table->size(1), c.pages, c.page, ws.get(), bytes, stream_of(index)))
    return nullptr;
  return triple(std::move(new_table), std::move(new_refs), std::move(map));
}

// (query, key, value, block_table, actual_seq_lengths_kv, scale_value, query_rope, key_rope,
// actual_seq_lengths_query, sparse_mode, pre_tokens, next_tokens, return_softmax_lse) -> triple
PyObject* attention(PyObject* const* a) {
  int index = -1;
  const at::Tensor *q = tensor(a[0], &index), *k = tensor(a[1], &index), *v = nullptr, *qr = nullptr, *kr = nullptr;
  const at::Tensor *table = ints(a[3], &index, 2), *act_k = ints(a[4], &index, 1), *act_q = nullptr;
  const bool latent = a[2] == Py_None;
  double scale;
  int64_t mode, pre, next;
  bool lse;
  if (!q || !k || !table || !act_k || !current(index) || q->dim() != 4 || k->dim() != 4) return nullptr;
  if (!number(a[5], &scale) || !integer(a[9], &mode) || !integer(a[10], &pre) || !integer(a[11], &next) ||
      !flag(a[12], &lse) || (mode != 0 && mode != 3))
    return nullptr;
  const auto kind = q->scalar_type();
  auto cache = [&](const at::Tensor* t) {
    return t && t->scalar_type() == kind && t->is_contiguous() && t->numel() > 0 && !differentiable(*t);
  };
  if ((kind != at::kBFloat16 && kind != at::kHalf) || !cache(q) || !cache(k)) return nullptr;
  const int64_t b = q->size(0), s1 = q->size(1), n1 = q->size(2), d = q->size(3);
  const int64_t pages = k->size(0), page = k->size(1), n2 = k->size(2);
  if (k->size(3) != d || n1 % n2 || table->size(0) < b || act_k->size(0) != b) return nullptr;
  if (latent) {
    qr = tensor(a[6], &index), kr = tensor(a[7], &index);
    if (!cache(qr) || !cache(kr) || n2 != 1 || qr->sizes() != at::IntArrayRef({b, s1, n1, 64}) ||
        kr->sizes() != at::IntArrayRef({pages, page, 1, 64}))
      return nullptr;
  } else {
    v = tensor(a[2], &index);
    if (!cache(v) || a[6] != Py_None || a[7] != Py_None || v->sizes() != k->sizes()) return nullptr;
  }
  if (a[8] != Py_None && (!(act_q = ints(a[8], &index, 1)) || act_q->size(0) != b)) return nullptr;
  const int64_t wide = table->size(1);
  const size_t bytes = entry.attn_bytes(b, s1, n1, n2, d, latent, wide, page);
  if (!bytes) return nullptr;
  at::Tensor out = fresh(q->sizes(), *q), mx = fresh({b, n2, s1, n1 / n2}, *q, at::kFloat);
  at::Tensor sm = fresh({b, n2, s1, n1 / n2}, *q, at::kFloat);
  c10::DataPtr ws = workspace(bytes);
  if (!launched(entry.attn, q->data_ptr(), latent ? qr->data_ptr() : nullptr, k->data_ptr(), latent ? kr->data_ptr() : nullptr,
                 latent ? nullptr : v->data_ptr(), out.data_ptr(), (float*)mx.data_ptr(), (float*)sm.data_ptr(),
                 data(act_q), data(act_k), data(table), b, s1, n1, n2, d, latent ? 64 : 0, pages, page, wide,
                 (int32_t)mode, pre, next, kind == at::kHalf ? DSA_DTYPE_FP16 : DSA_DTYPE_BF16, (float)scale, lse,
                 ws.get(), bytes, stream_of(index)))
    return nullptr;
  return triple(std::move(out), std::move(mx), std::move(sm));
}

// whether two elements of a strided tensor may share an address
bool overlaps_itself(const at::Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> d;  // stride, size
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) d.emplace_back(t.stride(i), t.size(i));
  std::sort(d.begin(), d.end());
  int64_t reach = 0;
  for (const auto& x : d) {
    if (x.first <= reach) return true;
    reach += (x.second - 1) * x.first;
  }
  return false;
}

// Whether a sum of strides, each as often as its range allows, lies in
// [from, to].  Strides descend, so that what the later ones reach leaves each
// of them a few counts; true where those would be too many to go through.
struct Step {
  int64_t stride, lo, hi;
};
bool reaches(const std::vector<Step>& steps, size_t k, int64_t from, int64_t to, int* budget) {
  if (k == steps.size()) return from <= 0 && 0 <= to;
  int64_t least = 0, most = 0;
  for (size_t i = k + 1; i < steps.size(); ++i) {
    least += steps[i].stride * steps[i].lo;
    most += steps[i].stride * steps[i].hi;
  }
  const Step& s = steps[k];
  auto floor_div = [](int64_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
  const int64_t x0 = std::max(s.lo, -floor_div(most - from, s.stride)), x1 = std::min(s.hi, floor_div(to - least, s.stride));
  for (int64_t x = x0; x <= x1; ++x)
    if (--*budget < 0 || reaches(steps, k + 1, from - x * s.stride, to - x * s.stride, budget)) return true;
  return false;
}

// whether the `cols` columns from start[0] of a's heads and those from
// start[1] of b's share memory
bool share_memory(const at::Tensor& a, const at::Tensor& b, const int64_t start[2], int64_t cols) {
  const int64_t es = (int64_t)a.element_size(), size = cols * es;
  std::vector<Step> steps;
  auto add = [&](int64_t stride, int64_t lo, int64_t hi) {
    if (lo == hi) return;
    for (Step& s : steps)
      if (s.stride == stride) {
        s.lo += lo, s.hi += hi;
        return;
      }
    steps.push_back({stride, lo, hi});
  };
  for (int64_t i = 0; i + 1 < a.dim(); ++i) add(a.stride(i) * es, 1 - a.size(i), 0);
  for (int64_t i = 0; i + 1 < b.dim(); ++i) add(b.stride(i) * es, 0, b.size(i) - 1);
  std::sort(steps.begin(), steps.end(), [](const Step& x, const Step& y) { return x.stride > y.stride; });
  // b's columns lie this far behind a's, and a sum of steps more
  const int64_t apart = ((char*)b.data_ptr() + start[1] * es) - ((char*)a.data_ptr() + start[0] * es);
  int budget = 1000;
  return reaches(steps, 0, -apart - size + 1, -apart + size - 1, &budget);
}

struct Rotation {
  int64_t start[2];  // of the query's and the key's rotated columns
  double scale;
  bool tnd, interleaved, inverse;
};

// Rotates in[0] and, if defined, in[1] into out; false if the call is not an
// ordinary one.
bool rotated(const Rotation& r, const at::Tensor in[2], const at::Tensor& pos, const at::Tensor& freq, bool inplace,
             at::Tensor out[2]) {
  const at::Tensor& q = in[0];
  const int64_t rank = r.tnd ? 3 : 4, lead = rank - 2;
  const auto kind = q.scalar_type();
  const int dtype = kind == at::kBFloat16 ? DSA_DTYPE_BF16
                    : kind == at::kHalf   ? DSA_DTYPE_FP16
                    : kind == at::kFloat  ? DSA_DTYPE_FP32
                                          : -1;
  if (dtype < 0 || freq.scalar_type() != at::kDouble || freq.dim() != 1 || freq.size(0) < 1 || !freq.is_contiguous())
    return false;
  if ((pos.scalar_type() != at::kInt && pos.scalar_type() != at::kLong) || !pos.is_contiguous()) return false;
  const int64_t rot = 2 * freq.size(0);
  int64_t si[2][3] = {}, so[2][3] = {}, heads[2] = {}, cols[2] = {};
  void *from[2] = {}, *to[2] = {};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& t = in[i];
    if (!t.defined()) continue;
    if (t.dim() != rank || t.scalar_type() != kind || t.numel() == 0 || t._is_zerotensor()) return false;
    for (int64_t j = 0; j < lead; ++j)
      if (t.size(j) != q.size(j)) return false;
    cols[i] = t.size(rank - 1), heads[i] = t.size(lead);
    if ((t.stride(rank - 1) != 1 && cols[i] != 1) || r.start[i] < 0 || r.start[i] > cols[i] - rot) return false;
    if (inplace && (t.stride(rank - 1) != 1 || t.is_inference() || overlaps_itself(t))) return false;
    out[i] = inplace ? t : fresh(t.sizes(), t);
    for (int64_t j = 0; j < lead + 1; ++j) {
      si[i][j + r.tnd] = t.stride(j);
      so[i][j + r.tnd] = out[i].stride(j);
    }
    from[i] = t.data_ptr(), to[i] = out[i].data_ptr();
  }
  if (inplace && in[1].defined() && (from[0] == from[1] || share_memory(q, in[1], r.start, rot))) return false;
  const int64_t b = r.tnd ? 1 : q.size(0), s = q.size(lead - 1);
  const bool full = pos.dim() == lead && (r.tnd || pos.size(0) == b) && pos.size(lead - 1) == s;
  const bool shared = !r.tnd && pos.dim() == 1 && pos.size(0) == s;
  if (!full && !shared) return false;
  return launched(entry.rope, from[0], to[0], si[0][0], si[0][1], si[0][2], so[0][0], so[0][1], so[0][2], heads[0],
                  cols[0], r.start[0], from[1], to[1], si[1][0], si[1][1], si[1][2], so[1][0], so[1][1], so[1][2],
                  heads[1], cols[1], in[1].defined() ? r.start[1] : 0, pos.data_ptr(), pos.scalar_type() == at::kLong,
                  full, (const double*)freq.data_ptr(), b, s, rot, r.interleaved, r.inverse, dtype, (float)r.scale,
                  stream_of((int)q.get_device()));
}

bool rotated_with_gradient(const Rotation& r, const at::Tensor in[2], const at::Tensor& pos, const at::Tensor& freq,
                           at::Tensor out[2]);

// The gradient of a rotation is the rotation by the opposite angles, with the
// same scale; nothing of the forward but the positions is kept.
struct RotaryBackward : torch::autograd::Node {
  Rotation r;
  torch::autograd::SavedVariable pos, freq;

  std::string name() const override { return "RotaryEmbeddingBackward"; }

  void release_variables() override {
    pos.reset_data();
    freq.reset_data();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    torch::autograd::variable_list result = turned(grads);
    // the tangent of a gradient turns as the gradient does
    torch::autograd::variable_list tangents(grads.size());
    bool dual = false;
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads[i].defined() && tangent(grads[i]).defined()) tangents[i] = tangent(grads[i]), dual = true;
    if (dual) {
      tangents = turned(tangents);
      for (size_t i = 0; i < result.size(); ++i)
        if (result[i].defined() && tangents[i].defined()) result[i]._set_fw_grad(tangents[i], /*level=*/0, false);
    }
    return result;
  }

  torch::autograd::variable_list turned(const torch::autograd::variable_list& grads) {
    const at::Tensor p = pos.unpack(), f = freq.unpack();
    const size_t n = num_outputs();
    at::Tensor in[2], out[2];
    int place[2];  // whose gradient in[i] is
    int count = 0;
    Rotation back = r;
    back.inverse = !r.inverse;
    for (int i = 0; i < (int)n; ++i)
      if (grads[i].defined() && task_should_compute_output(i)) {
        if (grads[i]._is_zerotensor()) in[count] = at::zeros(grads[i].sizes(), grads[i].options());  // (it has no memory)
        else in[count] = grads[i].stride(-1) == 1 ? grads[i] : grads[i].contiguous();
        back.start[count] = r.start[i];
        place[count++] = i;
      }
    torch::autograd::variable_list result(n);
    if (!count) return result;
    const bool ok = c10::GradMode::is_enabled() ? rotated_with_gradient(back, in, p, f, out)
                                                : rotated(back, in, p, f, false, out);
    TORCH_CHECK(ok, "the backward of rotary_embedding could not be launched");
    for (int i = 0; i < count; ++i) result[place[i]] = out[i];
    return result;
  }
};

bool rotated_with_gradient(const Rotation& r, const at::Tensor in[2], const at::Tensor& pos, const at::Tensor& freq,
                           at::Tensor out[2]) {
  {
    c10::AutoGradMode off(false);
    if (!rotated(r, in, pos, freq, false, out)) return false;
  }
  const bool two = in[1].defined();
  if (!in[0].requires_grad() && !(two && in[1].requires_grad())) return true;
  std::shared_ptr<RotaryBackward> node(new RotaryBackward(), torch::autograd::deleteNode);
  node->r = r;
  node->pos = torch::autograd::SavedVariable(pos, false);
  node->freq = torch::autograd::SavedVariable(freq, false);
  node->set_next_edges(two ? torch::autograd::collect_next_edges(in[0], in[1])
                           : torch::autograd::collect_next_edges(in[0]));
  for (int i = 0; i < 1 + two; ++i) torch::autograd::set_history(out[i], node);
  return true;
}

// (query, key, positions, inv_freq, interleaved, rotary_offset, key_rotary_offset, attention_scale, layout,
// inverse, inplace) -> (query_out, key_out)
PyObject* rotate(PyObject* const* a) {
  const int tnd = layout(a[8]);
  int index = -1;
  const at::Tensor *q = tensor(a[0], &index), *k = nullptr, *pos = tensor(a[2], &index), *freq = tensor(a[3], &index);
  if (tnd < 0 || !q || !pos || !freq || !current(index)) return nullptr;
  if (a[1] != Py_None && !(k = tensor(a[1], &index))) return nullptr;
  if (tangent(*q).defined() || (k && tangent(*k).defined())) return nullptr;
  Rotation r;
  bool inplace;
  r.tnd = tnd;
  if (!flag(a[4], &r.interleaved) || !integer(a[5], &r.start[0]) || !number(a[7], &r.scale) ||
      !flag(a[9], &r.inverse) || !flag(a[10], &inplace))
    return nullptr;
  r.start[1] = r.start[0];
  if (a[6] != Py_None && !integer(a[6], &r.start[1])) return nullptr;
  const bool grad = c10::GradMode::is_enabled() && (q->requires_grad() || (k && k->requires_grad()));
  if (grad && (inplace || pos->requires_grad() || freq->requires_grad())) return nullptr;
  const at::Tensor in[2] = {*q, k ? *k : at::Tensor()};
  at::Tensor out[2];
  if (grad ? !rotated_with_gradient(r, in, *pos, *freq, out) : !rotated(r, in, *pos, *freq, inplace, out))
    return nullptr;
  if (inplace)
    for (auto& t : out)
      if (t.defined()) changed(t);
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(out[0])));
  if (!k) Py_INCREF(Py_None);
  PyTuple_SET_ITEM(pair, 1, k ? THPVariable_Wrap(std::move(out[1])) : Py_None);
  return pair;
}

// A call that is not an ordinary one, and one that torch refuses (no memory),
// is left to the Python function.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  PyObject* r = nullptr;
  if (n == N && entry.attn) {
    try {
      r = F(args);
    } catch (python_error& e) {
      // raised by Python code on the way (a hook on saved tensors, which
      // checkpoints stop their recomputation by): the caller's
      e.restore();
      return nullptr;
    } catch (const HipError& e) {
      PyErr_SetString(PyExc_RuntimeError, e.what());
      return nullptr;
    } catch (...) {
      r = nullptr;
    }
  }
  if (r) return r;
  if (PyErr_Occurred()) PyErr_Clear();
  Py_RETURN_NONE;
}

// addresses of the entry points, in the order of Entries
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr int kEntries = sizeof(Entries) / sizeof(void*);
  if (n != kEntries) {
    PyErr_SetString(PyExc_TypeError, "one address per entry point expected");
    return nullptr;
  }
  void* at[kEntries];
  for (int i = 0; i < kEntries; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  std::copy(at, at + kEntries, (void**)&entry);
  Py_RETURN_NONE;
}

#define FAST(f) ((PyCFunction)(void (*)(void))(f))
PyMethodDef methods[] = {
    {"bind", FAST(bind), METH_FASTCALL, nullptr},
    {"write", FAST((call<write, 6>)), METH_FASTCALL, nullptr},
    {"fork", FAST((call<fork, 7>)), METH_FASTCALL, nullptr},
    {"compact", FAST((call<compact, 4>)), METH_FASTCALL, nullptr},
    {"attention", FAST((call<attention, 13>)), METH_FASTCALL, nullptr},
    {"rotate", FAST((call<rotate, 11>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__torch_calls() { return PyModule_Create(&module); }
