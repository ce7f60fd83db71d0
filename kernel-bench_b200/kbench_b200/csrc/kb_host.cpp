// Host side of the row scores and the fitting step, as a Python extension: what is asked of every tensor
// of a list (address, count, dtype, device, layout, overlap) in one pass -- a list of 2,048 tensors takes
// 2 ms in Python, 0.1 ms here --, and whole calls for arguments that need no second look: score_rows,
// score_rows_backward, clip and adam check, allocate and launch, or return None for anything else,
// which the Python layer then refuses, copies or calls itself (a score_rows of one row 15 us of host
// time by way of Python, 10 here).
#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "kb_solver.h"

#include <algorithm>
#include <cstdint>
#include <utility>
#include <vector>

namespace {

enum Flags { kOtherDevice = 1, kOtherDtype = 2, kStrided = 4, kNotF32 = 8 };

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}

// The tensors of a list or tuple; false with a Python error set where it holds something else.
bool unpack(PyObject* seq, std::vector<const at::Tensor*>& out) {
  if (!PyList_Check(seq) && !PyTuple_Check(seq)) {
    PyErr_SetString(PyExc_TypeError, "expected a list of tensors");
    return false;
  }
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  out.reserve((size_t)n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(seq, i);
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "expected a list of tensors (item %zd is %s)", i, Py_TYPE(o)->tp_name);
      return false;
    }
    out.push_back(&THPVariable_Unpack(o));
  }
  return true;
}

// With torch's exceptions as the Python ones they stand for (the allocator's: torch.OutOfMemoryError).
template <typename F>
PyObject* guarded(const F& f) {
  HANDLE_TH_ERRORS
  return f();
  END_HANDLE_TH_ERRORS
}

// What a kernel wrote to through its address counts as changed in place: the version by which autograd and
// whoever remembers something of a tensor know it (inference tensors have none).  Views of one block share a
// counter, which moves on once, where it is still what it was: a step of an atomic is most of what this costs.
struct Written {
  std::vector<std::pair<at::TensorImpl*, uint32_t>> versions;  // as they are before the call
  void add(const at::Tensor& t) {
    at::TensorImpl* impl = t.unsafeGetTensorImpl();
    if (impl->version_counter().enabled()) versions.emplace_back(impl, impl->version_counter().current_version());
  }
  void mark() const {
    for (const auto& [impl, was] : versions)
      if (impl->version_counter().current_version() == was) impl->bump_version();
  }
};

struct Span {
  uintptr_t begin, end;
  uint32_t i;
  bool written;
};

// Whether two written spans meet, or a written one meets a read one; with in_place, written span i may
// be read span i itself.  Sorts the spans of each list, then merges.
bool spans_meet(std::vector<Span>& spans, const std::vector<size_t>& list_ends, bool in_place) {
  const auto before = [](const Span& x, const Span& y) {
    return x.begin != y.begin ? x.begin < y.begin : x.written > y.written;
  };
  size_t from = 0;
  for (const size_t to : list_ends) {
    const auto a = spans.begin() + (std::ptrdiff_t)from, b = spans.begin() + (std::ptrdiff_t)to;
    // tensors made one after another are mostly in order already
    if (!std::is_sorted(a, b, before)) std::sort(a, b, before);
    std::inplace_merge(spans.begin(), a, b, before);
    from = to;
  }
  Span last_w{0, 0, 0, true}, last_r{0, 0, 0, false};  // the furthest end so far, and whose it is
  for (const Span& s : spans) {
    const bool itself = in_place && !s.written && s.i == last_w.i && s.begin == last_w.begin && s.end == last_w.end;
    if (s.begin < last_w.end && !itself) return true;
    if (s.written && s.begin < last_r.end) return true;
    Span& last = s.written ? last_w : last_r;
    if (s.end > last.end) last = s;
  }
  return false;
}

// What is asked of lists of tensors.  The first n_written are written, the others read.
struct Lists {
  size_t n = 0;
  std::vector<std::vector<int64_t>> ptrs;  // per list, as the C entry points take them
  std::vector<std::vector<int32_t>> dtypes;
  Written written;
  std::vector<int64_t> counts;             // of the first list
  std::vector<int> flags;                  // what is unusual in each list
  bool same = false;                       // tensor i has the same shape in all
  bool meet = false;  // written tensors share memory with one another or with read ones (with in_place, written
                      // tensor i may be read tensor i), each taken to fill its memory

  // False with a Python error set where a list holds something else.
  bool look(PyObject* const* lists, size_t n_lists, int device, int n_written, bool in_place) {
    std::vector<std::vector<const at::Tensor*>> ts(n_lists);
    same = n_lists > 0;
    for (size_t l = 0; l < n_lists; ++l) {
      if (!unpack(lists[l], ts[l])) return false;
      same = same && ts[l].size() == ts[0].size();
    }
    n = n_lists ? ts[0].size() : 0;
    ptrs.resize(n_lists);
    dtypes.resize(n_lists);
    flags.assign(n_lists, 0);
    written.versions.reserve(n * (size_t)std::max(n_written, 0));
    counts.assign(n, 0);
    std::vector<std::vector<Span>> spans(n_lists);
    for (size_t l = 0; l < n_lists; ++l) {
      ptrs[l].assign(ts[l].size(), 0);
      dtypes[l].assign(ts[l].size(), 0);
      spans[l].reserve(ts[l].size());
    }
    const auto one = [&](size_t l, size_t i) {
      const at::Tensor& t = *ts[l][i];
      if (!t.is_cuda() || t.layout() != at::kStrided || t.device().index() != device) {
        flags[l] |= kOtherDevice;
        return;
      }
      const int code = dtype_code(t.scalar_type());
      if (code < 0) flags[l] |= kOtherDtype;
      if (code != 0) flags[l] |= kNotF32;
      if (!t.is_contiguous()) flags[l] |= kStrided;
      const int64_t count = t.numel();
      if (l == 0) counts[i] = count;
      if ((int)l < n_written) written.add(t);
      dtypes[l][i] = code < 0 ? 0 : code;
      if (count == 0) return;
      const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
      ptrs[l][i] = (int64_t)p;
      spans[l].push_back({p, p + (uintptr_t)count * t.element_size(), (uint32_t)i, (int)l < n_written});
    };
    if (!same) return true;
    for (size_t i = 0; i < n; ++i) {
      const at::IntArrayRef sizes = ts[0][i]->sizes();
      for (size_t l = 0; l < n_lists; ++l) {
        one(l, i);
        same = same && (l == 0 || ts[l][i]->sizes() == sizes);
      }
    }
    if (same && n_written > 0) {
      std::vector<Span> all;
      std::vector<size_t> ends;
      for (auto& s : spans) {
        all.insert(all.end(), s.begin(), s.end());
        ends.push_back(all.size());
      }
      meet = spans_meet(all, ends, in_place);
    }
    return true;
  }
  bool usual(size_t l, bool f32) const {
    return (flags[l] & (kOtherDevice | kOtherDtype | kStrided | (f32 ? kNotF32 : 0))) == 0;
  }
};

// gather(lists, device index, n_written, in_place) -> (described, flags, same, meet): Lists, described being
// per list (addresses int64, dtypes int32) as bytes and the first list's counts int64 last.
PyObject* gather(PyObject*, PyObject* args) {
  PyObject* lists;
  int device, n_written, in_place;
  if (!PyArg_ParseTuple(args, "O!iip", &PyTuple_Type, &lists, &device, &n_written, &in_place)) return nullptr;
  return guarded([&]() -> PyObject* {
    const size_t n_lists = (size_t)PyTuple_GET_SIZE(lists);
    std::vector<PyObject*> items;
    for (size_t l = 0; l < n_lists; ++l) items.push_back(PyTuple_GET_ITEM(lists, (Py_ssize_t)l));
    Lists x;
    if (!x.look(items.data(), n_lists, device, n_written, in_place)) return nullptr;
    const auto bytes = [](const void* p, size_t size) { return PyBytes_FromStringAndSize((const char*)p, (Py_ssize_t)size); };
    PyObject* described = PyTuple_New((Py_ssize_t)n_lists + 1);
    PyObject* flag_tuple = PyTuple_New((Py_ssize_t)n_lists);
    if (!described || !flag_tuple) {
      Py_XDECREF(described);
      Py_XDECREF(flag_tuple);
      return nullptr;
    }
    for (size_t l = 0; l < n_lists; ++l) {
      PyTuple_SET_ITEM(described, (Py_ssize_t)l,
                       Py_BuildValue("(NN)", bytes(x.ptrs[l].data(), 8 * x.ptrs[l].size()),
                                     bytes(x.dtypes[l].data(), 4 * x.dtypes[l].size())));
      PyTuple_SET_ITEM(flag_tuple, (Py_ssize_t)l, PyLong_FromLong(x.flags[l]));
    }
    PyTuple_SET_ITEM(described, (Py_ssize_t)n_lists, bytes(x.counts.data(), 8 * x.counts.size()));
    return Py_BuildValue("(NNNN)", described, flag_tuple, PyBool_FromLong(x.same), PyBool_FromLong(x.meet));
  });
}

// overlap(written, read, in_place): gather's `meet` alone, of tensors on any device, so that the search can be tested
// without a GPU.
PyObject* overlap(PyObject*, PyObject* args) {
  PyObject *a, *b;
  int in_place;
  if (!PyArg_ParseTuple(args, "OOp", &a, &b, &in_place)) return nullptr;
  return guarded([&]() -> PyObject* {
    std::vector<const at::Tensor*> ts[2];
    if (!unpack(a, ts[0]) || !unpack(b, ts[1])) return nullptr;
    std::vector<Span> spans;
    std::vector<size_t> ends;
    for (int l = 0; l < 2; ++l) {
      for (size_t i = 0; i < ts[l].size(); ++i) {
        if (ts[l][i]->numel() == 0) continue;
        const uintptr_t p = reinterpret_cast<uintptr_t>(ts[l][i]->data_ptr());
        spans.push_back({p, p + ts[l][i]->nbytes(), (uint32_t)i, l == 0});
      }
      ends.push_back(spans.size());
    }
    return PyBool_FromLong(spans_meet(spans, ends, in_place));
  });
}

// written(list): what the Python layer's own calls wrote to.
PyObject* written(PyObject*, PyObject* list) {
  return guarded([&]() -> PyObject* {
    std::vector<const at::Tensor*> ts;
    if (!unpack(list, ts)) return nullptr;
    Written w;
    for (const at::Tensor* t : ts) w.add(*t);
    w.mark();
    Py_RETURN_NONE;
  });
}

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

// The six tensors of RowScores for rows, given (or NULL) and top.
PyObject* empty_scores(const at::Tensor& rows, const at::Tensor* given, int64_t top, at::Tensor (&t)[6]) {
  const int64_t R = rows.size(0);
  const auto f32 = at::TensorOptions().device(rows.device()).dtype(at::kFloat);
  t[0] = at::empty({R}, f32);
  t[1] = at::empty({R}, f32);
  if (given) t[2] = at::empty(given->sizes(), f32);
  if (top) {
    t[3] = at::empty({R, top}, f32);
    t[4] = at::empty({R, top}, f32.dtype(at::kLong));
  }
  t[5] = at::empty({R, 2}, f32);
  PyObject* out = PyTuple_New(6);
  if (!out) return nullptr;
  for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(out, i, t[i].defined() ? wrap(t[i]) : Py_NewRef(Py_None));
  return out;
}

// score_outputs(rows, given or None, top) -> the six tensors of RowScores.
PyObject* score_outputs(PyObject*, PyObject* args) {
  PyObject *rows_o, *given_o;
  long long top;
  if (!PyArg_ParseTuple(args, "OOL", &rows_o, &given_o, &top)) return nullptr;
  return guarded([&]() -> PyObject* {
    if (!THPVariable_Check(rows_o) || (given_o != Py_None && !THPVariable_Check(given_o))) {
      PyErr_SetString(PyExc_TypeError, "expected tensors");
      return nullptr;
    }
    at::Tensor t[6];
    return empty_scores(THPVariable_Unpack(rows_o), given_o == Py_None ? nullptr : &THPVariable_Unpack(given_o), top, t);
  });
}

// Whether a row matrix can be taken as it is, on the device.
bool usual_rows(const at::Tensor& t, int device) {
  return t.is_cuda() && t.layout() == at::kStrided && t.device().index() == device && dtype_code(t.scalar_type()) >= 0 &&
         t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1);
}
// None, or given columns that can be; *n columns a row.
bool usual_given(PyObject* o, int device, int64_t R, const at::Tensor** t, int* n) {
  *t = nullptr;
  *n = 0;
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& g = THPVariable_Unpack(o);
  if (!g.is_cuda() || g.device().index() != device || g.scalar_type() != at::kLong || !g.is_contiguous() ||
      (g.dim() != 1 && g.dim() != 2) || g.size(0) != R || (g.dim() == 2 && g.size(1) > KB_MAX_GIVEN))
    return false;
  *t = &g;
  *n = g.dim() == 1 ? 1 : (int)g.size(1);
  return true;
}
// None, or an fp32 tensor of these sizes that can be; *p its address.
bool usual_f32(PyObject* o, int device, at::IntArrayRef sizes, const float** p) {
  *p = nullptr;
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.device().index() != device || t.scalar_type() != at::kFloat || !t.is_contiguous() ||
      t.sizes() != sizes)
    return false;
  *p = t.data_ptr<float>();
  return true;
}
uintptr_t address(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }

// score_rows(kb_score_rows, rows, given or None, top, natural, device index, stream) -> (status, outputs), or
// None.
PyObject* score_rows(PyObject*, PyObject* args) {
  unsigned long long fn, stream;
  PyObject *rows_o, *given_o;
  int top, natural, device;
  if (!PyArg_ParseTuple(args, "KOOiiiK", &fn, &rows_o, &given_o, &top, &natural, &device, &stream)) return nullptr;
  return guarded([&]() -> PyObject* {
    if (!THPVariable_Check(rows_o)) Py_RETURN_NONE;
    const at::Tensor& rows = THPVariable_Unpack(rows_o);
    const at::Tensor* given;
    int n_given;
    if (!usual_rows(rows, device) || top < 0 || top > KB_MAX_TOP || rows.size(1) > KB_MAX_SCORE_COLS ||
        !usual_given(given_o, device, rows.size(0), &given, &n_given))
      Py_RETURN_NONE;
    at::Tensor t[6];
    PyObject* out = empty_scores(rows, given, top, t);
    if (!out) return nullptr;
    const int status = reinterpret_cast<decltype(&kb_score_rows)>(fn)(
        rows.data_ptr(), rows.stride(0), dtype_code(rows.scalar_type()), rows.size(0), (int)rows.size(1), natural,
        given ? reinterpret_cast<const long long*>(given->data_ptr()) : nullptr, n_given, top, t[0].data_ptr<float>(),
        t[1].data_ptr<float>(), given ? t[2].data_ptr<float>() : nullptr, top ? t[3].data_ptr<float>() : nullptr,
        top ? reinterpret_cast<long long*>(t[4].data_ptr()) : nullptr, t[5].data_ptr<float>(), (void*)stream);
    return Py_BuildValue("(iN)", status, out);
  });
}

// score_rows_backward(kb_score_rows_backward, rows, stats, entropy, given, grad_log_mass, grad_given,
// grad_entropy, natural, out, device index, stream) -> (status, gradient), or None; all but rows and stats may be
// None.
PyObject* score_rows_backward(PyObject*, PyObject* args) {
  unsigned long long fn, stream;
  PyObject *rows_o, *stats_o, *entropy_o, *given_o, *gm_o, *gg_o, *ge_o, *out_o;
  int natural, device;
  if (!PyArg_ParseTuple(args, "KOOOOOOOiOiK", &fn, &rows_o, &stats_o, &entropy_o, &given_o, &gm_o, &gg_o, &ge_o, &natural,
                        &out_o, &device, &stream))
    return nullptr;
  return guarded([&]() -> PyObject* {
    if (!THPVariable_Check(rows_o) || (out_o != Py_None && !THPVariable_Check(out_o))) Py_RETURN_NONE;
    const at::Tensor& rows = THPVariable_Unpack(rows_o);
    if (!usual_rows(rows, device) || rows.size(1) > KB_MAX_SCORE_COLS) Py_RETURN_NONE;
    const int64_t R = rows.size(0), S = rows.size(1);
    const at::Tensor* given;
    int n_given;
    const float *stats, *entropy, *gm, *gg, *ge;
    if (!usual_f32(stats_o, device, {R, 2}, &stats) || stats_o == Py_None ||
        !usual_f32(entropy_o, device, {R}, &entropy) || !usual_given(given_o, device, R, &given, &n_given) ||
        !usual_f32(gm_o, device, {R}, &gm) || !usual_f32(ge_o, device, {R}, &ge) ||
        (gg_o != Py_None && !given) || !usual_f32(gg_o, device, given ? given->sizes() : at::IntArrayRef(), &gg) ||
        (ge_o != Py_None && entropy_o == Py_None))
      Py_RETURN_NONE;
    at::Tensor out;
    if (out_o == Py_None) {
      out = at::empty({R, S}, rows.options());
    } else {
      out = THPVariable_Unpack(out_o);
      const auto end = [](const at::Tensor& t) {
        return t.numel() ? address(t) + (uintptr_t)((t.size(0) - 1) * t.stride(0) + t.size(1)) * t.element_size()
                         : address(t);
      };
      if (!usual_rows(out, device) || out.scalar_type() != rows.scalar_type() || out.sizes() != rows.sizes() ||
          (R > 1 && out.stride(0) < S) || (address(out) < end(rows) && address(rows) < end(out)))
        Py_RETURN_NONE;
    }
    const int status = reinterpret_cast<decltype(&kb_score_rows_backward)>(fn)(
        rows.data_ptr(), rows.stride(0), dtype_code(rows.scalar_type()), R, (int)S, natural, stats, entropy,
        given ? reinterpret_cast<const long long*>(given->data_ptr()) : nullptr, n_given, gm, gg, ge, out.data_ptr(),
        out.stride(0), (void*)stream);
    if (status == 0 && out_o != Py_None) {
      Written w;
      w.add(out);
      w.mark();
    }
    return Py_BuildValue("(iN)", status, out_o == Py_None ? wrap(out) : Py_NewRef(out_o));
  });
}

struct Buffers {
  at::Tensor norm, ws;
  Buffers(int device, int64_t bytes) {
    const auto on = at::TensorOptions().device(at::Device(at::kCUDA, (at::DeviceIndex)device));
    norm = at::empty({}, on.dtype(at::kFloat));
    ws = at::empty({bytes}, on.dtype(at::kByte));
  }
};

// clip(kb_clip_gradients, grads, out list or None, write, kind, max_norm, workspace bytes, device index, stream) ->
// (status, norm), or None.  out None: in place with `write`, else the norm alone.
PyObject* clip(PyObject*, PyObject* args) {
  unsigned long long fn, stream;
  PyObject *grads, *outs;
  int write, kind, device;
  double max_norm;
  long long bytes;
  if (!PyArg_ParseTuple(args, "KOOpidLiK", &fn, &grads, &outs, &write, &kind, &max_norm, &bytes, &device, &stream))
    return nullptr;
  return guarded([&]() -> PyObject* {
    const bool apart = outs != Py_None;
    PyObject* const lists[2] = {apart ? outs : grads, grads};
    Lists x;
    if (!x.look(lists, apart ? 2 : 1, device, write ? 1 : 0, true)) return nullptr;
    const size_t g = apart ? 1 : 0;
    if (!x.same || x.meet || !x.usual(0, false) || !x.usual(g, false) || x.dtypes[0] != x.dtypes[g] || x.n == 0)
      Py_RETURN_NONE;
    Buffers b(device, bytes);
    const auto* src = reinterpret_cast<const long long*>(x.ptrs[g].data());
    const auto* dst = reinterpret_cast<const long long*>(x.ptrs[0].data());
    const int status = reinterpret_cast<decltype(&kb_clip_gradients)>(fn)(
        src, write ? dst : nullptr, reinterpret_cast<const long long*>(x.counts.data()), x.dtypes[g].data(), (int)x.n, kind,
        max_norm, b.norm.data_ptr<float>(), b.ws.data_ptr(), bytes, (void*)stream);
    if (status == 0 && write) x.written.mark();
    return Py_BuildValue("(iN)", status, wrap(b.norm));
  });
}

// adam(kb_adam_step, params, grads, exp_avg, exp_avg_sq, lr, beta1, beta2, eps, weight_decay, correction1,
// correction2, kind, max_norm, workspace bytes, device index, stream) -> (status, norm), or None.
PyObject* adam(PyObject*, PyObject* args) {
  unsigned long long fn, stream;
  PyObject *p, *g, *m, *v;
  double lr, b1, b2, eps, wd, c1, c2, max_norm;
  int kind, device;
  long long bytes;
  if (!PyArg_ParseTuple(args, "KOOOOdddddddidLiK", &fn, &p, &g, &m, &v, &lr, &b1, &b2, &eps, &wd, &c1, &c2, &kind, &max_norm,
                        &bytes, &device, &stream))
    return nullptr;
  return guarded([&]() -> PyObject* {
    PyObject* const lists[4] = {p, m, v, g};
    Lists x;
    if (!x.look(lists, 4, device, 3, false)) return nullptr;
    if (!x.same || x.meet || !x.usual(0, true) || !x.usual(1, true) || !x.usual(2, true) || !x.usual(3, false) || x.n == 0)
      Py_RETURN_NONE;
    Buffers b(device, bytes);
    const auto at = [&](size_t l) { return reinterpret_cast<const long long*>(x.ptrs[l].data()); };
    const int status = reinterpret_cast<decltype(&kb_adam_step)>(fn)(
        at(0), at(3), at(1), at(2), reinterpret_cast<const long long*>(x.counts.data()), x.dtypes[3].data(), (int)x.n, lr,
        b1, b2, eps, wd, c1, c2, kind, max_norm, b.norm.data_ptr<float>(), b.ws.data_ptr(), bytes, (void*)stream);
    if (status == 0) x.written.mark();
    return Py_BuildValue("(iN)", status, wrap(b.norm));
  });
}

// fit_buffers(like, bytes) -> (a scalar for the norm, a workspace of so many bytes) on like's device.
PyObject* fit_buffers(PyObject*, PyObject* args) {
  PyObject* like_o;
  long long bytes;
  if (!PyArg_ParseTuple(args, "OL", &like_o, &bytes)) return nullptr;
  return guarded([&]() -> PyObject* {
    if (!THPVariable_Check(like_o)) {
      PyErr_SetString(PyExc_TypeError, "expected a tensor");
      return nullptr;
    }
    const auto on = at::TensorOptions().device(THPVariable_Unpack(like_o).device());
    return Py_BuildValue("(NN)", wrap(at::empty({}, on.dtype(at::kFloat))),
                         wrap(at::empty({(int64_t)bytes}, on.dtype(at::kByte))));
  });
}

PyMethodDef kMethods[] = {
    {"gather", gather, METH_VARARGS, nullptr},
    {"overlap", overlap, METH_VARARGS, nullptr},
    {"written", written, METH_O, nullptr},
    {"score_outputs", score_outputs, METH_VARARGS, nullptr},
    {"score_rows", score_rows, METH_VARARGS, nullptr},
    {"score_rows_backward", score_rows_backward, METH_VARARGS, nullptr},
    {"clip", clip, METH_VARARGS, nullptr},
    {"adam", adam, METH_VARARGS, nullptr},
    {"fit_buffers", fit_buffers, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_kb_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kb_host(void) {
  PyObject* m = PyModule_Create(&kModule);
  if (m && PyModule_AddStringConstant(m, "target", KB_TARGET) != 0) {  // the Python and torch it is built for
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
