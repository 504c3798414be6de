// The ordinary call of the operators of moe_rd.sorting and moe_rd.experts without Python in between: dense, aligned
// tensors of the right types on the current device, no gradient, no tangent.  Each function looks at its arguments, calls the C
// entry on the current stream and returns
//   True           done, results are in `out`;
//   the results    done, where `out` was None;
//   False          anything else: the Python function that called goes its own way, which knows every other case and the
//                  reason of every refusal.  A C entry that reports an error comes out here too (its outputs are then
//                  written again, or refused with their reason).
// A call with `out` costs the host 2.4 to 3.2 us this way and 8.6 to 11.7 the Python way; the launch is 2.3 of both.  The
// smallest calls take the GPU 3 to 6 us, so that a decode step pays for the host in every one of them.
//
// The C entries come as addresses from the Python side, which has loaded the library (bind).
//
// The objects of torch and Python are read in place, so a module fits the versions that it was compiled for and no others:
// it carries their names (BUILT_FOR), and is loaded only where they are the running ones.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>

#include "moe_rd.h"

namespace {

using at::Tensor;

// The C entries, in the order in which bind takes them.
struct Entries {
  decltype(&moe_rd_sort_workspace_bytes) sort_workspace_bytes;
  decltype(&moe_rd_sort_tokens) sort_tokens;
  decltype(&moe_rd_unsort_tokens) unsort_tokens;
  decltype(&moe_rd_unsort_tokens_backward) unsort_tokens_backward;
  decltype(&moe_rd_routing_weights) routing_weights;
  decltype(&moe_rd_routing_weights_backward) routing_weights_backward;
  decltype(&moe_rd_expert_matvec_w4) expert_matvec_w4;
} g_entry = {};
constexpr Py_ssize_t kEntries = sizeof(Entries) / sizeof(void*);

const Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

// Dense, on the device, of the type, in memory as it is (not the imaginary part of a conjugate, whose sign is still to change).
bool packed(const Tensor* t, int device, at::ScalarType type) {
  return t != nullptr && t->defined() && t->is_cuda() && t->get_device() == device && t->layout() == at::kStrided &&
         t->unsafeGetTensorImpl()->has_storage() && t->is_contiguous() &&
         t->scalar_type() == type && !t->is_neg();
}

// The same with an address that is a multiple of 16: what the kernels read in vectors.
bool dense(const Tensor* t, int device, at::ScalarType type) {
  return packed(t, device, type) && (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15) == 0;
}

// Carries a tangent of forward mode that an operation would have to carry on.
bool dual(const Tensor* t) { return t != nullptr && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined(); }

bool no_grad(const Tensor* t) { return t == nullptr || ((!t->requires_grad() || !c10::GradMode::is_enabled()) && !dual(t)); }

struct Span {
  uintptr_t lo, hi;
  explicit Span(const Tensor* t)
      : lo(t != nullptr ? reinterpret_cast<uintptr_t>(t->const_data_ptr()) : 0), hi(t != nullptr ? lo + t->nbytes() : 0) {}
  bool meets(const Span& o) const { return lo < o.hi && o.lo < hi; }
};

// A buffer of the caller: of this shape and type, written by nobody's graph, apart from the inputs.
bool writable(const Tensor* t, int device, at::ScalarType type, at::IntArrayRef shape, std::initializer_list<const Tensor*> inputs,
              bool aligned = true) {
  if (t == nullptr || !t->defined() || !t->is_cuda() || t->get_device() != device || t->layout() != at::kStrided ||
      !t->unsafeGetTensorImpl()->has_storage() || t->scalar_type() != type || t->sizes() != shape || !t->is_contiguous() ||
      t->requires_grad() || t->is_neg() ||
      (aligned && (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15) != 0))
    return false;
  const Span mine(t);
  for (const Tensor* i : inputs)
    if (i != nullptr && mine.meets(Span(i))) return false;
  return true;
}

void written(const Tensor* t) {
  if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// Addresses, null for no tensor.
template <typename T = void>
const T* in(const Tensor* t) {
  return t != nullptr ? static_cast<const T*>(t->const_data_ptr()) : nullptr;
}
template <typename T = void>
T* to(const Tensor* t) {
  return t != nullptr ? static_cast<T*>(t->mutable_data_ptr()) : nullptr;
}

bool number(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool real(PyObject* o, double* v) {
  if (PyFloat_CheckExact(o)) {
    *v = PyFloat_AS_DOUBLE(o);
    return true;
  }
  int64_t i;
  if (!number(o, &i)) return false;
  *v = (double)i;
  return true;
}

// Row types of the C entries; -1: another type.
int row_type(const Tensor* t) {
  switch (t->scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: return -1;
  }
}

int here(const Tensor* t) {  // the tensor's device where that is the current one, else -1
  if (t == nullptr || !t->defined() || !t->is_cuda()) return -1;
  const int device = t->get_device();
  return device == c10::cuda::current_device() ? device : -1;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

PyObject* refuse() { Py_RETURN_FALSE; }

// Allocations and launches go on without the interpreter's lock, as torch's own do: the allocator's lock is never waited
// for while holding it.
struct WithoutLock {
  PyThreadState* const state = PyEval_SaveThread();
  ~WithoutLock() { PyEval_RestoreThread(state); }
};

// C++ exceptions (an allocation that fails): the Python way meets the same and raises it.
template <typename Body>
PyObject* guarded(Body body) {
  try {
    return body();
  } catch (...) {
    return refuse();
  }
}

// The tensors as a tuple, None for an undefined one.
PyObject* results(const Tensor* made, Py_ssize_t n) {
  PyObject* r = PyTuple_New(n);
  for (Py_ssize_t i = 0; r != nullptr && i < n; ++i) {
    PyObject* o = made[i].defined() ? THPVariable_Wrap(made[i]) : Py_NewRef(Py_None);
    if (o == nullptr)
      Py_CLEAR(r);
    else
      PyTuple_SET_ITEM(r, i, o);
  }
  return r;
}

// sort_tokens(x, expert_ids, num_experts, capacity, out: tuple of 5 or None)
PyObject* sort_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const Tensor *x = n == 5 ? tensor(a[0]) : nullptr, *ids = n == 5 ? tensor(a[1]) : nullptr;
    const int device = here(x);
    int64_t E, capacity;
    if (device < 0 || !number(a[2], &E) || !number(a[3], &capacity) || !dense(x, device, x->scalar_type()) || !packed(ids, device, at::kInt) ||
        !no_grad(x))
      return refuse();
    const int type = row_type(x);
    if (type < 0 || x->dim() != 2 || ids->dim() != 2 || E < 1 || E > 256 || capacity < 0) return refuse();
    const int64_t T = ids->size(0), K = ids->size(1), H = x->size(1);
    if (x->size(0) != T || K < 1 || K > 32 || H < 1 || H > (1 << 20) || H * x->element_size() % 16 != 0) return refuse();
    const int64_t all = T * K, R = capacity > 0 && capacity < all / E + 1 && E * capacity < all ? E * capacity : all;
    Tensor made[5];
    const Tensor* out[5];
    const bool given = a[4] != Py_None;
    if (given) {
      if (!PyTuple_Check(a[4]) || PyTuple_GET_SIZE(a[4]) != 5) return refuse();
      for (int i = 0; i < 5; ++i) out[i] = tensor(PyTuple_GET_ITEM(a[4], i));
      if (!writable(out[0], device, x->scalar_type(), {R, H}, {x, ids}) || !writable(out[1], device, at::kInt, {E + 1}, {x, ids}, false) ||
          !writable(out[2], device, at::kInt, {T, K}, {x, ids}, false) || !writable(out[3], device, at::kInt, {R}, {x, ids}, false) ||
          !writable(out[4], device, at::kInt, {E}, {x, ids}, false))
        return refuse();
    }
    int code;
    {
      WithoutLock lock;
      if (!given) {
        // parts of one buffer would share its version: a change of the counts would look like one of the places, which
        // a graph may have saved
        made[0] = at::empty({R, H}, x->options());
        made[1] = at::empty({E + 1}, ids->options());
        made[2] = at::empty({T, K}, ids->options());
        made[3] = at::empty({R}, ids->options());
        made[4] = at::empty({E}, ids->options());
        for (int i = 0; i < 5; ++i) out[i] = &made[i];
      }
      size_t bytes = 0;
      code = g_entry.sort_workspace_bytes(T, (int32_t)H, (int32_t)E, (int32_t)K, type, &bytes);
      if (code == 0) {
        Tensor workspace;
        if (bytes > 0) workspace = at::empty({(int64_t)bytes}, x->options().dtype(at::kByte));
        code = g_entry.sort_tokens(T, (int32_t)H, (int32_t)E, (int32_t)K, type, capacity, R, in(x), in<int32_t>(ids), to(out[0]), to<int32_t>(out[1]),
                                   to<int32_t>(out[2]), to<int32_t>(out[3]), to<int32_t>(out[4]), bytes > 0 ? to(&workspace) : nullptr, bytes,
                                   stream_of(device));
      }
    }
    if (code != 0) return refuse();
    if (given) {
      for (const Tensor* t : out) written(t);
      Py_RETURN_TRUE;
    }
    return results(made, 5);
  });
}

// [E+1] offsets, or None for none.
bool offsets_of(PyObject* o, int device, const Tensor** t) {
  *t = nullptr;
  if (o == Py_None) return true;
  *t = tensor(o);
  return *t != nullptr && (*t)->defined() && (*t)->is_cuda() && (*t)->get_device() == device && (*t)->layout() == at::kStrided &&
         (*t)->unsafeGetTensorImpl()->has_storage() && (*t)->scalar_type() == at::kInt && (*t)->dim() == 1 && (*t)->numel() > 0 && (*t)->is_contiguous();
}

// What unsort_tokens and its gradient share: rows of one type, places, weights or None, a [T,H] tensor or None.
struct Way {
  const Tensor *y, *inv, *w, *other;
  int device, type;
  int64_t T, K, H, R;
  bool look(PyObject* y_, PyObject* inv_, PyObject* w_, PyObject* other_) {
    y = tensor(y_);
    inv = tensor(inv_);
    w = w_ == Py_None ? nullptr : tensor(w_);
    other = other_ == Py_None ? nullptr : tensor(other_);
    device = here(y);
    if (device < 0 || !dense(y, device, y->scalar_type()) || !packed(inv, device, at::kInt) || (w_ != Py_None && !packed(w, device, at::kFloat)) ||
        (other_ != Py_None && !dense(other, device, y->scalar_type())) || !no_grad(y) || !no_grad(w) || !no_grad(other))
      return false;
    type = row_type(y);
    if (type < 0 || y->dim() != 2 || inv->dim() != 2) return false;
    T = inv->size(0);
    K = inv->size(1);
    R = y->size(0);
    H = y->size(1);
    if (K < 1 || K > 32 || H < 1 || H > (1 << 20) || H * y->element_size() % 16 != 0) return false;
    if (w != nullptr && w->sizes() != inv->sizes()) return false;
    return other == nullptr || other->sizes() == at::IntArrayRef({T, H});
  }
};

// unsort_tokens(y, inverse_perm, weights, shared, offsets, out); the offsets are looked at and have no part in it
PyObject* unsort_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Way s;
    const Tensor* offsets;
    if (n != 6 || !s.look(a[0], a[1], a[2], a[3]) || !offsets_of(a[4], s.device, &offsets)) return refuse();
    Tensor made;
    const Tensor* out = &made;
    const bool given = a[5] != Py_None;
    if (given && !writable(out = tensor(a[5]), s.device, s.y->scalar_type(), {s.T, s.H}, {s.y, s.inv, s.w, s.other})) return refuse();
    int code;
    {
      WithoutLock lock;
      if (!given) made = at::empty({s.T, s.H}, s.y->options());
      code = g_entry.unsort_tokens(s.T, (int32_t)s.H, (int32_t)s.K, s.type, in(s.y), s.R, in<int32_t>(s.inv), in<float>(s.w), in(s.other), to(out),
                                   stream_of(s.device));
    }
    if (code != 0) return refuse();
    if (!given) return THPVariable_Wrap(made);
    written(out);
    Py_RETURN_TRUE;
  });
}

// unsort_tokens_backward(grad_out, y, inverse_perm, weights, offsets, need_rows, need_weights, out: (rows, weights) or None)
PyObject* unsort_tokens_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Way s;
    if (n != 8 || !s.look(a[1], a[2], a[3], a[0]) || s.other == nullptr) return refuse();
    const Tensor* offsets;
    if (!offsets_of(a[4], s.device, &offsets)) return refuse();
    const bool rows = a[5] == Py_True, weights = a[6] == Py_True;
    if ((!rows && a[5] != Py_False) || (!weights && a[6] != Py_False) || !(rows || weights)) return refuse();
    Tensor made[2];
    const Tensor* out[2] = {rows ? &made[0] : nullptr, weights ? &made[1] : nullptr};
    const bool given = a[7] != Py_None;
    if (given) {
      if (!PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 2) return refuse();
      for (int i = 0; i < 2; ++i) {
        PyObject* o = PyTuple_GET_ITEM(a[7], i);
        if ((o != Py_None) != (i == 0 ? rows : weights)) return refuse();
        if (o != Py_None) out[i] = tensor(o);
      }
      if ((rows && !writable(out[0], s.device, s.y->scalar_type(), {s.R, s.H}, {s.y, s.inv, s.w, s.other, offsets})) ||
          (weights && !writable(out[1], s.device, at::kFloat, {s.T, s.K}, {s.y, s.inv, s.w, s.other, offsets}, false)))
        return refuse();
    }
    const int32_t* end = offsets == nullptr ? nullptr : in<int32_t>(offsets) + offsets->numel() - 1;
    int code;
    {
      WithoutLock lock;
      if (!given && rows) made[0] = at::empty({s.R, s.H}, s.y->options());
      if (!given && weights) made[1] = at::empty({s.T, s.K}, s.y->options().dtype(at::kFloat));
      code = g_entry.unsort_tokens_backward(s.T, (int32_t)s.H, (int32_t)s.K, s.type, in(s.other), weights ? in(s.y) : nullptr, s.R, in<int32_t>(s.inv),
                                            in<float>(s.w), end, to(out[0]), to<float>(out[1]), stream_of(s.device));
    }
    if (code != 0) return refuse();
    if (given) {
      written(out[0]);
      written(out[1]);
      Py_RETURN_TRUE;
    }
    return results(made, 2);
  });
}

// routing_weights(grad_weights or None, logits, expert_ids, bias or None, use of the bias (0 none, 1 logits, 2 scores), score_fn, renorm,
//                 routed_scale, norm_min, out)
PyObject* routing_weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 10) return refuse();
    const Tensor *g = a[0] == Py_None ? nullptr : tensor(a[0]), *z = tensor(a[1]), *ids = tensor(a[2]), *b = a[3] == Py_None ? nullptr : tensor(a[3]);
    const int device = here(z);
    int64_t use, score_fn;
    double scale, least;
    if (device < 0 || !number(a[4], &use) || !number(a[5], &score_fn) || (a[6] != Py_True && a[6] != Py_False) || !real(a[7], &scale) ||
        !real(a[8], &least) || !packed(z, device, at::kFloat) || !packed(ids, device, at::kInt) || (a[0] != Py_None && !packed(g, device, at::kFloat)) ||
        (a[3] != Py_None && !packed(b, device, at::kFloat)) || !no_grad(z) || !no_grad(b) || dual(g))
      return refuse();
    if (z->dim() != 2 || ids->dim() != 2 || z->size(0) != ids->size(0) || z->size(1) < 1 || z->size(1) > 256 ||
        ids->size(1) < 1 || ids->size(1) > 32 || (b != nullptr && b->numel() != z->size(1)) ||
        (g != nullptr && g->sizes() != ids->sizes()))
      return refuse();
    const int64_t T = z->size(0), E = z->size(1), K = ids->size(1);
    const at::IntArrayRef shape = g != nullptr ? z->sizes() : ids->sizes();
    Tensor made;
    const Tensor* out = &made;
    const bool given = a[9] != Py_None;
    if (given && !writable(out = tensor(a[9]), device, at::kFloat, shape, {z, ids, b, g}, false)) return refuse();
    const float *lb = use == 1 ? in<float>(b) : nullptr, *sb = use == 2 ? in<float>(b) : nullptr;
    const int renorm = a[6] == Py_True;
    int code;
    {
      WithoutLock lock;
      if (!given) made = at::empty(shape, z->options());
      code = g == nullptr ? g_entry.routing_weights(T, (int32_t)E, (int32_t)K, (int32_t)score_fn, renorm, (float)scale, (float)least, in<float>(z),
                                                    in<int32_t>(ids), lb, sb, to<float>(out), stream_of(device))
                          : g_entry.routing_weights_backward(T, (int32_t)E, (int32_t)K, (int32_t)score_fn, renorm, (float)scale, (float)least,
                                                             in<float>(z), in<int32_t>(ids), lb, sb, in<float>(g), to<float>(out), stream_of(device));
    }
    if (code != 0) return refuse();
    if (!given) return THPVariable_Wrap(made);
    written(out);
    Py_RETURN_TRUE;
  });
}

// expert_matvec_w4(x, weights: (packed, scales, zeros or None, N, K, group), offsets or None, out)
PyObject* expert_matvec_w4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 4 || !PyTuple_Check(a[1]) || PyTuple_GET_SIZE(a[1]) != 6) return refuse();
    PyObject* zo = PyTuple_GET_ITEM(a[1], 2);
    const Tensor *x = tensor(a[0]), *w = tensor(PyTuple_GET_ITEM(a[1], 0)), *sc = tensor(PyTuple_GET_ITEM(a[1], 1)), 
               *z = zo == Py_None ? nullptr : tensor(zo), *offsets = nullptr;
    const int device = here(x);
    int64_t N, K, group;
    if (device < 0 || !number(PyTuple_GET_ITEM(a[1], 3), &N) || !number(PyTuple_GET_ITEM(a[1], 4), &K) || !number(PyTuple_GET_ITEM(a[1], 5), &group) ||
        !dense(x, device, x->scalar_type()) || !dense(w, device, at::kByte) || !dense(sc, device, x->scalar_type()) ||
        (zo != Py_None && !dense(z, device, at::kByte)) ||
        !no_grad(x) || !no_grad(sc))
      return refuse();
    const int type = row_type(x);
    if (type < 0 || type > 1 || x->dim() != 2 || x->size(1) != K || w->dim() != 4 || N < 1 || N > (1 << 24) || K < 32 || K > (1 << 20) || group < 32 ||
        K % group != 0)
      return refuse();
    const int64_t R = x->size(0), E = w->size(0), B = (N + 31) / 32, G = K / group;
    if (w->sizes() != at::IntArrayRef({E, B, (K + 127) / 128, 2048}) || sc->sizes() != at::IntArrayRef({E, B, G, 8, 4}) ||
        (z != nullptr && z->sizes() != at::IntArrayRef({E, B, G, 8, 2})))
      return refuse();
    if (!offsets_of(a[2], device, &offsets) || (offsets == nullptr ? E != 1 : offsets->numel() != E + 1)) return refuse();
    Tensor made;
    const Tensor* out = &made;
    const bool given = a[3] != Py_None;
    if (given && !writable(out = tensor(a[3]), device, x->scalar_type(), {R, N}, {x, w, sc, z, offsets}, false)) return refuse();
    int code;
    {
      WithoutLock lock;
      if (!given) made = at::empty({R, N}, x->options());
      code = g_entry.expert_matvec_w4(R, (int32_t)N, (int32_t)K, (int32_t)E, (int32_t)group, type, in(x), in(w), in(sc), in<uint16_t>(z),
                                      in<int32_t>(offsets), to(out), stream_of(device));
    }
    if (code != 0) return refuse();
    if (!given) return THPVariable_Wrap(made);
    written(out);
    Py_RETURN_TRUE;
  });
}

// bind(addresses of the C entries, in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != kEntries) {
    PyErr_SetString(PyExc_TypeError, "bind: wrong number of entries");
    return nullptr;
  }
  void* entry[kEntries];
  for (Py_ssize_t i = 0; i < n; ++i) {
    entry[i] = PyLong_AsVoidPtr(a[i]);
    if (entry[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null entry");
      return nullptr;
    }
  }
  std::memcpy(&g_entry, entry, sizeof g_entry);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FAST(bind),
                           FAST(sort_tokens),
                           FAST(unsort_tokens),
                           FAST(unsort_tokens_backward),
                           FAST(routing_weights),
                           FAST(expert_matvec_w4),
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall(void) {
  PyObject* m = PyModule_Create(&g_module);
  if (m != nullptr && PyModule_AddStringConstant(m, "BUILT_FOR", MOE_RD_BUILT_FOR) != 0) Py_CLEAR(m);
  return m;
}
