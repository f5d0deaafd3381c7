// The host side of the router's hot operators for plain calls, in native code.
//
// An eager step enqueues three launches whose kernels take a few microseconds each at decode
// sizes, and the Python around them (argument checks, allocation, views, a foreign call with
// twenty converted arguments) took 12 to 19 us per operator, more than the GPU did.  These
// functions do the same for the calls that programs make all the time - contiguous tensors of
// the right types on the current device, sizes known - and return None for any other
// call, before anything has been enqueued: the Python operator then takes it and does the
// checking and the explaining.  They call the same entry points of the C library, and like the
// foreign calls they stand for they let other Python threads run meanwhile: an allocation may
// synchronise, a launch waits while the queue of the stream is full.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_cpp_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../include/brt_b200.h"

namespace {

PyObject* g_dense;  // attribute name on index tensors

// A plain torch.Tensor (no subclass, no functional wrapper) with memory on the GPU and without a
// forward-mode derivative.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || !t.has_storage()) return nullptr;
  if (t.unsafeGetTensorImpl()->key_set().has_any(
          c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize,
                               c10::DispatchKey::Negative, c10::DispatchKey::Conjugate})))
    return nullptr;
  if (t._fw_grad(0).defined()) return nullptr;
  return &t;
}
bool modes_active() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() ||
         at::impl::torch_function_mode_enabled();
}
bool int32c(const at::Tensor* t, int64_t dims) {
  return t != nullptr && t->scalar_type() == at::kInt && t->dim() == dims && t->is_contiguous();
}
int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return BRT_F32;
    case at::kHalf: return BRT_F16;
    case at::kBFloat16: return BRT_BF16;
    default: return -1;
  }
}
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, c10::Device device) {
  return at::detail::empty_cuda(sizes, type, device, std::nullopt);
}

// The device all tensors of a call must be on, when it is the current one; its stream.
struct Place {
  c10::Device device;
  c10::cuda::CUDAStream stream;
  static bool of(const at::Tensor& t) { return t.get_device() == c10::cuda::current_device(); }
  explicit Place(const at::Tensor& t)
      : device(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device())) {}
  void* handle() const { return stream.stream(); }
};
bool same_device(const at::Tensor& a, const at::Tensor* b) {
  return b == nullptr || a.get_device() == b->get_device();
}

// Other Python threads run while this lives.  Everything that touches a Python object comes before
// or after; what is made inside (tensors that no Python object wraps yet) needs no lock.
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
// The addresses of a call's tensors, and the memory behind them kept until the call has been
// enqueued: meanwhile another thread may drop a tensor or give it other memory.
struct Memory {
  c10::SmallVector<c10::Storage, 8> held;
  void* of(const at::Tensor* t) {
    if (t == nullptr) return nullptr;
    held.push_back(t->storage());
    return t->data_ptr();
  }
  int32_t* ints(const at::Tensor* t) { return static_cast<int32_t*>(of(t)); }
};

// The note of an index operator on the tensor it returns, see _C/router.py.
bool mark(PyObject* indices, const at::Tensor& counts) {
  PyObject* c = THPVariable_Wrap(counts);
  const bool ok = c != nullptr && PyObject_SetAttr(indices, g_dense, c) == 0;
  Py_XDECREF(c);
  return ok;
}
// A new reference or null (no error set) when there is no such attribute.
PyObject* attribute(PyObject* o, PyObject* name) {
  PyObject* v = PyObject_GetAttr(o, name);
  if (v == nullptr) PyErr_Clear();
  return v;
}

// The dense counts noted on `indices`, or null.
const int32_t* dense_counts(PyObject* indices, int64_t paths, Memory& memory) {
  PyObject* note = attribute(indices, g_dense);
  if (note == nullptr) return nullptr;
  const at::Tensor* t = plain(note);
  const bool ok = int32c(t, 1) && t->numel() == paths &&
                  same_device(THPVariable_Unpack(indices), t);
  const int32_t* const p = ok ? memory.ints(t) : nullptr;
  Py_DECREF(note);
  return p;
}

struct Caps {
  const int32_t* ptr = nullptr;
  int num = 0;
  bool ok = true;
  Caps(PyObject* o, const at::Tensor& like, Memory& memory) {
    if (o == Py_None) return;
    const at::Tensor* t = plain(o);
    ok = int32c(t, 1) && same_device(like, t);
    if (!ok) return;
    ptr = memory.ints(t);
    num = (int)t->numel();
  }
};

// 0, 1, or -1 for an object without a truth value (no error is left set).
int truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) PyErr_Clear();
  return v;
}

// Errors keep the kind that torch gives them in Python: torch.OutOfMemoryError above all.
template <typename F>
PyObject* guarded(F&& body) {
  try {
    PyObject* r = body();
    if (r != nullptr || PyErr_Occurred()) return r;
    Py_RETURN_NONE;
  } catch (const std::exception&) {
    torch::translate_exception_to_python(std::current_exception());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error in a router operator");
  }
  return nullptr;
}
void* data_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// scan(hot_mask, prefix | None, threshold | None, caps | None, capacity_padding, path_wise,
//      with_mask): seat indices; with prefix and threshold of the mask throttled on the way.
// -> (indices, loads) or (indices, loads, throttled mask | None)
PyObject* scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7 || modes_active() || brt_index_status() != BRT_OK) return nullptr;
    const at::Tensor* mask = plain(a[0]);
    if (!int32c(mask, 2) || mask->numel() == 0 || !Place::of(*mask)) return nullptr;
    const bool throttle = a[1] != Py_None;
    const at::Tensor *prefix = nullptr, *threshold = nullptr;
    const int64_t T = mask->size(0), E = mask->size(1);
    if (throttle) {
      prefix = plain(a[1]);
      threshold = plain(a[2]);
      if (!int32c(prefix, 1) || !int32c(threshold, 1) || prefix->numel() != E ||
          threshold->numel() != E || !same_device(*mask, prefix) ||
          !same_device(*mask, threshold))
        return nullptr;
    }
    Memory memory;
    const Caps caps(a[3], *mask, memory);
    if (!caps.ok) return nullptr;
    const int cpad = truth(a[4]), pwise = truth(a[5]), with_mask = truth(a[6]);
    if (cpad < 0 || pwise < 0 || with_mask < 0) return nullptr;
    if (throttle && E % 4 != 0) return nullptr;  // takes two launches
    const Place p(*mask);
    const int32_t* const m = memory.ints(mask);
    int32_t* const before = memory.ints(prefix);
    const int32_t* const limit = memory.ints(threshold);
    at::Tensor indices, loads, counts, throttled;
    int rc;
    {
      const Unlocked unlocked;
      indices = empty({T, E}, at::kInt, p.device);
      const at::Tensor both = empty({2, E}, at::kInt, p.device);
      loads = both.select(0, 0);
      counts = both.select(0, 1);
      if (with_mask) throttled = empty({T, E}, at::kInt, p.device);
      const int64_t bytes = (int64_t)brt_index_scratch_bytes(T, (int)E);
      const at::Tensor scratch = empty({bytes}, at::kByte, p.device);
      const auto out = static_cast<int32_t*>(indices.data_ptr());
      const auto l = static_cast<int32_t*>(loads.data_ptr());
      const auto c = static_cast<int32_t*>(counts.data_ptr());
      rc = throttle ? brt_throttle_and_generate_indices(
                          m, out, l, c, before, limit,
                          static_cast<int32_t*>(data_or_null(throttled)), T, (int)E, caps.ptr,
                          caps.num, cpad, pwise, scratch.data_ptr(), (size_t)bytes, p.handle())
                    : brt_generate_indices_and_loads(m, out, l, c, T, (int)E, caps.ptr, caps.num,
                                                     cpad, pwise, 0, scratch.data_ptr(),
                                                     (size_t)bytes, p.handle());
    }
    if (rc != BRT_OK) return nullptr;  // nothing was enqueued: the operator says why
    PyObject* i = THPVariable_Wrap(indices);
    if (i == nullptr || !mark(i, counts)) {
      Py_XDECREF(i);
      return nullptr;
    }
    if (!throttle) return Py_BuildValue("(NN)", i, THPVariable_Wrap(loads));
    if (with_mask)
      return Py_BuildValue("(NNN)", i, THPVariable_Wrap(loads), THPVariable_Wrap(throttled));
    return Py_BuildValue("(NNO)", i, THPVariable_Wrap(loads), Py_None);
  });
}

// route_scores(score, decision, top_k, threshold, residual_path, output, caps | None,
//              capacity_padding, path_wise, prefix | None, throttle_capacity | None, with_gates,
//              with_mask) -> (out, loads, gates | None, mask | None)
PyObject* route_scores(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 13 || modes_active() || brt_index_status() != BRT_OK) return nullptr;
    const at::Tensor* score = plain(a[0]);
    if (score == nullptr || score->scalar_type() != at::kFloat || score->dim() != 2 ||
        !score->is_contiguous() || score->numel() == 0 || !Place::of(*score))
      return nullptr;
    const int64_t T = score->size(0), E = score->size(1);
    if (E > 256 || E % 4 != 0) return nullptr;
    const long decision = PyLong_AsLong(a[1]), top_k = PyLong_AsLong(a[2]);
    const double threshold = PyFloat_AsDouble(a[3]);
    const long residual = PyLong_AsLong(a[4]), output = PyLong_AsLong(a[5]);
    if (PyErr_Occurred()) {  // numbers of other kinds: the operator converts them
      PyErr_Clear();
      return nullptr;
    }
    if (top_k != (int)top_k || residual != (int)residual) return nullptr;
    Memory memory;
    const Caps caps(a[6], *score, memory);
    const int cpad = truth(a[7]), pwise = truth(a[8]);
    const int with_gates = truth(a[11]), with_mask = truth(a[12]);
    if (cpad < 0 || pwise < 0 || with_gates < 0 || with_mask < 0) return nullptr;
    if (!caps.ok || (cpad != 0 && caps.num < 1)) return nullptr;
    const bool seats =
        output == BRT_ROUTE_SEAT_INDICES || output == BRT_ROUTE_THROTTLED_SEAT_INDICES;
    const bool throttles =
        output == BRT_ROUTE_THROTTLED_MASK || output == BRT_ROUTE_THROTTLED_SEAT_INDICES;
    const at::Tensor *prefix = nullptr, *limit = nullptr;
    if (throttles) {
      prefix = plain(a[9]);
      limit = plain(a[10]);
      if (!int32c(prefix, 1) || !int32c(limit, 1) || prefix->numel() != E ||
          limit->numel() != E || !same_device(*score, prefix) || !same_device(*score, limit))
        return nullptr;
    }
    if (with_mask && !seats) return nullptr;
    const Place p(*score);
    const auto s = static_cast<const float*>(memory.of(score));
    int32_t* const before = memory.ints(prefix);
    const int32_t* const room = memory.ints(limit);
    at::Tensor out, loads, counts, gates, mask;
    int rc;
    {
      const Unlocked unlocked;
      out = empty({T, E}, at::kInt, p.device);
      const at::Tensor both = empty({2, E}, at::kInt, p.device);
      loads = both.select(0, 0);
      counts = both.select(0, 1);
      if (with_gates) gates = empty({T, E}, at::kFloat, p.device);
      if (with_mask) mask = empty({T, E}, at::kInt, p.device);
      const int64_t bytes = (int64_t)brt_index_scratch_bytes(T, (int)E);
      const at::Tensor scratch = empty({bytes}, at::kByte, p.device);
      rc = brt_route_scores(
          s, T, (int)E, (int)decision, (int)top_k, (float)threshold, (int)residual, (int)output,
          static_cast<int32_t*>(out.data_ptr()), static_cast<int32_t*>(loads.data_ptr()),
          seats ? static_cast<int32_t*>(counts.data_ptr()) : nullptr, caps.ptr, caps.num, cpad,
          pwise, before, room, static_cast<float*>(data_or_null(gates)),
          static_cast<int32_t*>(data_or_null(mask)), scratch.data_ptr(), (size_t)bytes,
          p.handle());
    }
    if (rc != BRT_OK) return nullptr;
    PyObject* o = THPVariable_Wrap(out);
    if (o == nullptr || (seats && !mark(o, counts))) {
      Py_XDECREF(o);
      return nullptr;
    }
    PyObject* g = with_gates ? THPVariable_Wrap(gates) : Py_NewRef(Py_None);
    PyObject* m = with_mask ? THPVariable_Wrap(mask) : Py_NewRef(Py_None);
    return Py_BuildValue("(NNNN)", o, THPVariable_Wrap(loads), g, m);
  });
}

// dispatch(in_data, route_indices, loads, gates | None, max_path_load, total_rows): 1-D routing,
// seat indices straight out of an index operator, no tags -> the rows
PyObject* dispatch(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || modes_active()) return nullptr;
    const at::Tensor *x = plain(a[0]), *indices = plain(a[1]), *loads = plain(a[2]);
    if (x == nullptr || x->dim() < 1 || !x->is_contiguous() || x->numel() == 0 ||
        !Place::of(*x) || !int32c(indices, 2) || !int32c(loads, 1) ||
        !same_device(*x, indices) || !same_device(*x, loads))
      return nullptr;
    const int dtype = dtype_of(*x);
    const int64_t T = x->size(0), E = indices->size(1);
    if (dtype < 0 || indices->size(0) != T || loads->numel() != E || E < 1 || E > 2048)
      return nullptr;
    const int64_t cell = x->numel() / T;
    if (dtype == BRT_F16 && cell % 2 != 0) return nullptr;
    const at::Tensor* gates = nullptr;
    if (a[3] != Py_None) {
      gates = plain(a[3]);
      if (gates == nullptr || gates->scalar_type() != x->scalar_type() ||
          !gates->is_contiguous() || gates->numel() != T * E || !same_device(*x, gates))
        return nullptr;
    }
    const long long mpl = PyLong_AsLongLong(a[4]), total = PyLong_AsLongLong(a[5]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return nullptr;
    }
    if (mpl < 0 || mpl > 0x7fffffffLL || total < 0) return nullptr;
    Memory memory;
    const int32_t* counts = dense_counts(a[1], E, memory);
    if (counts == nullptr) return nullptr;
    const Place p(*x);
    c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
    shape[0] = total;
    const auto type = x->scalar_type();
    const void* const src = memory.of(x);
    const void* const g = memory.of(gates);
    const int32_t* const at_rows = memory.ints(indices);
    const int32_t* const l = memory.ints(loads);
    at::Tensor out;
    int rc;
    {
      const Unlocked unlocked;
      out = empty(shape, type, p.device);
      rc = brt_dispatch_with_indices_and_loads(src, out.data_ptr(), g, at_rows, l, nullptr, nullptr,
                                               T, cell, (int)E, (int)mpl, total, 1, 0, dtype,
                                               counts, nullptr, 0, p.handle());
    }
    if (rc != BRT_OK) return nullptr;
    return THPVariable_Wrap(out);
  });
}

// combine(in_data, route_indices, loads, gates | None, out_data | None, max_path_padding): seat
// indices, at least two cells -> the cells (out_data itself when given)
PyObject* combine(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || modes_active()) return nullptr;
    const at::Tensor *x = plain(a[0]), *indices = plain(a[1]), *loads = plain(a[2]);
    if (x == nullptr || x->dim() < 1 || !x->is_contiguous() || x->numel() == 0 ||
        !Place::of(*x) || !int32c(indices, 2) || !int32c(loads, 1) ||
        !same_device(*x, indices) || !same_device(*x, loads))
      return nullptr;
    const int dtype = dtype_of(*x);
    const int64_t T = indices->size(0), E = indices->size(1);
    if (dtype < 0 || T < 2 || E < 1 || loads->numel() != E) return nullptr;
    const int64_t rows = x->size(0), cell = x->numel() / rows;
    const at::Tensor* gates = nullptr;
    int gate_type = 0;
    if (a[3] != Py_None) {
      gates = plain(a[3]);
      if (gates == nullptr || !gates->is_contiguous() || gates->numel() != T * E ||
          !same_device(*x, gates))
        return nullptr;
      gate_type = dtype_of(*gates);
      if (gate_type != BRT_F32 && gate_type != dtype) return nullptr;
    }
    const at::Tensor* residual = nullptr;
    if (a[4] != Py_None) {
      residual = plain(a[4]);
      if (residual == nullptr || !residual->is_contiguous() || residual->numel() != T * cell ||
          residual->scalar_type() != x->scalar_type() || !same_device(*x, residual))
        return nullptr;
    }
    const int padded = truth(a[5]);
    if (padded < 0) return nullptr;
    const int64_t mpl = padded ? rows / E : 0;
    if (mpl > 0x7fffffffLL) return nullptr;
    Memory memory;
    const Place p(*x);
    c10::SmallVector<int64_t, 6> shape(x->sizes().begin(), x->sizes().end());
    shape[0] = T;
    const auto type = x->scalar_type();
    const void* const src = memory.of(x);
    const void* const g = memory.of(gates);
    const int32_t* const at_rows = memory.ints(indices);
    const int32_t* const l = memory.ints(loads);
    void* dst = memory.of(residual);
    at::Tensor out;
    int rc;
    {
      const Unlocked unlocked;
      if (residual == nullptr) {
        out = empty(shape, type, p.device);
        dst = out.data_ptr();
      }
      rc = brt_combine_with_indices_and_loads(src, dst, g, at_rows, l, T, cell, (int)E,
                                              (int32_t)mpl, residual != nullptr, dtype, gate_type,
                                              p.handle());
    }
    if (rc != BRT_OK) return nullptr;
    return residual != nullptr ? Py_NewRef(a[4]) : THPVariable_Wrap(out);
  });
}

// ---- compact picks: rows sorted by path, back to cells, and their gradients -----------------

bool is_places(const at::Tensor* t) { return int32c(t, 2) && t->numel() > 0; }
bool wants_grad(const at::Tensor* t) {
  return t != nullptr && t->requires_grad() && c10::GradMode::is_enabled();
}
void done(int rc) { TORCH_CHECK(rc == BRT_OK, brt_last_error()); }
void* stream_of(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}
at::Tensor like_rows(const at::Tensor& t, int64_t rows) {
  c10::SmallVector<int64_t, 6> shape(t.sizes().begin(), t.sizes().end());
  shape[0] = rows;
  return empty(shape, t.scalar_type(), t.device());
}

// The kernels over contiguous tensors; `cells` and `rows` not empty.
at::Tensor sorted_rows(const at::Tensor& cells, const at::Tensor& places) {
  const int64_t T = places.size(0), k = places.size(1);
  at::Tensor rows = like_rows(cells, T * k);
  done(brt_sort_cells(cells.data_ptr(), static_cast<const int32_t*>(places.data_ptr()),
                      rows.data_ptr(), T, (int)k, cells.numel() / T, dtype_of(cells),
                      stream_of(cells)));
  return rows;
}
at::Tensor cells_of(const at::Tensor& rows, const at::Tensor& places, const at::Tensor& gates) {
  const int64_t T = places.size(0), k = places.size(1);
  at::Tensor cells = like_rows(rows, T);
  done(brt_unsort_cells(rows.data_ptr(), static_cast<const int32_t*>(places.data_ptr()),
                        data_or_null(gates), cells.data_ptr(), T, (int)k,
                        rows.numel() / (T * k), dtype_of(rows),
                        gates.defined() ? dtype_of(gates) : 0, stream_of(rows)));
  return cells;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// While a backward pass is captured into a CUDA graph: whether `node` hands its gradient to a leaf
// that belongs to another stream, because an eager graph made on that stream still holds the leaf's
// accumulator.  Autograd would then let that stream wait for the captured one, which breaks the
// capture and may end the process.
bool breaks_capture(torch::autograd::Node* node) {
  if (dynamic_cast<torch::autograd::AccumulateGrad*>(node) == nullptr) return false;
  const auto leaf_stream = node->stream();
  return leaf_stream.has_value() &&
         *leaf_stream != c10::cuda::getCurrentCUDAStream(leaf_stream->device_index()).unwrap();
}
constexpr const char* kBreaksCapture =
    "a backward pass is being captured while an eager autograd graph of the same leaves lives on "
    "another stream: release that graph, or capture on its stream";
void check_capture() {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (node == nullptr) return;
  for (const torch::autograd::Edge& edge : node->next_edges())
    TORCH_CHECK(!breaks_capture(edge.function.get()), kBreaksCapture);
}

// Neither have the gradients forward-mode derivatives.
void refuse_tangent(const at::Tensor& grad) {
  TORCH_CHECK(!grad._fw_grad(0).defined(),
              "the gradients of sorted rows have no forward-mode derivative");
}
// The gradients are not differentiable themselves: asking for that says so.
variable_list once(variable_list grads) {
  if (!c10::GradMode::is_enabled()) return grads;
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "the gradients of sorted rows cannot be differentiated", (int64_t)grads.size());
  for (at::Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  return (*error)(std::move(grads));
}

struct SortCells : public torch::autograd::Function<SortCells> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& cells,
                            const at::Tensor& places) {
    ctx->save_for_backward({places});
    return sorted_rows(cells, places);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    check_capture();
    refuse_tangent(grads[0]);
    return once({cells_of(grads[0].contiguous(), saved[0], {}), at::Tensor()});
  }
};

struct SumCells : public torch::autograd::Function<SumCells> {  // unsort without gates
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows,
                            const at::Tensor& places) {
    ctx->save_for_backward({places});
    return cells_of(rows, places, {});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    check_capture();
    refuse_tangent(grads[0]);
    return once({sorted_rows(grads[0].contiguous(), saved[0]), at::Tensor()});
  }
};

struct UnsortCells : public torch::autograd::Function<UnsortCells> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows,
                            const at::Tensor& places, const at::Tensor& gates) {
    // the rows are only read again for the gradient of the gates
    ctx->save_for_backward({gates.requires_grad() ? rows : at::Tensor(), places, gates});
    return cells_of(rows, places, gates);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &rows = saved[0], &places = saved[1], &gates = saved[2];
    const c10::cuda::CUDAGuard guard(places.device());
    check_capture();
    refuse_tangent(grads[0]);
    const at::Tensor grad = grads[0].contiguous();
    const int64_t T = places.size(0), k = places.size(1);
    at::Tensor row_grads, gate_grads;
    if (ctx->needs_input_grad(0)) row_grads = like_rows(grad, T * k);
    if (ctx->needs_input_grad(2)) gate_grads = empty({T, k}, gates.scalar_type(), gates.device());
    done(brt_unsort_cells_backward(
        grad.data_ptr(), data_or_null(rows), static_cast<const int32_t*>(places.data_ptr()),
        gates.data_ptr(), data_or_null(row_grads), data_or_null(gate_grads), T, (int)k,
        grad.numel() / T, dtype_of(grad), dtype_of(gates), stream_of(grad)));
    return once({row_grads, at::Tensor(), gate_grads});
  }
};

// order_picks(picks, path_num) -> (places, loads)
PyObject* order_picks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 2 || modes_active()) return nullptr;
    const at::Tensor* picks = plain(a[0]);
    if (picks == nullptr || picks->dim() != 2 || !picks->is_contiguous() || picks->numel() == 0 ||
        !Place::of(*picks) ||
        (picks->scalar_type() != at::kInt && picks->scalar_type() != at::kLong))
      return nullptr;
    const long paths = PyLong_AsLong(a[1]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return nullptr;
    }
    if (paths < 1 || paths > 1024) return nullptr;
    Memory memory;
    const Place p(*picks);
    const int64_t T = picks->size(0), k = picks->size(1);
    const bool wide = picks->scalar_type() == at::kLong;
    const void* const from = memory.of(picks);
    at::Tensor places, loads;
    int rc;
    {
      const Unlocked unlocked;
      places = empty({T, k}, at::kInt, p.device);
      loads = empty({paths}, at::kInt, p.device);
      const int64_t bytes = (int64_t)brt_pick_order_scratch_bytes(T * k, (int)paths);
      at::Tensor scratch;
      if (bytes > 0) scratch = empty({bytes}, at::kByte, p.device);
      rc = brt_order_picks(from, wide, T * k, (int)paths,
                           static_cast<int32_t*>(places.data_ptr()),
                           static_cast<int32_t*>(loads.data_ptr()), data_or_null(scratch),
                           (size_t)bytes, p.handle());
    }
    if (rc != BRT_OK) return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(places), THPVariable_Wrap(loads));
  });
}

// sort_cells(in_data, places) -> rows
PyObject* sort_cells(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 2 || modes_active()) return nullptr;
    const at::Tensor *x = plain(a[0]), *places = plain(a[1]);
    if (x == nullptr || x->dim() < 1 || !x->is_contiguous() || x->numel() == 0 ||
        dtype_of(*x) < 0 || !Place::of(*x) || !is_places(places) || !same_device(*x, places) ||
        x->size(0) != places->size(0))
      return nullptr;
    const at::Tensor cells = *x, at_rows = *places;  // kept while other threads run
    const bool grad = wants_grad(x);
    at::Tensor rows;
    {
      const Unlocked unlocked;
      rows = grad ? SortCells::apply(cells, at_rows) : sorted_rows(cells, at_rows);
    }
    return THPVariable_Wrap(rows);
  });
}

// sort_cells_fp8(in_data, places) -> (codes, scales)
PyObject* sort_cells_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 2 || modes_active()) return nullptr;
    const at::Tensor *x = plain(a[0]), *places = plain(a[1]);
    if (x == nullptr || x->dim() != 2 || !x->is_contiguous() || x->numel() == 0 ||
        dtype_of(*x) < 0 || x->size(1) % 16 != 0 || wants_grad(x) || !Place::of(*x) ||
        !is_places(places) || !same_device(*x, places) || x->size(0) != places->size(0))
      return nullptr;
    Memory memory;
    const Place p(*x);
    const int64_t T = x->size(0), k = places->size(1), width = x->size(1);
    const int dtype = dtype_of(*x);
    const void* const from = memory.of(x);
    if (reinterpret_cast<uintptr_t>(from) % 16 != 0) return nullptr;
    const int32_t* const at_rows = memory.ints(places);
    at::Tensor codes, scales;
    int rc;
    {
      const Unlocked unlocked;
      codes = empty({T * k, width}, at::kFloat8_e4m3fn, p.device);
      scales = empty({(width + 127) / 128, T * k}, at::kFloat, p.device);
      rc = brt_sort_cells_fp8(from, at_rows, codes.data_ptr(),
                              static_cast<float*>(scales.data_ptr()), T, (int)k, width, dtype,
                              p.handle());
      scales = scales.t();
    }
    if (rc != BRT_OK) return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(codes), THPVariable_Wrap(scales));
  });
}

// unsort_cells(rows, places, gates | None) -> cells
PyObject* unsort_cells(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 3 || modes_active()) return nullptr;
    const at::Tensor *x = plain(a[0]), *places = plain(a[1]), *weights = nullptr;
    if (x == nullptr || x->dim() < 1 || !x->is_contiguous() || x->numel() == 0 ||
        dtype_of(*x) < 0 || !Place::of(*x) || !is_places(places) || !same_device(*x, places) ||
        x->size(0) != places->numel())
      return nullptr;
    if (a[2] != Py_None) {
      weights = plain(a[2]);
      if (weights == nullptr || !weights->is_contiguous() || weights->sizes() != places->sizes() ||
          !same_device(*x, weights) ||
          (weights->scalar_type() != at::kFloat && weights->scalar_type() != x->scalar_type()))
        return nullptr;
    }
    const at::Tensor rows = *x, at_rows = *places;  // kept while other threads run
    const at::Tensor gates = weights != nullptr ? *weights : at::Tensor();
    const bool grad = wants_grad(x) || wants_grad(weights);
    at::Tensor cells;
    {
      const Unlocked unlocked;
      cells = !grad              ? cells_of(rows, at_rows, gates)
              : gates.defined() ? UnsortCells::apply(rows, at_rows, gates)
                                : SumCells::apply(rows, at_rows);
    }
    return THPVariable_Wrap(cells);
  });
}

// ---- expert layers in 8 bits -----------------------------------------------------------------

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool matrix(const at::Tensor* t, at::ScalarType type) {
  return t != nullptr && t->scalar_type() == type && t->dim() == 2 && t->is_contiguous() &&
         t->numel() > 0 && t->size(1) % 16 == 0;
}
int64_t blocks_of(int64_t features) { return (features + 127) / 128; }

// quantize_rows(rows) -> (codes, scales)
PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 1 || modes_active()) return nullptr;
    const at::Tensor* x = plain(a[0]);
    if (x == nullptr || dtype_of(*x) < 0 || !matrix(x, x->scalar_type()) || wants_grad(x) ||
        !Place::of(*x))
      return nullptr;
    Memory memory;
    const Place p(*x);
    const int64_t L = x->size(0), width = x->size(1);
    const int dtype = dtype_of(*x);
    const void* const from = memory.of(x);
    if (!aligned16(from)) return nullptr;
    at::Tensor codes, scales;
    int rc;
    {
      const Unlocked unlocked;
      codes = empty({L, width}, at::kFloat8_e4m3fn, p.device);
      scales = empty({blocks_of(width), L}, at::kFloat, p.device);
      rc = brt_quantize_rows(from, codes.data_ptr(), static_cast<float*>(scales.data_ptr()), L,
                             width, dtype, p.handle());
      scales = scales.t();
    }
    if (rc != BRT_OK) return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(codes), THPVariable_Wrap(scales));
  });
}

// grouped_expert_linear_fp8(rows, row_scales, weights, weight_scales, loads, slot, relu,
//                           out | None, zero_unused, error_word) -> out
PyObject* grouped_expert_linear_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 10 || modes_active()) return nullptr;
    const at::Tensor *x = plain(a[0]), *rs = plain(a[1]), *w = plain(a[2]), *ws = plain(a[3]);
    const at::Tensor *loads = plain(a[4]), *word = plain(a[9]), *out = nullptr;
    if (!matrix(x, at::kFloat8_e4m3fn) || rs == nullptr || w == nullptr || ws == nullptr ||
        loads == nullptr || word == nullptr || wants_grad(x) || wants_grad(rs) || wants_grad(w) ||
        wants_grad(ws) || !Place::of(*x))
      return nullptr;
    const int64_t L = x->size(0), K = x->size(1);
    if (w->scalar_type() != at::kFloat8_e4m3fn || w->dim() != 3 || !w->is_contiguous() ||
        w->size(2) != K || w->size(1) < 1 || w->size(1) % 16 != 0)
      return nullptr;
    const int64_t E = w->size(0), N = w->size(1);
    if (E < 1 || E > 1024 || rs->scalar_type() != at::kFloat || rs->dim() != 2 ||
        rs->size(0) != L || rs->size(1) != blocks_of(K) || ws->scalar_type() != at::kFloat ||
        ws->dim() != 3 || !ws->is_contiguous() || ws->size(0) != E ||
        ws->size(1) != blocks_of(N) || ws->size(2) != blocks_of(K) || !int32c(loads, 1) ||
        loads->numel() != E)
      return nullptr;
    for (const at::Tensor* t : {rs, w, ws, loads, word})
      if (!same_device(*x, t)) return nullptr;
    const long long slot = PyLong_AsLongLong(a[5]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return nullptr;
    }
    if (slot < 0 || slot > 0x7fffffffLL || (slot > 0 && slot * E != L)) return nullptr;
    const int relu = truth(a[6]), zero_unused = truth(a[8]);
    if (relu < 0 || zero_unused < 0) return nullptr;
    if (a[7] != Py_None) {
      out = plain(a[7]);
      if (out == nullptr || out->scalar_type() != at::kBFloat16 || out->dim() != 2 ||
          !out->is_contiguous() || out->size(0) != L || out->size(1) != N || wants_grad(out) ||
          !same_device(*x, out))
        return nullptr;
    }
    Memory memory;
    const Place p(*x);
    const void *const rows = memory.of(x), *const weights = memory.of(w);
    const auto row_scales = static_cast<const float*>(memory.of(rs));
    const auto weight_scales = static_cast<const float*>(memory.of(ws));
    const int32_t* const counts = memory.ints(loads);
    void* const error = memory.of(word);
    void* dst = memory.of(out);
    if (!aligned16(rows) || !aligned16(weights) || !aligned16(dst)) return nullptr;
    const int64_t row_stride = rs->stride(0), block_stride = rs->stride(1);
    at::Tensor made;
    int rc;
    {
      const Unlocked unlocked;
      if (out == nullptr) {
        made = empty({L, N}, at::kBFloat16, p.device);
        dst = made.data_ptr();
      }
      rc = brt_grouped_expert_gemm_fp8(rows, row_scales, row_stride, block_stride, weights,
                                       weight_scales, dst, counts, (int)E, L, (int32_t)slot, K, N,
                                       relu, zero_unused, error, p.handle());
    }
    if (rc != BRT_OK) return nullptr;
    if (out == nullptr) return THPVariable_Wrap(made);
    // autograd notices when it had saved what was in the buffer
    if (!out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
    return Py_NewRef(a[7]);
  });
}

// grouped_expert_weight_grad(grads, rows, loads, slot, fp32, error_word) -> the gradients
PyObject* grouped_expert_weight_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || modes_active()) return nullptr;
    const at::Tensor *g = plain(a[0]), *x = plain(a[1]), *loads = plain(a[2]),
                     *word = plain(a[5]);
    if (!matrix(g, at::kBFloat16) || !matrix(x, at::kBFloat16) || g->size(0) != x->size(0) ||
        wants_grad(g) || wants_grad(x) || !int32c(loads, 1) || loads->numel() < 1 ||
        loads->numel() > 1024 || word == nullptr || !Place::of(*x) || !same_device(*x, g) ||
        !same_device(*x, loads) || !same_device(*x, word))
      return nullptr;
    const int64_t L = x->size(0), N = g->size(1), K = x->size(1), E = loads->numel();
    const long long slot = PyLong_AsLongLong(a[3]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return nullptr;
    }
    if (slot < 0 || slot > 0x7fffffffLL || (slot > 0 && slot * E != L)) return nullptr;
    const int wide = truth(a[4]);
    if (wide < 0) return nullptr;
    Memory memory;
    const Place p(*x);
    const void *const grads = memory.of(g), *const rows = memory.of(x);
    const int32_t* const counts = memory.ints(loads);
    void* const error = memory.of(word);
    if (!aligned16(grads) || !aligned16(rows)) return nullptr;
    at::Tensor out;
    int rc;
    {
      const Unlocked unlocked;
      out = empty({E, N, K}, wide ? at::kFloat : at::kBFloat16, p.device);
      rc = brt_grouped_expert_weight_grad(grads, rows, out.data_ptr(), counts, (int)E, L,
                                          (int32_t)slot, K, N, wide ? BRT_F32 : BRT_BF16, error,
                                          p.handle());
    }
    if (rc != BRT_OK) return nullptr;
    return THPVariable_Wrap(out);
  });
}

// check_capture(next_functions): the same for the node of a Python autograd function.
PyObject* check_capture_of(PyObject*, PyObject* next) {
  return guarded([&]() -> PyObject* {
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None ||
        !PyTuple_Check(next))
      return nullptr;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(next); i++) {
      PyObject* const edge = PyTuple_GET_ITEM(next, i);
      if (!PyTuple_Check(edge) || PyTuple_GET_SIZE(edge) != 2) continue;
      PyObject* const fn = PyTuple_GET_ITEM(edge, 0);
      if (!torch::autograd::THPCppFunction_Check(fn)) continue;
      auto* const node = reinterpret_cast<torch::autograd::THPCppFunction*>(fn)->cdata.get();
      TORCH_CHECK(!breaks_capture(node), kBreaksCapture);
    }
    return nullptr;
  });
}

PyMethodDef methods[] = {
    {"scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(scan)), METH_FASTCALL, nullptr},
    {"route_scores", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(route_scores)),
     METH_FASTCALL, nullptr},
    {"dispatch", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(dispatch)), METH_FASTCALL,
     nullptr},
    {"combine", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(combine)), METH_FASTCALL,
     nullptr},
    {"order_picks", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(order_picks)),
     METH_FASTCALL, nullptr},
    {"sort_cells", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(sort_cells)),
     METH_FASTCALL, nullptr},
    {"sort_cells_fp8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(sort_cells_fp8)),
     METH_FASTCALL, nullptr},
    {"unsort_cells", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(unsort_cells)),
     METH_FASTCALL, nullptr},
    {"quantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(quantize_rows)),
     METH_FASTCALL, nullptr},
    {"grouped_expert_linear_fp8",
     reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(grouped_expert_linear_fp8)),
     METH_FASTCALL, nullptr},
    {"grouped_expert_weight_grad",
     reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(grouped_expert_weight_grad)),
     METH_FASTCALL, nullptr},
    {"check_capture", check_capture_of, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_ops", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_ops() {
  g_dense = PyUnicode_InternFromString("_brt_dense_counts");
  PyObject* const m = g_dense != nullptr ? PyModule_Create(&module) : nullptr;
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
