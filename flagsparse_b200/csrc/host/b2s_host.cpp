// The host side of the selection products for the usual call: plain strided CUDA tensors of one
// device, new results, nothing recorded for autograd.  A call that finds everything in order
// allocates the result, launches through the C ABI and returns the tensor; anything else (another
// layout, out=, a wrong argument, a device error to report) returns None, and
// flagsparse_b200/selection.py takes the call from the start, with its checks and messages.
//
// On a few rows the kernels take 2 to 8 microseconds; the same steps in Python take 10.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <optional>

#include "../../../include/b200sparse.h"

namespace {

// entry points of libb200sparse.so, handed over by bind()
decltype(&b2s_select_rows) p_select_rows;
decltype(&b2s_select_grad_bytes) p_select_grad_bytes;
decltype(&b2s_select_grad) p_select_grad;
decltype(&b2s_route_plan_bytes) p_route_plan_bytes;
decltype(&b2s_route_plan) p_route_plan;
decltype(&b2s_route_dispatch) p_route_dispatch;
decltype(&b2s_route_combine) p_route_combine;
decltype(&b2s_route_combine_grad) p_route_combine_grad;

constexpr int kMaxDevices = 64;
int32_t* status_of[kMaxDevices];  // the word of each device that selection.py has made
PyTypeObject* parameter_type;

// the error word of a device, or NULL when there is none yet or it holds an error
int32_t* clean_status(int device) {
  if (device < 0 || device >= kMaxDevices || !status_of[device]) return nullptr;
  return *reinterpret_cast<volatile int32_t*>(status_of[device]) ? nullptr : status_of[device];
}

// a plain CUDA tensor that no transform or mode has wrapped and that has no tangent (forward-mode
// derivatives: such a tensor does not require a gradient), or NULL
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o) && Py_TYPE(o) != parameter_type) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) return nullptr;
  const c10::DispatchKeySet keys = t.key_set();
  if (keys.has(c10::DispatchKey::Python) || keys.has(c10::DispatchKey::FuncTorchBatched) ||
      keys.has(c10::DispatchKey::FuncTorchGradWrapper) ||
      keys.has(c10::DispatchKey::Functionalize) || keys.has(c10::DispatchKey::Conjugate) ||
      keys.has(c10::DispatchKey::Negative) || t._fw_grad(0).defined())
    return nullptr;
  return &t;
}
bool recorded(const at::Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

int value_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return B2S_F32;
    case at::kDouble: return B2S_F64;
    case at::kHalf: return B2S_F16;
    case at::kBFloat16: return B2S_BF16;
    default: return -1;
  }
}
int index_code(const at::Tensor& t) {
  return t.scalar_type() == at::kInt ? B2S_I32 : t.scalar_type() == at::kLong ? B2S_I64 : -1;
}
// rows the kernels can take as they are, and their pitch
bool row_major(const at::Tensor& t, int64_t* pitch) {
  if (t.dim() != 2) return false;
  const int64_t rows = t.size(0), cols = t.size(1);
  *pitch = rows > 1 ? t.stride(0) : cols;
  return (cols <= 1 || t.stride(1) == 1) && (rows <= 1 || *pitch >= (cols > 1 ? cols : 1));
}
// whether two arrays of rows of `dim` values have addresses in common (storage objects do not say:
// one memory can have several of them); rows of one array side by side count as meeting
bool meet(const at::Tensor& a, int64_t rows_a, int64_t pitch_a, const at::Tensor& b, int64_t rows_b,
          int64_t pitch_b, int64_t dim) {
  if (rows_a <= 0 || rows_b <= 0 || dim <= 0) return false;
  const auto at_a = reinterpret_cast<uintptr_t>(a.const_data_ptr());
  const auto at_b = reinterpret_cast<uintptr_t>(b.const_data_ptr());
  return at_a < at_b + ((rows_b - 1) * pitch_b + dim) * b.element_size() &&
         at_b < at_a + ((rows_a - 1) * pitch_a + dim) * a.element_size();
}
bool number(PyObject* o, double* v) {
  if (PyFloat_CheckExact(o)) {
    *v = PyFloat_AS_DOUBLE(o);
    return true;
  }
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsDouble(o);
  if (*v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
bool integer(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0;
}
bool ignored(PyObject* o, int* has, int64_t* v) {
  *has = o != Py_None;
  *v = 0;
  return !*has || integer(o, v);
}

// the device made current where it is not, and its stream
struct On {
  std::optional<c10::cuda::CUDAGuard> guard;
  cudaStream_t stream;
  explicit On(c10::DeviceIndex device) {
    if (c10::cuda::current_device() != device) guard.emplace(device);
    stream = c10::cuda::getCurrentCUDAStream(device).stream();
  }
};

// The interpreter's lock is given up while a call allocates and launches: both may wait (for memory
// that another stream frees, for room in the queue of launches), and other threads run meanwhile.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// a new tensor beside `like`
at::Tensor fresh(c10::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

#define NOT_HERE Py_RETURN_NONE
// C++ exceptions (an allocation that failed) become Python's
#define GUARDED(...)                                    \
  try {                                                 \
    __VA_ARGS__                                         \
  } catch (const c10::OutOfMemoryError& e) {            \
    PyErr_SetString(oom_type, e.what_without_backtrace()); \
    return nullptr;                                     \
  } catch (const std::exception& e) {                   \
    PyErr_SetString(PyExc_RuntimeError, e.what());      \
    return nullptr;                                     \
  }
PyObject* oom_type;

// embedding(tokens, table, alpha, ignore_index)
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  GUARDED({
    double alpha;
    int has;
    int64_t ignore, pitch;
    if (n_args != 4 || !number(a[2], &alpha) || !ignored(a[3], &has, &ignore)) NOT_HERE;
    const at::Tensor *tokens = plain(a[0]), *table = plain(a[1]);
    if (!tokens || !table || recorded(*table)) NOT_HERE;
    const int vcode = value_code(*table), icode = index_code(*tokens), dev = table->get_device();
    int32_t* status = clean_status(dev);
    if (vcode < 0 || icode < 0 || !status || tokens->get_device() != dev ||
        !tokens->is_contiguous() || !row_major(*table, &pitch))
      NOT_HERE;
    const On on(static_cast<c10::DeviceIndex>(dev));
    const int64_t dim = table->size(1);
    c10::DimVector shape(tokens->sizes().begin(), tokens->sizes().end());
    shape.push_back(dim);
    at::Tensor out;
    int st;
    {
      const Unlocked unlocked;
      out = fresh(shape, table->scalar_type(), *table);
      st = p_select_rows(vcode, icode, tokens->const_data_ptr(), tokens->numel(), has, ignore,
                         table->const_data_ptr(), table->size(0), pitch, dim, out.data_ptr(), dim,
                         alpha, 0.0, status, on.stream);
    }
    if (st != B2S_OK) NOT_HERE;
    return THPVariable_Wrap(std::move(out));
  })
}

// embedding_grad(tokens, grad, n_rows, alpha, ignore_index, out, beta, out_dtype)
PyObject* embedding_grad(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  GUARDED({
    double alpha, beta;
    int has;
    int64_t ignore, n_rows, pitch, out_pitch;
    if (n_args != 8 || !integer(a[2], &n_rows) || n_rows < 0 || !number(a[3], &alpha) ||
        !ignored(a[4], &has, &ignore) || !number(a[6], &beta))
      NOT_HERE;
    const at::Tensor *tokens = plain(a[0]), *grad = plain(a[1]);
    if (!tokens || !grad || grad->dim() != tokens->dim() + 1 ||
        grad->sizes().slice(0, tokens->dim()) != tokens->sizes())
      NOT_HERE;
    const int vcode = value_code(*grad), icode = index_code(*tokens), dev = grad->get_device();
    int32_t* status = clean_status(dev);
    const int64_t n = tokens->numel(), dim = grad->size(grad->dim() - 1);
    pitch = dim;
    if (vcode < 0 || icode < 0 || !status || tokens->get_device() != dev ||
        !tokens->is_contiguous() || !(row_major(*grad, &pitch) || grad->is_contiguous()))
      NOT_HERE;
    at::ScalarType out_type = grad->scalar_type();
    if (a[7] != Py_None) {
      if (!THPDtype_Check(a[7])) NOT_HERE;
      out_type = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
      if (out_type != grad->scalar_type() &&
          !(out_type == at::kFloat && grad->element_size() == 2))
        NOT_HERE;
    }
    const On on(static_cast<c10::DeviceIndex>(dev));
    at::Tensor made;
    const at::Tensor* out = nullptr;
    if (a[5] != Py_None) {
      out = plain(a[5]);
      if (!out || out->get_device() != dev || out->dim() != 2 || out->size(0) != n_rows ||
          out->size(1) != dim || recorded(*out) || recorded(*grad) ||
          !row_major(*out, &out_pitch) ||
          meet(*out, n_rows, out_pitch, *grad, dim > 0 ? grad->numel() / dim : 0, pitch, dim))
        NOT_HERE;
      if (a[7] == Py_None) {
        if (out->scalar_type() != out_type && !(out->scalar_type() == at::kFloat &&
                                                grad->element_size() == 2))
          NOT_HERE;
        out_type = out->scalar_type();
      } else if (out->scalar_type() != out_type) {
        NOT_HERE;
      }
    } else {
      if (beta != 0) NOT_HERE;
      out_pitch = dim;
    }
    int st;
    {
      const Unlocked unlocked;
      if (!out) {
        made = fresh({n_rows, dim}, out_type, *grad);
        out = &made;
      }
      const int64_t bytes = p_select_grad_bytes(vcode, n, n_rows, dim);
      at::Tensor ws = fresh({bytes}, at::kByte, *grad);
      st = p_select_grad(vcode, value_code(*out), icode, tokens->const_data_ptr(), n, has, ignore,
                         grad->const_data_ptr(), pitch, n_rows, dim, out->data_ptr(), out_pitch,
                         alpha, beta, ws.data_ptr(), bytes, status, on.stream);
    }
    if (st != B2S_OK) NOT_HERE;
    if (a[5] == Py_None) return THPVariable_Wrap(std::move(made));
    if (!out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
    Py_INCREF(a[5]);
    return a[5];
  })
}

// A route: its buffer (slots, indptr, indices), n_tokens, k, n_experts, and the stream it was
// made on (a call on another one is selection.py's, which records it).
struct Route {
  const int32_t *slots, *held;
  int64_t n_tokens, k, n_rows;
  int dev;
};
bool route(PyObject* const* a, Route* r, cudaStream_t* made_on) {
  const at::Tensor* buffer = plain(a[0]);
  int64_t n_experts, stream;
  if (!buffer || !integer(a[1], &r->n_tokens) || !integer(a[2], &r->k) ||
      !integer(a[3], &n_experts) || !integer(a[4], &stream))
    return false;
  r->n_rows = r->n_tokens * r->k;
  r->dev = buffer->get_device();
  r->slots = static_cast<const int32_t*>(buffer->const_data_ptr());
  r->held = r->slots + r->n_rows + n_experts;
  *made_on = reinterpret_cast<cudaStream_t>(stream);
  return true;
}
constexpr int kRouteArgs = 5;

// route_plan(experts, n_experts) -> the buffer and the stream
PyObject* route_plan(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  GUARDED({
    int64_t n_experts;
    if (n_args != 2 || !integer(a[1], &n_experts)) NOT_HERE;
    const at::Tensor* experts = plain(a[0]);
    if (!experts || experts->dim() != 2 || !experts->is_contiguous()) NOT_HERE;
    const int icode = index_code(*experts), dev = experts->get_device();
    int32_t* status = clean_status(dev);
    if (icode < 0 || !status || n_experts < 0 || n_experts > 2047) NOT_HERE;
    const int64_t n_tokens = experts->size(0), k = experts->size(1), n = n_tokens * k;
    if (n > 0x7fffffff) NOT_HERE;
    const On on(static_cast<c10::DeviceIndex>(dev));
    at::Tensor buffer;
    int st;
    {
      const Unlocked unlocked;
      const int64_t bytes = p_route_plan_bytes(n_tokens, k, n_experts);
      const int64_t scratch = (2 * n + n_experts + 1 + 63) / 64 * 64;
      buffer = fresh({scratch + bytes / 4}, at::kInt, *experts);
      int32_t* arrays = buffer.data_ptr<int32_t>();
      st = p_route_plan(icode, experts->const_data_ptr(), n_tokens, k, n_experts, arrays,
                        arrays + n, arrays + n + n_experts + 1, arrays + scratch, bytes, status,
                        on.stream);
    }
    if (st != B2S_OK) NOT_HERE;
    PyObject* stream = PyLong_FromLongLong(reinterpret_cast<intptr_t>(on.stream));
    PyObject* wrapped = THPVariable_Wrap(std::move(buffer));
    PyObject* pair = stream && wrapped ? PyTuple_Pack(2, wrapped, stream) : nullptr;
    Py_XDECREF(stream);
    Py_XDECREF(wrapped);
    return pair;
  })
}

// dispatch(route..., x)
PyObject* dispatch(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  GUARDED({
    Route r;
    cudaStream_t made_on;
    int64_t pitch;
    if (n_args != kRouteArgs + 1 || !route(a, &r, &made_on)) NOT_HERE;
    const at::Tensor* x = plain(a[kRouteArgs]);
    if (!x || recorded(*x) || x->get_device() != r.dev || !row_major(*x, &pitch) ||
        x->size(0) != r.n_tokens)
      NOT_HERE;
    const int vcode = value_code(*x);
    const On on(static_cast<c10::DeviceIndex>(r.dev));
    if (vcode < 0 || on.stream != made_on) NOT_HERE;
    const int64_t dim = x->size(1);
    at::Tensor out;
    int st;
    {
      const Unlocked unlocked;
      out = fresh({r.n_rows, dim}, x->scalar_type(), *x);
      st = p_route_dispatch(vcode, x->const_data_ptr(), pitch, r.n_tokens, r.k, dim, r.slots,
                            r.held, out.data_ptr(), dim, on.stream);
    }
    if (st != B2S_OK) NOT_HERE;
    return THPVariable_Wrap(std::move(out));
  })
}

// weights None or contiguous (n_tokens, k), of the rows' type or float32
bool weights_of(PyObject* o, const Route& r, int vcode, const at::Tensor** w, int* wcode) {
  *w = nullptr;
  *wcode = 0;
  if (o == Py_None) return true;
  *w = plain(o);
  if (!*w || (*w)->get_device() != r.dev || !(*w)->is_contiguous() || (*w)->dim() != 2 ||
      (*w)->size(0) != r.n_tokens || (*w)->size(1) != r.k)
    return false;
  *wcode = value_code(**w);
  return *wcode == vcode || *wcode == B2S_F32;
}

// combine(route..., y, weights, alpha)
PyObject* combine(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  GUARDED({
    Route r;
    cudaStream_t made_on;
    int64_t pitch;
    double alpha;
    int wcode;
    const at::Tensor* w;
    if (n_args != kRouteArgs + 3 || !route(a, &r, &made_on) || !number(a[kRouteArgs + 2], &alpha))
      NOT_HERE;
    const at::Tensor* y = plain(a[kRouteArgs]);
    if (!y || recorded(*y) || y->get_device() != r.dev || !row_major(*y, &pitch) ||
        y->size(0) != r.n_rows)
      NOT_HERE;
    const int vcode = value_code(*y);
    const On on(static_cast<c10::DeviceIndex>(r.dev));
    if (vcode < 0 || on.stream != made_on ||
        !weights_of(a[kRouteArgs + 1], r, vcode, &w, &wcode) || (w && recorded(*w)))
      NOT_HERE;
    const int64_t dim = y->size(1);
    at::Tensor out;
    int st;
    {
      const Unlocked unlocked;
      out = fresh({r.n_tokens, dim}, y->scalar_type(), *y);
      st = p_route_combine(vcode, y->const_data_ptr(), pitch, r.slots, wcode,
                           w ? w->const_data_ptr() : nullptr, r.n_tokens, r.k, dim,
                           out.data_ptr(), dim, alpha, 0.0, on.stream);
    }
    if (st != B2S_OK) NOT_HERE;
    return THPVariable_Wrap(std::move(out));
  })
}

// combine_grad(route..., grad, y, weights, alpha) -> (grad_y, grad_weights)
PyObject* combine_grad(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  GUARDED({
    Route r;
    cudaStream_t made_on;
    int64_t pitch, y_pitch;
    double alpha;
    int wcode;
    const at::Tensor* w;
    if (n_args != kRouteArgs + 4 || !route(a, &r, &made_on) || !number(a[kRouteArgs + 3], &alpha))
      NOT_HERE;
    const at::Tensor *g = plain(a[kRouteArgs]), *y = plain(a[kRouteArgs + 1]);
    if (!g || !y || g->get_device() != r.dev || y->get_device() != r.dev ||
        !row_major(*g, &pitch) || !row_major(*y, &y_pitch) || g->size(0) != r.n_tokens ||
        y->size(0) != r.n_rows || g->size(1) != y->size(1) ||
        g->scalar_type() != y->scalar_type())
      NOT_HERE;
    const int vcode = value_code(*g);
    const On on(static_cast<c10::DeviceIndex>(r.dev));
    if (vcode < 0 || on.stream != made_on || a[kRouteArgs + 2] == Py_None ||
        !weights_of(a[kRouteArgs + 2], r, vcode, &w, &wcode))
      NOT_HERE;
    const int64_t dim = g->size(1);
    at::Tensor grad_y, grad_w;
    int st;
    {
      const Unlocked unlocked;
      grad_y = fresh({r.n_rows, dim}, g->scalar_type(), *g);
      grad_w = fresh({r.n_tokens, r.k}, w->scalar_type(), *w);
      st = p_route_combine_grad(vcode, g->const_data_ptr(), pitch, y->const_data_ptr(), y_pitch,
                                r.slots, r.held, wcode, w->const_data_ptr(), r.n_tokens, r.k, dim,
                                alpha, grad_y.data_ptr(), dim, grad_w.data_ptr(), on.stream);
    }
    if (st != B2S_OK) NOT_HERE;
    PyObject* first = THPVariable_Wrap(std::move(grad_y));
    PyObject* second = THPVariable_Wrap(std::move(grad_w));
    PyObject* pair = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return pair;
  })
}

// bind(eight addresses in the order below, torch.nn.Parameter, torch.OutOfMemoryError)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 10 || !PyType_Check(a[8]) || !PyExceptionClass_Check(a[9])) {
    PyErr_SetString(PyExc_TypeError, "bind takes eight addresses and two types");
    return nullptr;
  }
  void* p[8];
  for (int i = 0; i < 8; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i] && PyErr_Occurred()) return nullptr;
  }
  p_select_rows = reinterpret_cast<decltype(p_select_rows)>(p[0]);
  p_select_grad_bytes = reinterpret_cast<decltype(p_select_grad_bytes)>(p[1]);
  p_select_grad = reinterpret_cast<decltype(p_select_grad)>(p[2]);
  p_route_plan_bytes = reinterpret_cast<decltype(p_route_plan_bytes)>(p[3]);
  p_route_plan = reinterpret_cast<decltype(p_route_plan)>(p[4]);
  p_route_dispatch = reinterpret_cast<decltype(p_route_dispatch)>(p[5]);
  p_route_combine = reinterpret_cast<decltype(p_route_combine)>(p[6]);
  p_route_combine_grad = reinterpret_cast<decltype(p_route_combine_grad)>(p[7]);
  Py_INCREF(a[8]);
  Py_INCREF(a[9]);
  parameter_type = reinterpret_cast<PyTypeObject*>(a[8]);
  oom_type = a[9];
  Py_RETURN_NONE;
}

// bind_status(device index, address of its error word)
PyObject* bind_status(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  int64_t device, address;
  if (n_args != 2 || !integer(a[0], &device) || !integer(a[1], &address) || device < 0) {
    PyErr_SetString(PyExc_TypeError, "bind_status takes a device index and an address");
    return nullptr;
  }
  if (device < kMaxDevices) status_of[device] = reinterpret_cast<int32_t*>(address);
  Py_RETURN_NONE;
}

#define METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(embedding), METHOD(embedding_grad), METHOD(route_plan),
                         METHOD(dispatch),  METHOD(combine),        METHOD(combine_grad),
                         METHOD(bind),      METHOD(bind_status),    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_b2s_host", nullptr, -1, methods,
                      nullptr,               nullptr,     nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__b2s_host(void) {
  PyObject* made = PyModule_Create(&module);
  // the PyTorch whose structures this reads; nothing else may be called under another one
  if (made && PyModule_AddStringConstant(made, "torch_version", B2S_TORCH_VERSION) != 0)
    Py_CLEAR(made);
  return made;
}
