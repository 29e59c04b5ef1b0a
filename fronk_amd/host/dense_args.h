// dense_args.h - what the torch sides of the dense operators share: arguments
// checked, outputs and workspaces allocated, the C ABI called on torch's current
// stream.
#pragma once
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>

#include <math.h>

#include <stdexcept>
#include <string>

#include "fronk_hip.h"
#include "overlap.h"

namespace {

typedef PyObject* const* Args;

PyObject *g_open, *g_stream;   // open the engine on a device; give torch's current stream of it

[[noreturn]] void refuse(const std::string& what) { throw std::invalid_argument(what); }

// A tensor argument; None where that is taken. There is no backward pass and no
// forward-mode one, so one that autograd would follow here is refused.
const at::Tensor* tensor(PyObject* o, const char* name, bool optional = false) {
  if (o == Py_None && optional) return nullptr;
  if (!THPVariable_Check(o)) refuse(std::string(name) + " is a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if ((t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined())
    refuse(std::string(name) + " carries a gradient, which is not followed here: detach it, or call under torch.no_grad()");
  return &t;
}
// What a call wrote to, so that autograd sees that it has changed.
void written(const at::Tensor* t) {
  if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

unsigned type_of(const at::Tensor& t, const char* name) {
  if (t.is_cuda()) switch (t.scalar_type()) {
      case at::kFloat: return FR_HIP_F32;
      case at::kHalf: return FR_HIP_F16;
      case at::kBFloat16: return FR_HIP_BF16;
      default: break;
    }
  refuse(std::string(name) + " is float32, float16 or bfloat16, on the GPU");
}

// A tensor of one device and type with a contiguous last axis.
void like(const at::Tensor& t, const at::Tensor& as, const char* name) {
  if (t.scalar_type() != as.scalar_type() || t.device() != as.device()) refuse(std::string(name) + " has another type or device");
}
void row(const at::Tensor& t, const char* name) {
  if (t.stride(-1) != 1 && t.size(-1) != 1) refuse(std::string(name) + "'s last axis is contiguous");
}
bool plain(const at::Tensor& t, at::ScalarType type, const at::Tensor& as) {
  return t.scalar_type() == type && t.device() == as.device() && t.is_contiguous();
}

template <typename P> P ints(const at::Tensor* t, int64_t n, const at::Tensor& as, const char* name) {
  if (!t) return nullptr;
  if (t->numel() != n || !plain(*t, at::kInt, as))
    refuse(std::string(name) + " is a contiguous int32 tensor of " + std::to_string(n) + " on the GPU");
  return static_cast<P>(t->data_ptr());
}

unsigned u32(int64_t n, const char* name) {
  if (n < 0 || n > 0xffffffffll) refuse(std::string(name) + " does not fit");
  return (unsigned)n;
}

// A tensor's places: within its storage where another one has the same (which may be of no
// memory yet), by address otherwise.
fronk::Strided strided(const at::Tensor& t, bool within) {
  const int64_t size = (int64_t)t.element_size();
  const uintptr_t at = within ? (uintptr_t)(t.storage_offset() * size) : (uintptr_t)t.data_ptr();
  return {at, size, t.dim(), t.sizes().data(), t.strides().data()};
}
at::Tensor make(const at::Tensor* out, at::IntArrayRef shape, const at::Tensor& as, const char* what) {
  if (!out) return at::empty(shape, as.options());
  if (out->sizes() != shape || out->scalar_type() != as.scalar_type() || out->device() != as.device()) refuse(what);
  if (out->numel() && fronk::shares(strided(*out, true))) refuse("out has places of its own for all elements");
  return *out;
}
// An output whose places are also read, by other workgroups than write them.
void apart(const at::Tensor* out, const at::Tensor& in, const char* name) {
  if (!out || !out->numel() || !in.numel()) return;
  const bool one = out->is_alias_of(in);
  if (!one && (!out->data_ptr() || !in.data_ptr())) return;
  if (fronk::share(strided(*out, one), strided(in, one))) refuse(std::string("out shares memory with ") + name);
}

// The engine is one GPU's: on another one's tensors it would work out of order with
// what made them, or not at all.
void on_engine(const at::Tensor& as) {
  const int device = fr_hip_device();
  if (device >= 0 && device != as.get_device())
    refuse("the tensors are on GPU " + std::to_string(as.get_device()) + ", the open engine on GPU " + std::to_string(device));
}

// The call on torch's current stream (HIP's default stream is 0 there), opening
// the engine first where nothing has. The C ABI makes its device current: torch's
// is put back behind it.
template <typename F> void call(const char* name, const at::Tensor& as, F f) {
  on_engine(as);
  const c10::DeviceGuard guard(as.device());
  PyObject* stream = PyObject_CallFunction(g_stream, "i", (int)as.get_device());
  if (!stream) throw python_error();
  void* s = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!s && PyErr_Occurred()) throw python_error();
  if (!s) s = FR_HIP_STREAM_DEFAULT;
  int rc = f(s);
  if (rc == -2) {   // no open engine
    PyObject* r = PyObject_CallFunction(g_open, "i", (int)as.get_device());
    if (!r) throw python_error();
    Py_DECREF(r);
    rc = f(s);
  }
  if (rc == -1) refuse(std::string(name) + ": invalid arguments (-1)");
  if (rc == -5) refuse(std::string(name) + ": sizes outside the supported range (-5)");
  if (rc) throw std::runtime_error(std::string(name) + " failed with " + std::to_string(rc));
}
template <typename R, typename W, typename F>
void call(const char* name, const at::Tensor& as, const R& request, W workspace, F f) {
  on_engine(as);
  const size_t n = workspace(&request);
  at::Tensor w;
  if (n) w = at::empty({(int64_t)n}, as.options().dtype(at::kByte));
  call(name, as, [&](void* s) { return f(&request, n ? w.data_ptr() : nullptr, n, s); });
}

template <typename F> PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F f) {
  HANDLE_TH_ERRORS
  if (given != wanted) refuse("wrong number of arguments");
  try {
    return f();
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw python_error();
  return x;
}
int64_t whole(PyObject* o) {
  const int64_t x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return x;
}

// The cache of four tensors that a tuple holds.
const at::Tensor& cache_of(PyObject* o, fr_hip_kv_cache* c) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) refuse("the cache is a tuple of four tensors");
  const at::Tensor *t[4];
  for (int i = 0; i < 4; ++i) t[i] = tensor(PyTuple_GET_ITEM(o, i), "each of the cache");
  const at::Tensor& k = *t[0];
  if (k.dim() != 4) refuse("k_codes is [pages, heads, page, dim]");
  const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2), dim = k.size(3);
  const int64_t v[5] = {pages, heads, page / 16, dim, 16};
  if (page % 16 || t[1]->sizes() != at::IntArrayRef(v)) refuse("v_codes is [pages, heads, page / 16, dim, 16]");
  for (int i = 2; i < 4; ++i)
    if (t[i]->sizes() != k.sizes().slice(0, 3)) refuse("k_exp and v_exp are [pages, heads, page]");
  for (const at::Tensor* x : t)
    if (!x->is_cuda() || !plain(*x, at::kByte, k)) refuse("the cache is of contiguous uint8 tensors on one GPU");
  c->pages = u32(pages, "pages"), c->heads = u32(heads, "heads"), c->page = u32(page, "page"), c->dim = u32(dim, "dim");
  uint8_t** to[4] = {&c->k_codes, &c->v_codes, &c->k_exp, &c->v_exp};
  for (int i = 0; i < 4; ++i) *to[i] = static_cast<uint8_t*>(t[i]->data_ptr());
  return k;
}

PyObject* bind(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 2, [&]() -> PyObject* {
    Py_INCREF(a[0]), Py_INCREF(a[1]);
    g_open = a[0], g_stream = a[1];
    Py_RETURN_NONE;
  });
}

template <PyObject* (*F)(PyObject*, Args, Py_ssize_t)> PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

}  // namespace
