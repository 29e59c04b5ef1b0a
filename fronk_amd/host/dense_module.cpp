// dense_module.cpp - fronk_amd._dense: the dense operators over torch tensors.
//
// What fronk_amd.dense documents: arguments checked, the output and workspace
// allocated, the C ABI called. It is C++ because a call of one token takes the
// card 3 to 5 us, and the same steps in Python took the host 7 to 12 (this: 3 to 5,
// where torch's zero_ takes 3.6).
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>

#include <math.h>

#include <stdexcept>
#include <string>

#include "fronk_hip.h"

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

at::Tensor make(const at::Tensor* out, at::IntArrayRef shape, const at::Tensor& as, const char* what) {
  if (!out) return at::empty(shape, as.options());
  if (out->sizes() != shape || out->scalar_type() != as.scalar_type() || out->device() != as.device()) refuse(what);
  if (at::has_internal_overlap(*out) == at::MemOverlap::Yes) refuse("out has places of its own for all elements");
  return *out;
}
// An output whose places are also read, by other workgroups than write them.
void apart(const at::Tensor* out, const at::Tensor& in, const char* name) {
  if (!out || !out->numel() || !in.numel()) return;
  const auto both = at::get_overlap_status(*out, in);
  if (both == at::MemOverlapStatus::Full || both == at::MemOverlapStatus::Partial || out->data_ptr() == in.data_ptr())
    refuse(std::string("out shares memory with ") + name);
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

// q k v g beta state_in state_out scale offsets slots max_tokens normalize out status
PyObject* delta_rule(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 14, [&]() -> PyObject* {
    const at::Tensor &q = *tensor(a[0], "q"), &k = *tensor(a[1], "k"), &v = *tensor(a[2], "v");
    const at::Tensor &g = *tensor(a[3], "g"), &beta = *tensor(a[4], "beta");
    const at::Tensor *in = tensor(a[5], "state_in", true), *after = tensor(a[6], "state_out", true);
    const at::Tensor *offsets = tensor(a[8], "offsets", true), *slots = tensor(a[9], "slots", true);
    const at::Tensor *out = tensor(a[12], "out", true), *status = tensor(a[13], "status", true);
    fr_hip_delta r = {};
    r.type = type_of(v, "v");
    if (q.dim() != 3 || k.sizes() != q.sizes() || v.dim() != 3 || v.size(0) != q.size(0))
      refuse("q and k are [tokens, key_heads, key_dim], v [tokens, heads, value_dim]");
    like(q, v, "q"), like(k, v, "k");
    const int64_t tokens = q.size(0), heads = v.size(1), dk = q.size(2), dv = v.size(2);
    if (dk <= 0) refuse("key_dim is positive");
    for (const at::Tensor* t : {&g, &beta})
      if (t->dim() != 2 || t->size(0) != tokens || t->size(1) != heads || t->scalar_type() != at::kFloat ||
          t->device() != v.device())
        refuse("g and beta are fp32 [tokens, heads]");
    const int64_t longest = a[10] == Py_None ? tokens : whole(a[10]);
    int64_t sequences = 0;
    if (offsets) {
      sequences = offsets->numel() - 1;
      if (sequences < 0) refuse("offsets has sequences + 1 elements");
    } else if (tokens) {
      if (longest <= 0 || tokens % longest) refuse("without offsets, max_tokens divides tokens");
      sequences = tokens / longest;
    }
    int64_t rows = sequences;
    for (const at::Tensor* s : {in, after}) {
      if (!s) continue;
      if (s->dim() != 4 || s->size(1) != heads || s->size(2) != dk || s->size(3) != dv || !plain(*s, at::kFloat, v))
        refuse("a state pool is a contiguous fp32 [rows, heads, key_dim, value_dim]");
      if (s == after && in && in->size(0) != s->size(0)) refuse("both state pools have the same rows");
      rows = s->size(0);
    }
    const at::Tensor o = make(out, v.sizes(), v, "out is like v");
    row(q, "q"), row(k, "k"), row(v, "v"), row(o, "out"), row(g, "g"), row(beta, "beta");
    apart(out, q, "q"), apart(out, k, "k"), apart(out, v, "v");
    r.sequences = u32(sequences, "sequences"), r.tokens = u32(tokens, "tokens"), r.max_tokens = u32(longest, "max_tokens");
    r.key_heads = u32(q.size(1), "key_heads"), r.heads = u32(heads, "heads");
    r.key_dim = u32(dk, "key_dim"), r.value_dim = u32(dv, "value_dim"), r.slots = u32(rows, "rows");
    const int normalize = PyObject_IsTrue(a[11]);
    if (normalize < 0) throw python_error();
    r.flags = normalize ? FR_HIP_DELTA_NORMALIZE : 0;
    r.scale = (float)(a[7] == Py_None ? 1.0 / sqrt((double)dk) : number(a[7]));
    r.q = q.data_ptr(), r.k = k.data_ptr(), r.v = v.data_ptr(), r.o = o.data_ptr();
    r.g = static_cast<const float*>(g.data_ptr()), r.beta = static_cast<const float*>(beta.data_ptr());
    r.q_token = q.stride(0), r.q_head = q.stride(1), r.k_token = k.stride(0), r.k_head = k.stride(1);
    r.v_token = v.stride(0), r.v_head = v.stride(1), r.o_token = o.stride(0), r.o_head = o.stride(1);
    r.g_token = g.stride(0), r.beta_token = beta.stride(0);
    r.offsets = ints<const int32_t*>(offsets, sequences + 1, v, "offsets");
    r.slot = ints<const int32_t*>(slots, sequences, v, "slots");
    r.state_in = in ? static_cast<const float*>(in->data_ptr()) : nullptr;
    r.state_out = after ? static_cast<float*>(after->data_ptr()) : nullptr;
    r.status = ints<uint32_t*>(status, 1, v, "status");
    call("fr_hip_delta_rule", v, r, fr_hip_delta_workspace, fr_hip_delta_rule);
    written(out), written(after), written(status);
    return THPVariable_Wrap(o);
  });
}

// x codes scales zeros out
PyObject* q4_product(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Tensor &x = *tensor(a[0], "x"), &codes = *tensor(a[1], "codes"), &scales = *tensor(a[2], "scales");
    const at::Tensor *zeros = tensor(a[3], "zeros", true), *out = tensor(a[4], "out", true);
    fr_hip_q4 r = {};
    r.type = type_of(x, "x");
    if (x.dim() != 2 || codes.dim() != 2 || scales.dim() != 2) refuse("x, codes and scales are matrices");
    const int64_t tokens = x.size(0), cols = x.size(1), rows = scales.size(0), groups = scales.size(1);
    if (codes.size(0) != rows || codes.size(1) * 2 != cols || !plain(codes, at::kByte, x))
      refuse("codes is a contiguous uint8 [rows, cols / 2]");
    if (!plain(scales, at::kHalf, x) && !plain(scales, at::kBFloat16, x))
      refuse("scales is a contiguous fp16 or bf16 [rows, cols / group]");
    if (groups <= 0 || cols % groups) refuse("scales' columns divide cols");
    if (zeros && (zeros->sizes() != scales.sizes() || !plain(*zeros, at::kByte, x)))
      refuse("zeros is a contiguous uint8 tensor like scales");
    const int64_t shape[2] = {tokens, rows};
    const at::Tensor y = make(out, shape, x, "out is [tokens, rows] of x's type");
    row(x, "x"), row(y, "out");
    apart(out, x, "x");
    r.tokens = u32(tokens, "tokens"), r.rows = u32(rows, "rows"), r.cols = u32(cols, "cols");
    r.group = u32(cols / groups, "group"), r.scale_type = scales.scalar_type() == at::kHalf ? FR_HIP_F16 : FR_HIP_BF16;
    r.x = x.data_ptr(), r.codes = static_cast<const uint8_t*>(codes.data_ptr()), r.scales = scales.data_ptr();
    r.zeros = zeros ? static_cast<const uint8_t*>(zeros->data_ptr()) : nullptr, r.y = y.data_ptr();
    r.x_token = x.stride(0), r.y_token = y.stride(0);
    call("fr_hip_q4_product", x, r, fr_hip_q4_workspace, fr_hip_q4_product);
    written(out);
    return THPVariable_Wrap(y);
  });
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

// What writes and reads have in common (fr_hip_kv_write, fr_hip_kv_values).
template <typename R>
void tokens_of(R* r, const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots, const at::Tensor* status,
               const at::Tensor& cache) {
  r->type = type_of(k, "k and v");
  if (k.dim() != 3 || k.size(1) != r->cache.heads || k.size(2) != r->cache.dim || v.sizes() != k.sizes())
    refuse("k and v are [tokens, heads, dim] of one type");
  like(v, k, "v");
  if (k.device() != cache.device()) refuse("k, v and the cache are on one GPU");
  row(k, "k"), row(v, "v");
  r->tokens = u32(k.size(0), "tokens"), r->k = k.data_ptr(), r->v = v.data_ptr();
  r->k_token = k.stride(0), r->k_head = k.stride(1), r->v_token = v.stride(0), r->v_head = v.stride(1);
  r->slot = ints<const int32_t*>(&slots, k.size(0), k, "slots");
  r->status = ints<uint32_t*>(status, 1, k, "status");
}

// cache k v slots status
PyObject* kv_append(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    fr_hip_kv_write r = {};
    const at::Tensor& cache = cache_of(a[0], &r.cache);
    const at::Tensor& k = *tensor(a[1], "k");
    const at::Tensor* status = tensor(a[4], "status", true);
    tokens_of(&r, k, *tensor(a[2], "v"), *tensor(a[3], "slots"), status, cache);
    call("fr_hip_kv_append", k, [&](void* s) { return fr_hip_kv_append(&r, s); });
    for (int i = 0; i < 4; ++i) written(&THPVariable_Unpack(PyTuple_GET_ITEM(a[0], i)));
    written(status);
    Py_RETURN_NONE;
  });
}

// cache slots dtype status
PyObject* kv_read(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    fr_hip_kv_values r = {};
    const at::Tensor &cache = cache_of(a[0], &r.cache), &slots = *tensor(a[1], "slots");
    if (!THPDtype_Check(a[2])) refuse("dtype is a torch.dtype");
    const auto type = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
    const auto options = cache.options().dtype(type);
    const int64_t shape[3] = {slots.numel(), cache.size(1), cache.size(3)};
    const at::Tensor k = at::empty(shape, options), v = at::empty(shape, options);
    const at::Tensor* status = tensor(a[3], "status", true);
    tokens_of(&r, k, v, slots, status, cache);
    call("fr_hip_kv_read", k, [&](void* s) { return fr_hip_kv_read(&r, s); });
    written(status);
    return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
  });
}

// cache q table lengths scale max_context out status
PyObject* kv_attend(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    fr_hip_kv_query r = {};
    const at::Tensor& cache = cache_of(a[0], &r.cache);
    const at::Tensor &q = *tensor(a[1], "q"), &table = *tensor(a[2], "table"), &lengths = *tensor(a[3], "lengths");
    const at::Tensor *out = tensor(a[6], "out", true), *status = tensor(a[7], "status", true);
    r.type = type_of(q, "q");
    if (q.device() != cache.device()) refuse("q and the cache are on one GPU");
    if (q.dim() != 3 || q.size(2) != r.cache.dim) refuse("q is [sequences * burst, heads, dim]");
    if (table.dim() != 2 || table.scalar_type() != at::kInt || table.device() != q.device() ||
        (table.stride(1) != 1 && table.size(1) > 1))
      refuse("table is an int32 matrix");
    const int64_t sequences = table.size(0), per = table.size(1);
    if (sequences ? q.size(0) % sequences : q.size(0)) refuse("q has the same burst of every sequence");
    const int64_t most = per * r.cache.page, context = a[5] == Py_None ? most : whole(a[5]);
    if (context < 0 || context > most) refuse("max_context is within a table row's pages");
    const at::Tensor o = make(out, q.sizes(), q, "out is like q");
    r.length = ints<const int32_t*>(&lengths, sequences, q, "lengths");
    r.status = ints<uint32_t*>(status, 1, q, "status");
    if (!sequences || !q.size(0)) return THPVariable_Wrap(o);
    row(q, "q"), row(o, "out");
    r.sequences = u32(sequences, "sequences"), r.burst = u32(q.size(0) / sequences, "burst");
    r.heads = u32(q.size(1), "heads"), r.max_context = u32(context, "max_context");
    r.table_stride = u32(sequences == 1 ? std::max(table.stride(0), per) : table.stride(0), "table's stride");
    r.scale = (float)(a[4] == Py_None ? 1.0 / sqrt((double)r.cache.dim) : number(a[4]));
    r.q = q.data_ptr(), r.o = o.data_ptr(), r.table = static_cast<const int32_t*>(table.data_ptr());
    r.q_token = q.stride(0), r.q_head = q.stride(1), r.o_token = o.stride(0), r.o_head = o.stride(1);
    call("fr_hip_kv_attend", q, r, fr_hip_kv_workspace, fr_hip_kv_attend);
    written(out), written(status);
    return THPVariable_Wrap(o);
  });
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
PyMethodDef methods[] = {{"delta_rule", fast<delta_rule>(), METH_FASTCALL, nullptr},
                         {"q4_product", fast<q4_product>(), METH_FASTCALL, nullptr},
                         {"kv_append", fast<kv_append>(), METH_FASTCALL, nullptr},
                         {"kv_read", fast<kv_read>(), METH_FASTCALL, nullptr},
                         {"kv_attend", fast<kv_attend>(), METH_FASTCALL, nullptr},
                         {"bind", fast<bind>(), METH_FASTCALL, "What opens the engine on a device, and what gives its current stream."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_dense", "fronk_amd.dense's calls.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__dense() { return PyModule_Create(&module); }
