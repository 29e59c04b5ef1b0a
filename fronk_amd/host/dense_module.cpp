// dense_module.cpp - fronk_amd._dense: the dense operators over torch tensors.
//
// What fronk_amd.dense documents: arguments checked, the output and workspace
// allocated, the C ABI called. It is C++ because a call of one token takes the
// card 3 to 5 us, and the same steps in Python took the host 7 to 12 (this: 3 to 5,
// where torch's zero_ takes 3.6).
#include "dense_args.h"

namespace {

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
