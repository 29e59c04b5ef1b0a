// attention_module.cpp - fronk_amd._attention: the operators of an attention layer
// around its cache over torch tensors, as dense_module.cpp has the other dense ones.
#include "dense_args.h"

namespace {

// q k positions frequencies interleaved magnitude out
PyObject* rotary(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const at::Tensor &q = *tensor(a[0], "q"), &positions = *tensor(a[2], "positions");
    const at::Tensor *k = tensor(a[1], "k", true), &frequencies = *tensor(a[3], "frequencies");
    const at::Tensor *q_out = nullptr, *k_out = nullptr;
    if (a[6] != Py_None) {
      if (!PyTuple_Check(a[6]) || PyTuple_GET_SIZE(a[6]) != 2) refuse("out is a pair of tensors");
      q_out = tensor(PyTuple_GET_ITEM(a[6], 0), "out"), k_out = tensor(PyTuple_GET_ITEM(a[6], 1), "out", !k);
      if (!k && k_out) refuse("out has no place for a k that is not given");
    }
    fr_hip_rotary r = {};
    r.type = type_of(q, "q");
    if (q.dim() != 3 || (k && (k->dim() != 3 || k->size(0) != q.size(0) || k->size(2) != q.size(2))))
      refuse("q is [tokens, heads, dim], k [tokens, kv_heads, dim]");
    if (k) like(*k, q, "k");
    const int64_t pairs = frequencies.numel();
    if (frequencies.dim() != 1 || !plain(frequencies, at::kDouble, q)) refuse("frequencies is a contiguous float64 vector on the GPU");
    if (pairs <= 0 || 2 * pairs > q.size(2)) refuse("frequencies has one to dim / 2 elements");
    r.positions = ints<const int32_t*>(&positions, q.size(0), q, "positions");
    const at::Tensor qo = make(q_out, q.sizes(), q, "out is like q and k");
    at::Tensor ko;
    if (k) ko = make(k_out, k->sizes(), q, "out is like q and k");
    // In place, or apart.
    auto same = [](const at::Tensor* out, const at::Tensor& in) {
      return out && out->data_ptr() == in.data_ptr() && out->strides() == in.strides();
    };
    if (!same(q_out, q)) apart(q_out, q, "q");
    if (k) apart(q_out, *k, "k"), apart(k_out, q, "q");
    if (k && !same(k_out, *k)) apart(k_out, *k, "k");
    if (q_out && k_out) apart(q_out, *k_out, "itself");
    apart(q_out, positions, "positions"), apart(q_out, frequencies, "frequencies");
    apart(k_out, positions, "positions"), apart(k_out, frequencies, "frequencies");
    row(q, "q"), row(qo, "out");
    if (k) row(*k, "k"), row(ko, "out");
    r.tokens = u32(q.size(0), "tokens"), r.heads = u32(q.size(1), "heads"), r.dim = u32(q.size(2), "dim"), r.pairs = u32(pairs, "pairs");
    const int interleaved = PyObject_IsTrue(a[4]);
    if (interleaved < 0) throw python_error();
    r.flags = interleaved ? FR_HIP_ROTARY_INTERLEAVED : 0, r.magnitude = (float)number(a[5]);
    r.q = q.data_ptr(), r.q_out = qo.data_ptr(), r.frequencies = static_cast<const double*>(frequencies.data_ptr());
    r.q_token = q.stride(0), r.q_head = q.stride(1), r.qo_token = qo.stride(0), r.qo_head = qo.stride(1);
    if (k) {
      r.kv_heads = u32(k->size(1), "kv_heads"), r.k = k->data_ptr(), r.k_out = ko.data_ptr();
      r.k_token = k->stride(0), r.k_head = k->stride(1), r.ko_token = ko.stride(0), r.ko_head = ko.stride(1);
    }
    call("fr_hip_rotate", q, [&](void* s) { return fr_hip_rotate(&r, s); });
    written(q_out), written(k_out);
    if (k) return Py_BuildValue("(NN)", THPVariable_Wrap(qo), THPVariable_Wrap(ko));
    return Py_BuildValue("(NO)", THPVariable_Wrap(qo), Py_None);
  });
}

// How many sequences there are, and how long they may be: by offsets, or as many tokens each.
int64_t sequences_of(const at::Tensor* offsets, int64_t tokens, int64_t longest) {
  if (offsets) {
    if (offsets->numel() < 1) refuse("offsets has sequences + 1 elements");
    return offsets->numel() - 1;
  }
  if (!tokens) return 0;
  if (longest <= 0 || tokens % longest) refuse("without offsets, max_tokens divides tokens");
  return tokens / longest;
}

// q k v offsets k_offsets max_tokens max_context scale out status
PyObject* prompt_attend(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject* {
    const at::Tensor &q = *tensor(a[0], "q"), &k = *tensor(a[1], "k"), &v = *tensor(a[2], "v");
    const at::Tensor *offsets = tensor(a[3], "offsets", true), *k_offsets = tensor(a[4], "k_offsets", true);
    const at::Tensor *out = tensor(a[8], "out", true), *status = tensor(a[9], "status", true);
    fr_hip_prompt r = {};
    r.type = type_of(q, "q");
    if (q.dim() != 3 || k.dim() != 3 || v.sizes() != k.sizes() || k.size(2) != q.size(2))
      refuse("q is [tokens, heads, dim], k and v [k_tokens, kv_heads, dim]");
    like(k, q, "k"), like(v, q, "v");
    const int64_t tokens = q.size(0), k_tokens = k.size(0), dim = q.size(2);
    if (dim <= 0) refuse("dim is positive");
    const int64_t longest = a[5] == Py_None ? tokens : whole(a[5]);
    const int64_t sequences = sequences_of(offsets, tokens, longest);
    int64_t context = k_tokens;
    if (!k_offsets && offsets) {
      if (k_tokens != tokens) refuse("without k_offsets, there are as many keys as queries");
      context = longest;
    } else if (!k_offsets && sequences) {
      if (k_tokens % sequences) refuse("without offsets, sequences divide the keys");
      context = k_tokens / sequences;
    }
    if (a[6] != Py_None) {
      const int64_t given = whole(a[6]);
      if (!k_offsets && !offsets && sequences && given != context) refuse("without offsets, max_context is k_tokens / sequences");
      context = given;
    }
    r.sequences = u32(sequences, "sequences"), r.max_tokens = u32(longest, "max_tokens"), r.max_context = u32(context, "max_context");
    r.offsets = ints<const int32_t*>(offsets, sequences + 1, q, "offsets");
    r.k_offsets = ints<const int32_t*>(k_offsets, sequences + 1, q, "k_offsets");
    r.status = ints<uint32_t*>(status, 1, q, "status");
    const at::Tensor o = make(out, q.sizes(), q, "out is like q");
    row(q, "q"), row(k, "k"), row(v, "v"), row(o, "out");
    apart(out, q, "q"), apart(out, k, "k"), apart(out, v, "v");
    if (offsets) apart(out, *offsets, "offsets");
    if (k_offsets) apart(out, *k_offsets, "k_offsets");
    r.tokens = u32(tokens, "tokens"), r.k_tokens = u32(k_tokens, "k_tokens");
    r.heads = u32(q.size(1), "heads"), r.kv_heads = u32(k.size(1), "kv_heads"), r.dim = u32(dim, "dim");
    r.scale = (float)(a[7] == Py_None ? 1.0 / sqrt((double)dim) : number(a[7]));
    r.q = q.data_ptr(), r.k = k.data_ptr(), r.v = v.data_ptr(), r.o = o.data_ptr();
    r.q_token = q.stride(0), r.q_head = q.stride(1), r.k_token = k.stride(0), r.k_head = k.stride(1);
    r.v_token = v.stride(0), r.v_head = v.stride(1), r.o_token = o.stride(0), r.o_head = o.stride(1);
    call("fr_hip_prompt_attend", q, r, fr_hip_prompt_workspace, fr_hip_prompt_attend);
    written(out), written(status);
    return THPVariable_Wrap(o);
  });
}

// cache q tree table lengths offsets max_tokens scale max_context out status
PyObject* kv_attend_tree(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    fr_hip_kv_tree r = {};
    const at::Tensor& cache = cache_of(a[0], &r.cache);
    const at::Tensor &q = *tensor(a[1], "q"), &tree = *tensor(a[2], "tree"), &table = *tensor(a[3], "table");
    const at::Tensor &lengths = *tensor(a[4], "lengths"), *offsets = tensor(a[5], "offsets", true);
    const at::Tensor *out = tensor(a[9], "out", true), *status = tensor(a[10], "status", true);
    r.type = type_of(q, "q");
    if (q.device() != cache.device()) refuse("q and the cache are on one GPU");
    if (q.dim() != 3 || q.size(2) != r.cache.dim) refuse("q is [tokens, heads, dim]");
    const int64_t tokens = q.size(0);
    if (tree.dim() != 1 || tree.size(0) != tokens || !plain(tree, at::kLong, q)) refuse("tree is a contiguous int64 [tokens] on the GPU");
    if (table.dim() != 2 || table.scalar_type() != at::kInt || table.device() != q.device() ||
        (table.stride(1) != 1 && table.size(1) > 1))
      refuse("table is an int32 matrix");
    const int64_t sequences = table.size(0), per = table.size(1);
    int64_t longest = 64;
    if (!offsets) {
      if (sequences ? tokens % sequences : tokens) refuse("without offsets, q has as many drafts of every sequence");
      longest = sequences ? tokens / sequences : 0;
    }
    if (a[6] != Py_None) {
      const int64_t given = whole(a[6]);
      if (!offsets && given != longest) refuse("without offsets, max_tokens is the drafts of a sequence");
      longest = given;
    }
    const int64_t most = per * r.cache.page, context = a[8] == Py_None ? most : whole(a[8]);
    if (context < 0 || context > most) refuse("max_context is within a table row's pages");
    const at::Tensor o = make(out, q.sizes(), q, "out is like q");
    r.offsets = ints<const int32_t*>(offsets, sequences + 1, q, "offsets");
    r.length = ints<const int32_t*>(&lengths, sequences, q, "lengths");
    r.status = ints<uint32_t*>(status, 1, q, "status");
    row(q, "q"), row(o, "out");
    apart(out, q, "q"), apart(out, tree, "tree"), apart(out, table, "table"), apart(out, lengths, "lengths");
    if (offsets) apart(out, *offsets, "offsets");
    for (int i = 0; i < 4; ++i) apart(out, THPVariable_Unpack(PyTuple_GET_ITEM(a[0], i)), "the cache");
    if (!sequences || !tokens) return THPVariable_Wrap(o);
    r.sequences = u32(sequences, "sequences"), r.tokens = u32(tokens, "tokens"), r.max_tokens = u32(longest, "max_tokens");
    r.heads = u32(q.size(1), "heads"), r.max_context = u32(context, "max_context");
    r.table_stride = u32(sequences == 1 ? std::max(table.stride(0), per) : table.stride(0), "table's stride");
    r.scale = (float)(a[7] == Py_None ? 1.0 / sqrt((double)r.cache.dim) : number(a[7]));
    r.q = q.data_ptr(), r.o = o.data_ptr(), r.tree = static_cast<const int64_t*>(tree.data_ptr());
    r.table = static_cast<const int32_t*>(table.data_ptr());
    r.q_token = q.stride(0), r.q_head = q.stride(1), r.o_token = o.stride(0), r.o_head = o.stride(1);
    call("fr_hip_kv_attend_tree", q, r, fr_hip_tree_workspace, fr_hip_kv_attend_tree);
    written(out), written(status);
    return THPVariable_Wrap(o);
  });
}

// What moves and copies have in common: cache source target status.
template <typename R> void places_of(R* r, Args a, int64_t n, const at::Tensor& cache, const at::Tensor* status) {
  const at::Tensor &source = *tensor(a[1], "source"), &target = *tensor(a[2], "target");
  r->source = ints<const int32_t*>(&source, n, cache, "source");
  r->target = ints<const int32_t*>(&target, n, cache, "target");
  if (target.sizes() != source.sizes()) refuse("source and target have one shape");
  r->status = ints<uint32_t*>(status, 1, cache, "status");
}

// cache source target status
PyObject* kv_move(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    fr_hip_kv_moves r = {};
    const at::Tensor &cache = cache_of(a[0], &r.cache), &source = *tensor(a[1], "source");
    const at::Tensor* status = tensor(a[3], "status", true);
    if (source.dim() != 1 && source.dim() != 2) refuse("source is [groups, moves] or [moves]");
    places_of(&r, a, source.numel(), cache, status);
    r.groups = source.dim() == 2 ? u32(source.size(0), "groups") : 1, r.moves = u32(source.size(-1), "moves");
    call("fr_hip_kv_move", cache, [&](void* s) { return fr_hip_kv_move(&r, s); });
    for (int i = 0; i < 4; ++i) written(&THPVariable_Unpack(PyTuple_GET_ITEM(a[0], i)));
    written(status);
    Py_RETURN_NONE;
  });
}

// cache source target status
PyObject* kv_copy(PyObject*, Args a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    fr_hip_kv_copies r = {};
    const at::Tensor &cache = cache_of(a[0], &r.cache), &source = *tensor(a[1], "source");
    const at::Tensor* status = tensor(a[3], "status", true);
    if (source.dim() != 1) refuse("source is [count]");
    places_of(&r, a, source.numel(), cache, status);
    r.count = u32(source.numel(), "count");
    call("fr_hip_kv_copy", cache, [&](void* s) { return fr_hip_kv_copy(&r, s); });
    for (int i = 0; i < 4; ++i) written(&THPVariable_Unpack(PyTuple_GET_ITEM(a[0], i)));
    written(status);
    Py_RETURN_NONE;
  });
}

PyMethodDef methods[] = {{"rotary", fast<rotary>(), METH_FASTCALL, nullptr},
                         {"prompt_attend", fast<prompt_attend>(), METH_FASTCALL, nullptr},
                         {"kv_attend_tree", fast<kv_attend_tree>(), METH_FASTCALL, nullptr},
                         {"kv_move", fast<kv_move>(), METH_FASTCALL, nullptr},
                         {"kv_copy", fast<kv_copy>(), METH_FASTCALL, nullptr},
                         {"bind", fast<bind>(), METH_FASTCALL, "What opens the engine on a device, and what gives its current stream."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attention", "fronk_amd.dense's calls.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attention() { return PyModule_Create(&module); }
