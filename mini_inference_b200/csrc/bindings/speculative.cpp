// Tensors to the C ABI for the speculative decoding step, compiled.
//
// A step calls these once or more per layer and the GPU takes a few microseconds a call,
// about what reading thirty tensor attributes from Python and converting thirty arguments
// through ctypes take. Each function checks its tensors, allocates the outputs that were not
// given and calls the library on the tensors' device and its current stream; ops.py holds the
// signatures, defaults and documentation. The result is the outputs, or an int: the status
// that the library refused the call with.
#include "common.h"

namespace {

// (tables, lengths, new_tokens, held, free_blocks, free_head, block_size, cu_seqlens, context_lens, positions,
//  slot_mapping, held_out, free_head_out, status)
PyObject* extend_tables(PyObject*, PyObject* const* a, Py_ssize_t) {
  HANDLE_TH_ERRORS
  try {
    const Tensor& lengths = tensor(a[1]);
    Call call("extend_tables", lengths);
    const int64_t batch = lengths.numel();
    const int32_t* len = call.i32(a[1], "lengths", batch);
    auto per_request = [&](PyObject* o, const char* what) {
      if (tensor(o).numel() != batch) call.refuse(std::string(what) + " must have one entry per request");
      return call.i32(o, what, batch);
    };
    const int32_t *fresh = per_request(a[2], "new_tokens"), *held = per_request(a[3], "held");
    const Tensor& free_blocks = call.flat(a[4], at::kInt, "free_blocks");
    const int32_t* head = call.i32(a[5], "free_head", 1);
    int32_t *cu = call.i32(a[7], "cu_seqlens", batch + 1), *ctx = call.i32(a[8], "context_lens", batch);
    int64_t total = 0x7fffffff;
    if (given(a[9])) total = tensor(a[9]).numel();
    else if (given(a[10])) total = tensor(a[10]).numel();
    int64_t* positions = given(a[9]) ? call.i64(a[9], "positions", total) : nullptr;
    int64_t* slots = given(a[10]) ? call.i64(a[10], "slot_mapping", total) : nullptr;
    int32_t* held_out = call.i32(given(a[11]) ? a[11] : a[3], "held_out", batch);
    int32_t* head_out = call.i32(given(a[12]) ? a[12] : a[5], "free_head_out", 1);
    return status_or_none(pkv_extend_tables(handle<pkv_tables>(a[0]), (int32_t)batch, len, fresh, held,
                                            free_blocks.data_ptr<int32_t>(), free_blocks.numel(), head, integer32(a[6]), cu,
                                            ctx, positions, slots, total, held_out, head_out, call.status(a[13]),
                                            call.stream));
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// (parents, cu_nodes, context_lens, mask, positions, status)
PyObject* build_tree_metadata(PyObject*, PyObject* const* a, Py_ssize_t) {
  HANDLE_TH_ERRORS
  try {
    const Tensor& parents = tensor(a[0]);
    Call call("build_tree_metadata", parents);
    const int64_t n = parents.numel(), batch = tensor(a[1]).numel() - 1;
    const Tensor& mask = call.flat(a[3], at::kLong, "mask");
    if (batch < 0 || mask.dim() != 2 || mask.size(0) != n) call.refuse("cu_nodes must be [B + 1] and mask [N, W]");
    return status_or_none(pkv_build_tree_metadata(
        call.i32(a[0], "parents", n), call.i32(a[1], "cu_nodes", batch + 1), (int32_t)batch,
        call.i32(a[2], "context_lens", batch), n, mask.data_ptr<int64_t>(), (int32_t)mask.size(1),
        call.i64(a[4], "positions", n), call.status(a[5]), call.stream));
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// (pool, layer, qkv, positions, inv_freq, num_q_heads, interleaved, attention_factor, q_out, k_out, v_out,
//  slot_mapping, status) -> (q, k, v)
PyObject* rotary_append(PyObject*, PyObject* const* a, Py_ssize_t) {
  HANDLE_TH_ERRORS
  try {
    const pkv_pool& pool = *handle<pkv_pool>(a[0]);
    const Tensor& qkv = tensor(a[2]);
    Call call("rotary_append", qkv);
    check_pool_type(call, pool, qkv);
    const int64_t hq = integer32(a[5]), hkv = pool.num_kv_heads, d = pool.head_dim;
    if (qkv.dim() != 2 || qkv.size(1) != (hq + 2 * hkv) * d || qkv.stride(1) != 1)
      call.refuse("qkv must be [N, (Hq + 2 Hkv) * head_dim] with a contiguous last dimension");
    const int64_t n = qkv.size(0);
    const int64_t* positions = call.i64(a[3], "positions", n);
    const Tensor& freq = call.flat(a[4], at::kDouble, "inv_freq");
    const int64_t* slots = given(a[11]) ? call.i64(a[11], "slot_mapping", n) : nullptr;
    struct Output {
      Tensor t;
      void* at = nullptr;
      int64_t row = 0, head = 0;
    };
    auto output = [&](PyObject* o, int64_t heads, bool always) {
      Output x;
      if (o == Py_True || (always && !given(o))) {
        x.t = fresh({n, heads, d}, qkv);
      } else if (given(o) && o != Py_False) {
        x.t = tensor(o);
        if (x.t.dim() != 3 || x.t.size(0) != n || x.t.size(1) != heads || x.t.size(2) != d ||
            x.t.scalar_type() != qkv.scalar_type() || x.t.stride(2) != 1)
          call.refuse("outputs must be [N, heads, head_dim] like qkv, last dimension contiguous");
        call.here(x.t);
      }
      if (x.t.defined()) x.at = x.t.data_ptr(), x.row = x.t.stride(0), x.head = x.t.stride(1);
      return x;
    };
    const Output q = output(a[8], hq, true), k = output(a[9], hkv, false), v = output(a[10], hkv, false);
    const int status = pkv_rotary_append(&pool, integer32(a[1]), qkv.data_ptr(), qkv.stride(0), n, (int32_t)hq, positions,
                                         freq.data_ptr<double>(), (int32_t)(2 * freq.numel()), PyObject_IsTrue(a[6]),
                                         (float)number(a[7]), q.at, q.row, q.head, k.at, k.row, k.head, v.at, v.row, v.head,
                                         slots, call.status(a[12]), call.stream);
    if (status != PKV_OK) return PyLong_FromLong(status);
    PyObject* out = PyTuple_New(3);
    if (!out) return nullptr;
    int i = 0;
    for (const Output* x : {&q, &k, &v}) PyTuple_SET_ITEM(out, i++, x->t.defined() ? wrap(x->t) : Py_NewRef(Py_None));
    return out;
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// Rows and heads that start on 16 bytes: the tensor itself, or a contiguous copy of it.
Tensor rows16(const Tensor& t) {
  const int64_t row = t.stride(0), head = t.stride(1);
  const bool ok = t.stride(2) == 1 && row >= (t.size(0) > 1) && head >= (t.size(1) > 1) && ((row | head) & 7) == 0 &&
                  (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// (pool, layer, tables, q, k_nodes, v_nodes, cu_nodes, context_lens, mask, max_nodes, workspace, out, scale, status)
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t) {
  HANDLE_TH_ERRORS
  try {
    const pkv_pool& pool = *handle<pkv_pool>(a[0]);
    const Tensor &q0 = tensor(a[3]), &k0 = tensor(a[4]), &v0 = tensor(a[5]);
    Call call("tree_attention", q0);
    check_pool_type(call, pool, q0);
    const int64_t hkv = pool.num_kv_heads, d = pool.head_dim;
    if (q0.dim() != 3 || q0.size(2) != d) call.refuse("q must be [N, heads, head_dim]");
    const int64_t n = q0.size(0), hq = q0.size(1);
    for (const Tensor* t : {&k0, &v0}) {
      if (t->dim() != 3 || t->size(0) != n || t->size(1) != hkv || t->size(2) != d || t->scalar_type() != q0.scalar_type())
        call.refuse("k_nodes and v_nodes must be [N, kv_heads, head_dim] of q's dtype");
      call.here(*t);
    }
    const int64_t batch = tensor(a[6]).numel() - 1;
    const Tensor& mask = call.flat(a[8], at::kLong, "mask");
    if (batch < 0 || mask.dim() != 2 || mask.size(0) != n) call.refuse("cu_nodes must be [B + 1] and mask [N, W]");
    const int32_t *cu = call.i32(a[6], "cu_nodes", batch + 1), *ctx = call.i32(a[7], "context_lens", batch);
    const Tensor& ws = tensor(a[10]);
    call.here(ws);
    const Tensor q = rows16(q0), k = rows16(k0), v = rows16(v0);
    Tensor out;
    if (given(a[11])) {
      out = tensor(a[11]);
      if (out.dim() != 3 || out.size(0) != n || out.size(1) != hq || out.size(2) != d ||
          out.scalar_type() != q.scalar_type() || out.stride(2) != 1)
        call.refuse("out must match q, last dimension contiguous");
      call.here(out);
    } else {
      out = fresh({n, hq, d}, q);
    }
    const int status = pkv_tree_attention(
        &pool, integer32(a[1]), handle<pkv_tables>(a[2]), (int32_t)batch, cu, ctx, integer32(a[9]), n, (int32_t)hq,
        out.data_ptr(), out.stride(0), out.stride(1), q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0),
        k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), mask.data_ptr<int64_t>(), (int32_t)mask.size(1),
        (float)number(a[12]), ws.data_ptr(), (int64_t)ws.nbytes(), call.status(a[13]), call.stream);
    return status == PKV_OK ? wrap(out) : PyLong_FromLong(status);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// (pool, tables, parents, cu_nodes, draft_tokens, target_tokens, k_nodes, v_nodes, context_lens, counts, path, tokens,
//  lengths_out, status)
PyObject* accept_tree(PyObject*, PyObject* const* a, Py_ssize_t) {
  HANDLE_TH_ERRORS
  try {
    const pkv_pool& pool = *handle<pkv_pool>(a[0]);
    const Tensor& parents = tensor(a[2]);
    Call call("accept_tree", parents);
    const int64_t n = parents.numel(), batch = tensor(a[3]).numel() - 1;
    const Tensor& path = call.flat(a[10], at::kInt, "path");
    const Tensor& tokens = call.flat(a[11], at::kLong, "tokens");
    if (batch < 0 || path.dim() != 2 || path.sizes() != tokens.sizes() || path.size(0) < batch)
      call.refuse("cu_nodes must be [B + 1], path and tokens [B, W]");
    const Tensor &k = tensor(a[6]), &v = tensor(a[7]);
    for (const Tensor* t : {&k, &v}) {
      if (t->dim() != 4 || t->size(0) != pool.num_layers || t->size(1) != n || t->size(2) != pool.num_kv_heads ||
          t->size(3) != pool.head_dim || t->scalar_type() != pool_type(pool) || t->stride(3) != 1)
        call.refuse("k_nodes and v_nodes must be [layers, N, kv_heads, head_dim] of the pool's dtype");
      call.here(*t);
    }
    return status_or_none(pkv_accept_tree(
        &pool, handle<pkv_tables>(a[1]), (int32_t)batch, call.i32(a[2], "parents", n),
        call.i32(a[3], "cu_nodes", batch + 1), n, call.i64(a[4], "draft_tokens", n), call.i64(a[5], "target_tokens", n),
        k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2),
        call.i32(a[8], "context_lens", batch), call.i32(a[9], "counts", batch), path.data_ptr<int32_t>(),
        tokens.data_ptr<int64_t>(), (int32_t)path.size(1), call.i32(given(a[12]) ? a[12] : a[8], "lengths_out", batch),
        call.status(a[13]), call.stream));
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {method<extend_tables, 14>("extend_tables"),
                         method<build_tree_metadata, 6>("build_tree_metadata"),
                         method<rotary_append, 13>("rotary_append"),
                         method<tree_attention, 14>("tree_attention"),
                         method<accept_tree, 14>("accept_tree"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_speculative", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__speculative() { return PyModule_Create(&module); }
