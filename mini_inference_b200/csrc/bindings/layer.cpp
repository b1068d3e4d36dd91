// Tensors to the C ABI for a decoder layer's norms with rotation, positions on several axes and
// experts, compiled: as the speculative step's binding, and for its reason (called once a layer,
// a few microseconds on the GPU each). ops.py holds the signatures, defaults and documentation.
#include "common.h"

namespace {

// Contiguous [n, heads, d] at `offset` of a buffer that several outputs share: one allocation (half a
// microsecond of the host's time each).
Tensor piece(const Tensor& buffer, int64_t offset, int64_t n, int64_t heads, int64_t d) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(), buffer.dtype());
  impl->set_storage_offset(offset);
  impl->set_sizes_contiguous({n, heads, d});
  return Tensor(std::move(impl));
}

// (pool, layer, qkv, positions, inv_freq, num_q_heads, axes, q_weight, k_weight, eps, interleaved, attention_factor, q_out,
//  k_out, v_out, slot_mapping, status) -> (q, k, v)
PyObject* norm_rotary_append(PyObject*, PyObject* const* a, Py_ssize_t) {
  HANDLE_TH_ERRORS
  try {
    const pkv_pool& pool = *handle<pkv_pool>(a[0]);
    const Tensor& qkv = tensor(a[2]);
    Call call("norm_rotary_append", qkv);
    check_pool_type(call, pool, qkv);
    const int64_t hq = integer32(a[5]), hkv = pool.num_kv_heads, d = pool.head_dim;
    if (qkv.dim() != 2 || qkv.size(1) != (hq + 2 * hkv) * d || qkv.stride(1) != 1)
      call.refuse("qkv must be [N, (Hq + 2 Hkv) * head_dim] with a contiguous last dimension");
    const int64_t n = qkv.size(0);
    const Tensor& positions = call.flat(a[3], at::kLong, "positions");
    const bool several = positions.dim() == 2;
    if (positions.dim() < 1 || positions.dim() > 2 || positions.size(positions.dim() - 1) != n)
      call.refuse("positions must be [N] or [axes, N]");
    const Tensor& freq = call.flat(a[4], at::kDouble, "inv_freq");
    const int32_t* axes = nullptr;
    if (given(a[6])) {
      axes = call.i32(a[6], "axes", freq.numel());
      if (tensor(a[6]).numel() != freq.numel()) call.refuse("axes must have one entry per frequency");
    }
    if (several && !axes) call.refuse("positions on several axes need axes, each pair's");
    auto weight = [&](PyObject* o, const char* what) -> const void* {
      if (!given(o)) return nullptr;
      const Tensor& t = call.flat(o, qkv.scalar_type(), what);
      if (t.numel() != d) call.refuse(std::string(what) + " must have head_dim elements");
      return t.data_ptr();
    };
    const void *qw = weight(a[7], "q_weight"), *kw = weight(a[8], "k_weight");
    if (!qw != !kw) call.refuse("q_weight and k_weight go together");
    const int64_t* slots = given(a[15]) ? call.i64(a[15], "slot_mapping", n) : nullptr;
    struct Output {
      Tensor t;
      void* at = nullptr;
      int64_t row = 0, head = 0;
    };
    const bool own[3] = {!given(a[12]) || a[12] == Py_True, a[13] == Py_True, a[14] == Py_True};
    const int64_t heads_of[3] = {hq, hkv, hkv};
    Tensor buffer;
    int64_t total = 0, at = 0;
    for (int i = 0; i < 3; ++i) total += own[i] ? (n * heads_of[i] * d + 63) / 64 * 64 : 0;
    if (own[0] + own[1] + own[2] > 1) buffer = fresh({total}, qkv);
    auto output = [&](PyObject* o, int64_t heads, bool always) {
      Output x;
      if (o == Py_True || (always && !given(o))) {
        x.t = buffer.defined() ? piece(buffer, at, n, heads, d) : fresh({n, heads, d}, qkv);
        at += (n * heads * d + 63) / 64 * 64;
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
    const Output q = output(a[12], hq, true), k = output(a[13], hkv, false), v = output(a[14], hkv, false);
    const int status = pkv_norm_rotary_append(
        &pool, integer32(a[1]), qkv.data_ptr(), n > 1 ? qkv.stride(0) : qkv.size(1), n, (int32_t)hq,
        positions.data_ptr<int64_t>(), n, axes, several ? (int32_t)positions.size(0) : 1, freq.data_ptr<double>(),
        (int32_t)(2 * freq.numel()), PyObject_IsTrue(a[10]), (float)number(a[11]), qw, kw, (float)number(a[9]), q.at, q.row,
        q.head, k.at, k.row, k.head, v.at, v.row, v.head, slots, call.status(a[16]), call.stream);
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

// (positions, media, media_counts, seq_rows, cu_seqlens, out, status) -> out
PyObject* media_positions(PyObject*, PyObject* const* a, Py_ssize_t) {
  HANDLE_TH_ERRORS
  try {
    const Tensor& positions = tensor(a[0]);
    Call call("media_positions", positions);
    const int64_t n = positions.numel();
    const int64_t* pos = call.i64(a[0], "positions", n);
    const Tensor& media = call.flat(a[1], at::kInt, "media");
    if (media.dim() != 3 || media.size(2) != 5) call.refuse("media must be [rows, spans, 5]");
    const int64_t rows = media.size(0);
    const int32_t* counts = call.i32(a[2], "media_counts", rows);
    int64_t seqs = n;
    const int32_t *cu = nullptr, *seq_rows = nullptr;
    if (given(a[4])) {
      seqs = tensor(a[4]).numel() - 1;
      if (seqs < 0) call.refuse("cu_seqlens must be [B + 1]");
      cu = call.i32(a[4], "cu_seqlens", seqs + 1);
    }
    if (given(a[3])) seq_rows = call.i32(a[3], "seq_rows", seqs);
    else if (rows < seqs) call.refuse("media needs a row for each sequence");
    Tensor out;
    if (given(a[5])) {
      out = tensor(a[5]);
      if (out.dim() != 2 || out.size(0) != 3 || out.size(1) != n || out.scalar_type() != at::kLong ||
          (n > 1 && out.stride(1) != 1))
        call.refuse("out must be int64 [3, N], last dimension contiguous");
      call.here(out);
    } else {
      out = fresh({3, n}, positions);
    }
    if (rows > 0x7fffffff || media.size(1) > 0x7fffffff || seqs > 0x7fffffff) call.refuse("a count is past 32 bits");
    const int status = pkv_media_positions(pos, n, cu, (int32_t)seqs, seq_rows, media.data_ptr<int32_t>(), counts,
                                           (int32_t)rows, (int32_t)media.size(1), out.data_ptr<int64_t>(), out.stride(0),
                                           call.status(a[6]), call.stream);
    return status == PKV_OK ? wrap(out) : PyLong_FromLong(status);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// (x, router, gate_up, down, top_k, renormalize, workspace, out, status) -> out
PyObject* expert_mlp(PyObject*, PyObject* const* a, Py_ssize_t) {
  HANDLE_TH_ERRORS
  try {
    const Tensor& x0 = tensor(a[0]);
    Call call("expert_mlp", x0);
    const at::ScalarType type = x0.scalar_type();
    if (type != at::kHalf && type != at::kBFloat16) {
      PyErr_Format(PyExc_NotImplementedError, "expert_mlp takes float16 or bfloat16, not %s", at::toString(type));
      throw python_error();
    }
    if (x0.dim() < 1) call.refuse("x must be [..., hidden]");
    const int64_t hidden = x0.size(-1);
    const Tensor &router = call.flat(a[1], type, "router"), &gate_up = call.flat(a[2], type, "gate_up"),
                 &down = call.flat(a[3], type, "down");
    if (router.dim() != 2 || router.size(1) != hidden) call.refuse("router must be [experts, hidden]");
    const int64_t experts = router.size(0);
    if (down.dim() != 3 || down.size(0) != experts || down.size(1) != hidden)
      call.refuse("down must be [experts, hidden, intermediate]");
    const int64_t inter = down.size(2);
    if (gate_up.dim() != 3 || gate_up.size(0) != experts || gate_up.size(1) != 2 * inter || gate_up.size(2) != hidden)
      call.refuse("gate_up must be [experts, 2 * intermediate, hidden]");
    if (experts > 0x7fffffff || hidden > 0x7fffffff || inter > 0x7fffffff) call.refuse("a size is past 32 bits");
    Tensor x = x0.dim() == 2 ? x0 : x0.reshape({-1, hidden});
    const int64_t n = x.size(0);
    if (n > 0 && (x.stride(1) != 1 || (n > 1 && (x.stride(0) < hidden || x.stride(0) % 8)) ||
                  (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15)))
      x = x.clone(at::MemoryFormat::Contiguous);
    const Tensor& ws = tensor(a[6]);
    call.here(ws);
    if (!ws.is_contiguous()) call.refuse("workspace must be contiguous");
    Tensor out;
    if (given(a[7])) {
      out = tensor(a[7]);
      if (out.sizes() != x0.sizes() || out.scalar_type() != type || !out.is_contiguous())
        call.refuse("out must be contiguous and match x");
      call.here(out);
    } else {
      out = fresh(x0.sizes(), x0);
    }
    const int status = pkv_expert_mlp(type == at::kHalf ? PKV_F16 : PKV_BF16, x.data_ptr(), n > 1 ? x.stride(0) : hidden, n,
                                      (int32_t)hidden, (int32_t)inter, (int32_t)experts, integer32(a[4]),
                                      PyObject_IsTrue(a[5]), router.data_ptr(), gate_up.data_ptr(), down.data_ptr(),
                                      out.data_ptr(), hidden, ws.data_ptr(), (int64_t)ws.nbytes(), call.status(a[8]),
                                      call.stream);
    return status == PKV_OK ? wrap(out) : PyLong_FromLong(status);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {method<norm_rotary_append, 17>("norm_rotary_append"),
                         method<media_positions, 7>("media_positions"),
                         method<expert_mlp, 9>("expert_mlp"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_layer", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layer() { return PyModule_Create(&module); }
