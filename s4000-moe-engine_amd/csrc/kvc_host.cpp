// Native host path of the decode step's calls.
//
// A decode step at a small batch is shorter on the GPU (14-20 us) than its
// Python call was on the host (20-31 us): the argument checks, the output and
// workspace allocations and a 34-argument ctypes call.  This extension does
// the same work for the form such a step has (exact torch.Tensor arguments on
// one GPU, bf16, the strides and index types the launch reads as they are)
// and returns None, having done nothing, for anything else: the Python
// function then checks, converts or raises as it always did.  Nothing is
// kept between calls.  Measured: one row of 333 tokens through norm, rotary,
// append and attention (16 q / 8 kv heads) 30 -> 16-18 us a pass, a decode
// step of 11 rows of 97-1501 tokens 20.0 -> 14.7 us (both now GPU-bound).  The
// same holds for the shaped-score, tree, multi-axis rotary and commit calls.
#include <Python.h>

#include <ATen/ATen.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <algorithm>
#include <cstdlib>
#include <cstring>

#include "kvc.h"

namespace {

decltype(&kvc_last_error) p_last_error;
decltype(&kvc_paged_decode_workspace_bytes) p_workspace;
decltype(&kvc_paged_decode) p_decode;
decltype(&kvc_paged_decode_append) p_decode_append;
decltype(&kvc_qk_norm_rope_store) p_rope;
decltype(&kvc_scored_workspace_bytes) p_scored_workspace;
decltype(&kvc_scored_attention) p_scored;
decltype(&kvc_tree_workspace_bytes) p_tree_workspace;
decltype(&kvc_tree_attention) p_tree;
decltype(&kvc_qk_norm_mrope_store) p_mrope;
decltype(&kvc_commit_rows) p_commit;

// The tensor behind an exact torch.Tensor / Parameter, else null.
const at::Tensor* tensor(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

// A plain dense-storage tensor of `type` on `like`'s GPU with `dim` dims.
bool plain(const at::Tensor* t, at::ScalarType type, int64_t dim, const at::Tensor& like) {
  return t != nullptr && t->defined() && t->is_cuda() && t->layout() == at::kStrided &&
         t->scalar_type() == type && t->dim() == dim && t->device() == like.device();
}

bool is_index(const at::Tensor* t, int64_t n, const at::Tensor& like, int* bytes) {
  if (t == nullptr || !t->defined() || t->dim() != 1 || t->numel() != n || !t->is_contiguous())
    return false;
  *bytes = t->scalar_type() == at::kLong ? 8 : 4;
  return plain(t, *bytes == 8 ? at::kLong : at::kInt, 1, like);
}

// [pages, page, kv heads, 128] pools of a decode over q [batch, heads, 128].
bool decode_shapes(const at::Tensor& q, const at::Tensor* kc, const at::Tensor* vc,
                   const at::Tensor* bt, const at::Tensor* lens) {
  if (!plain(kc, at::kBFloat16, 4, q) || !plain(vc, at::kBFloat16, 4, q) ||
      !plain(bt, at::kInt, 2, q) || !plain(lens, at::kInt, 1, q))
    return false;
  const int64_t page = kc->size(1), kvh = kc->size(2);
  return q.size(0) > 0 && q.size(2) == 128 && q.stride(2) == 1 && kc->sizes() == vc->sizes() &&
         kc->size(3) == 128 && kvh > 0 && q.size(1) > 0 && q.size(1) % kvh == 0 && page > 0 &&
         page % 32 == 0 && kc->is_contiguous() && vc->is_contiguous() && bt->stride(1) == 1 &&
         bt->size(0) >= q.size(0) && bt->size(1) > 0 && lens->is_contiguous() &&
         lens->numel() >= q.size(0);
}

at::Tensor output_like(const at::Tensor& q) {
  at::Tensor out = at::empty_like(q);
  return out.stride(2) == 1 ? out : at::empty(q.sizes(), q.options());
}

// nullptr with the exception _native.call raises for the status.
PyObject* fail(int rc, const char* what) {
  const char* msg = p_last_error();
  PyObject* type = rc == KVC_ERR_ASSERT ? PyExc_AssertionError
                   : rc == KVC_ERR_RUNTIME || (rc != KVC_ERR_VALUE && rc != KVC_ERR_WORKSPACE)
                       ? PyExc_RuntimeError
                       : PyExc_ValueError;
  if (msg != nullptr && *msg != '\0') {
    PyErr_SetString(type, msg);
  } else {
    PyErr_Format(type, "%s failed with status %d", what, rc);
  }
  return nullptr;
}

// A torch C++ exception before the launch (an allocation that fails, a tensor
// without storage): the Python path takes the call and raises its own error
// (torch.OutOfMemoryError, not a plain RuntimeError).
PyObject* declined() {
  PyErr_Clear();
  Py_RETURN_NONE;
}

// Every torch call that can throw (data_ptr() of a tensor without storage
// among them) comes before a launch, with the interpreter lock held; Unlocked
// covers the library call alone.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// A tensor of a call as the library takes it.
struct Rows {
  void* p = nullptr;
  int64_t s0 = 0, s1 = 0;
};
Rows rows(const at::Tensor* t) {
  return t != nullptr && t->defined() ? Rows{t->data_ptr(), t->stride(0), t->stride(1)} : Rows{};
}
void* address(const at::Tensor* t) { return t != nullptr ? t->data_ptr() : nullptr; }

// A new reference to `t` after a launch: an error here is raised, the call is
// not made again.
PyObject* wrap(at::Tensor&& t) {
  try {
    return THPVariable_Wrap(std::move(t));
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// decode(out or None, q, k_cache, v_cache, block_tables, context_lens, scale,
//        stream, key or None, value, slot_mapping)
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11) {
    PyErr_SetString(PyExc_TypeError, "decode takes 11 arguments");
    return nullptr;
  }
  at::Tensor out, ws;
  Rows q_r, k_r, v_r, out_r;
  void *slots_p, *kc_p, *vc_p, *bt_p, *lens_p, *ws_p, *stream;
  int64_t batch, heads, kvh, pages, page, bt_stride, blocks;
  size_t bytes;
  float scale;
  int sb = 4;
  const bool append = a[8] != Py_None;
  try {
    const at::Tensor* q = tensor(a[1]);
    if (q == nullptr || !q->defined() || !plain(q, at::kBFloat16, 3, *q)) Py_RETURN_NONE;
    const at::Tensor *kc = tensor(a[2]), *vc = tensor(a[3]), *bt = tensor(a[4]),
                     *lens = tensor(a[5]);
    if (!decode_shapes(*q, kc, vc, bt, lens) || !PyFloat_CheckExact(a[6])) Py_RETURN_NONE;
    batch = q->size(0), heads = q->size(1), kvh = kc->size(2);
    pages = kc->size(0), page = kc->size(1), bt_stride = bt->stride(0), blocks = bt->size(1);
    const at::Tensor *key = nullptr, *value = nullptr, *slots = nullptr;
    if (append) {
      key = tensor(a[8]);
      value = tensor(a[9]);
      slots = tensor(a[10]);
      const char* check = std::getenv("KVC_CHECK_APPEND");
      if (!plain(key, at::kBFloat16, 3, *q) || !plain(value, at::kBFloat16, 3, *q) ||
          key->sizes() != value->sizes() || key->size(0) != batch || key->size(1) != kvh ||
          key->size(2) != 128 || key->stride(2) != 1 || value->stride(2) != 1 ||
          !is_index(slots, batch, *q, &sb) || (check != nullptr && std::strcmp(check, "1") == 0))
        Py_RETURN_NONE;
    }
    if (a[0] != Py_None) {
      const at::Tensor* given = tensor(a[0]);
      if (!plain(given, at::kBFloat16, 3, *q) || given->sizes() != q->sizes() ||
          given->stride(2) != 1)
        Py_RETURN_NONE;
      out = *given;
    } else {
      out = output_like(*q);
    }
    stream = PyLong_AsVoidPtr(a[7]);
    if (PyErr_Occurred()) return nullptr;
    scale = float(PyFloat_AS_DOUBLE(a[6]));
    bytes = p_workspace(batch, heads, kvh, 128, page, blocks);
    if (bytes > 0) ws = at::empty({int64_t(bytes)}, q->options().dtype(at::kByte));
    ws_p = bytes > 0 ? ws.data_ptr() : nullptr;
    q_r = rows(q), k_r = rows(key), v_r = rows(value), out_r = rows(&out);
    slots_p = address(slots);
    kc_p = address(kc), vc_p = address(vc), bt_p = address(bt), lens_p = address(lens);
  } catch (const std::exception&) {
    return declined();
  }
  int rc;
  if (append) {
    Unlocked unlocked;
    rc = p_decode_append(q_r.p, q_r.s0, q_r.s1, k_r.p, k_r.s0, k_r.s1, v_r.p, v_r.s0, v_r.s1,
                         slots_p, sb, kc_p, vc_p, pages, page, kvh, 128,
                         static_cast<const int32_t*>(bt_p), bt_stride, blocks,
                         static_cast<const int32_t*>(lens_p), batch, heads, scale, out_r.p,
                         out_r.s0, out_r.s1, ws_p, bytes, stream);
  } else {
    Unlocked unlocked;
    rc = p_decode(q_r.p, q_r.s0, q_r.s1, kc_p, vc_p, pages, page, kvh, 128, KVC_KV_BF16, nullptr,
                  nullptr, nullptr, nullptr, nullptr, nullptr, 0,
                  static_cast<const int32_t*>(bt_p), bt_stride, blocks,
                  static_cast<const int32_t*>(lens_p), batch, heads, scale, out_r.p, out_r.s0,
                  out_r.s1, ws_p, bytes, stream);
  }
  if (rc != KVC_OK) return fail(rc, "paged_decode");
  if (a[0] != Py_None) {
    Py_INCREF(a[0]);
    return a[0];
  }
  return wrap(std::move(out));
}

// rope(q, k, v or None, positions, cos_sin, q_weight or None, k_weight or
//      None, eps, k_cache or None, v_cache, slot_mapping, return_k, stream)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13) {
    PyErr_SetString(PyExc_TypeError, "rope takes 13 arguments");
    return nullptr;
  }
  at::Tensor q_out, k_out;
  Rows q_r, k_r, v_r, qo_r, ko_r;
  void *pos_p, *cs_p, *qw_p, *kw_p, *kc_p, *vc_p, *slots_p, *stream;
  int64_t tokens, heads, kvh, max_position, num_slots = 0;
  int pb = 4, sb = 4;
  float eps;
  try {
    const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *pos = tensor(a[3]),
                     *cs = tensor(a[4]);
    if (q == nullptr || !q->defined() || !plain(q, at::kBFloat16, 3, *q) ||
        !plain(k, at::kBFloat16, 3, *q) || !plain(cs, at::kFloat, 2, *q))
      Py_RETURN_NONE;
    tokens = q->size(0), heads = q->size(1), kvh = k->size(1);
    if (tokens == 0 || q->size(2) != 128 || k->size(0) != tokens || k->size(2) != 128 ||
        kvh == 0 || heads == 0 || q->stride(2) != 1 || k->stride(2) != 1 || cs->size(1) != 128 ||
        !cs->is_contiguous() || !is_index(pos, tokens, *q, &pb) || !PyFloat_CheckExact(a[7]) ||
        (a[11] != Py_True && a[11] != Py_False))
      Py_RETURN_NONE;
    const at::Tensor* w[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; ++i) {
      if (a[5 + i] == Py_None) continue;
      w[i] = tensor(a[5 + i]);
      if (!plain(w[i], at::kBFloat16, 1, *q) || w[i]->size(0) != 128 || !w[i]->is_contiguous())
        Py_RETURN_NONE;
    }
    const at::Tensor* v = nullptr;
    if (a[2] != Py_None) {
      v = tensor(a[2]);
      if (!plain(v, at::kBFloat16, 3, *q) || v->sizes() != k->sizes() || v->stride(2) != 1)
        Py_RETURN_NONE;
    }
    const at::Tensor *kc = nullptr, *vc = nullptr, *slots = nullptr;
    if (a[8] != Py_None) {
      kc = tensor(a[8]);
      vc = tensor(a[9]);
      slots = tensor(a[10]);
      if (v == nullptr || !plain(kc, at::kBFloat16, 4, *q) || !plain(vc, at::kBFloat16, 4, *q) ||
          kc->sizes() != vc->sizes() || !kc->is_contiguous() || !vc->is_contiguous() ||
          !is_index(slots, tokens, *q, &sb))
        Py_RETURN_NONE;
      num_slots = kc->numel() / (kvh * 128);
    } else if (a[9] != Py_None) {
      Py_RETURN_NONE;  // a v pool alone is refused
    }
    stream = PyLong_AsVoidPtr(a[12]);
    if (PyErr_Occurred()) return nullptr;
    eps = float(PyFloat_AS_DOUBLE(a[7]));
    max_position = cs->size(0);
    q_out = at::empty({tokens, heads, 128}, q->options());
    if (a[11] == Py_True) k_out = at::empty({tokens, kvh, 128}, k->options());
    q_r = rows(q), k_r = rows(k), v_r = rows(v), qo_r = rows(&q_out), ko_r = rows(&k_out);
    pos_p = address(pos), cs_p = address(cs), qw_p = address(w[0]), kw_p = address(w[1]);
    kc_p = address(kc), vc_p = address(vc), slots_p = address(slots);
  } catch (const std::exception&) {
    return declined();
  }
  int rc;
  {
    Unlocked unlocked;
    rc = p_rope(q_r.p, q_r.s0, q_r.s1, k_r.p, k_r.s0, k_r.s1, v_r.p, v_r.s0, v_r.s1, tokens,
                heads, kvh, 128, pos_p, pb, qw_p, kw_p, eps, static_cast<const float*>(cs_p),
                max_position, qo_r.p, qo_r.s0, qo_r.s1, ko_r.p, ko_r.s0, ko_r.s1, kc_p, vc_p,
                num_slots, slots_p, sb, stream);
  }
  if (rc != KVC_OK) return fail(rc, "kvc_qk_norm_rope_store");
  PyObject* r = PyTuple_New(2);
  if (r == nullptr) return nullptr;
  PyObject* q_py = wrap(std::move(q_out));
  PyObject* k_py = nullptr;
  if (ko_r.p != nullptr) {
    k_py = wrap(std::move(k_out));
  } else {
    Py_INCREF(Py_None);
    k_py = Py_None;
  }
  PyTuple_SET_ITEM(r, 0, q_py);
  PyTuple_SET_ITEM(r, 1, k_py);
  if (q_py != nullptr && k_py != nullptr) return r;
  Py_DECREF(r);
  return nullptr;
}

// A vector of n int32 on like's GPU, as the launch reads it.
bool ints(const at::Tensor* t, int64_t n, const at::Tensor& like) {
  return plain(t, at::kInt, 1, like) && t->numel() == n && t->is_contiguous();
}

// Rows that the kernels read 16 bytes at a time.
bool rows16(const at::Tensor& t) {
  return t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// q [tokens, heads, 128] and, paged, its bf16 pools and tables.
bool shaped_shapes(const at::Tensor& q, const at::Tensor* kc, const at::Tensor* vc,
                   const at::Tensor* bt) {
  if (!plain(kc, at::kBFloat16, 4, q) || !plain(vc, at::kBFloat16, 4, q) ||
      !plain(bt, at::kInt, 2, q))
    return false;
  const int64_t page = kc->size(1), kvh = kc->size(2);
  return q.size(0) > 0 && q.size(2) == 128 && rows16(q) && kc->sizes() == vc->sizes() &&
         kc->size(3) == 128 && kvh > 0 && q.size(1) > 0 && q.size(1) % kvh == 0 && page > 0 &&
         page % 32 == 0 && kc->is_contiguous() && vc->is_contiguous() && bt->stride(1) == 1;
}

// softcap, alibi slopes or None, window, scale.
struct Shape {
  float cap, scale;
  const at::Tensor* slopes = nullptr;
  int64_t window;
};
bool shape_args(PyObject* cap, PyObject* slopes, PyObject* window, PyObject* scale,
                const at::Tensor& q, Shape& s) {
  if (!PyFloat_CheckExact(cap) || !PyLong_CheckExact(window) || !PyFloat_CheckExact(scale))
    return false;
  s.cap = float(PyFloat_AS_DOUBLE(cap));
  s.scale = float(PyFloat_AS_DOUBLE(scale));
  s.window = PyLong_AsLongLong(window);
  if (s.window == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  if (slopes == Py_None) return true;
  s.slopes = tensor(slopes);
  return plain(s.slopes, at::kFloat, 1, q) && s.slopes->numel() == q.size(1) &&
         s.slopes->is_contiguous();
}

// Entry i of a list of Python ints; false for anything else.
bool item(PyObject* list, Py_ssize_t i, int64_t* v) {
  PyObject* o = PyList_GET_ITEM(list, i);
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// scored(q, k_cache or None, v_cache, block_tables or None, num_decode_rows,
//        decode_context_lens, cu_seqlens_q or None, cu_seqlens_k,
//        cu_seqlens_q_list, cu_seqlens_k_list, k, v, softcap, alibi_slopes,
//        window, prefix_lens, scale, stream)
PyObject* scored(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 18) {
    PyErr_SetString(PyExc_TypeError, "scored takes 18 arguments");
    return nullptr;
  }
  at::Tensor out, ws;
  Rows q_r, out_r, k_r, v_r;
  void *kc_p = nullptr, *vc_p = nullptr, *bt_p = nullptr, *lens_p, *cuq_p, *cuk_p, *pre_p,
       *slopes_p, *ws_p, *stream;
  int64_t tokens, heads, kvh, pages = 0, page = 0, bt_stride = 0, blocks = 0, fresh = 0;
  int64_t decode_rows, prefill = 0, max_q = 0, last_q = 0, last_k = 0;
  size_t bytes;
  Shape sh;
  try {
    const at::Tensor* q = tensor(a[0]);
    if (q == nullptr || !q->defined() || !plain(q, at::kBFloat16, 3, *q) ||
        !PyLong_CheckExact(a[4]))
      Py_RETURN_NONE;
    tokens = q->size(0), heads = q->size(1);
    decode_rows = PyLong_AsLongLong(a[4]);
    if (decode_rows < 0 || decode_rows > tokens) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    const at::Tensor *lens = nullptr, *cu_q = nullptr, *cu_k = nullptr, *pre = nullptr;
    if (decode_rows > 0 && !ints(lens = tensor(a[5]), decode_rows, *q)) Py_RETURN_NONE;
    if (a[8] != Py_None) {
      if (!PyList_CheckExact(a[8]) || !PyList_CheckExact(a[9]) || PyList_GET_SIZE(a[8]) < 1 ||
          PyList_GET_SIZE(a[8]) != PyList_GET_SIZE(a[9]))
        Py_RETURN_NONE;
      prefill = PyList_GET_SIZE(a[8]) - 1;
      if (!item(a[8], 0, &last_q) || !item(a[9], 0, &last_k) || last_q != 0 || last_k != 0)
        Py_RETURN_NONE;
      for (int64_t i = 1; i <= prefill; ++i) {
        int64_t cq, ck;
        if (!item(a[8], i, &cq) || !item(a[9], i, &ck) || cq < last_q || ck < last_k ||
            (cq > last_q && ck - last_k < cq - last_q))
          Py_RETURN_NONE;
        max_q = std::max(max_q, cq - last_q);
        last_q = cq, last_k = ck;
      }
      if (prefill > 0 && (!ints(cu_q = tensor(a[6]), prefill + 1, *q) ||
                          !ints(cu_k = tensor(a[7]), prefill + 1, *q)))
        Py_RETURN_NONE;
    } else if (a[6] != Py_None) {
      Py_RETURN_NONE;
    }
    if (decode_rows + last_q != tokens) Py_RETURN_NONE;
    if (a[15] != Py_None && !ints(pre = tensor(a[15]), prefill, *q)) Py_RETURN_NONE;
    if (!shape_args(a[12], a[13], a[14], a[16], *q, sh)) Py_RETURN_NONE;
    if (a[3] != Py_None) {
      const at::Tensor *kc = tensor(a[1]), *vc = tensor(a[2]), *bt = tensor(a[3]);
      if (!shaped_shapes(*q, kc, vc, bt) || bt->size(0) < decode_rows + prefill) Py_RETURN_NONE;
      kvh = kc->size(2), pages = kc->size(0), page = kc->size(1);
      bt_stride = bt->stride(0), blocks = bt->size(1);
      kc_p = address(kc), vc_p = address(vc), bt_p = address(bt);
    } else {
      const at::Tensor *k = tensor(a[10]), *v = tensor(a[11]);
      if (decode_rows > 0 || !plain(k, at::kBFloat16, 3, *q) || !plain(v, at::kBFloat16, 3, *q) ||
          k->sizes() != v->sizes() || k->size(2) != 128 || k->size(1) == 0 || heads == 0 ||
          heads % k->size(1) != 0 || k->size(0) < last_k || tokens == 0 || q->size(2) != 128 ||
          !rows16(*q) || !rows16(*k) || !rows16(*v))
        Py_RETURN_NONE;
      kvh = k->size(1), fresh = k->size(0);
      k_r = rows(k), v_r = rows(v);
    }
    stream = PyLong_AsVoidPtr(a[17]);
    if (PyErr_Occurred()) return nullptr;
    out = at::empty({tokens, heads, 128}, q->options());
    bytes = p_scored_workspace(tokens, heads, kvh, decode_rows, prefill, max_q);
    if (bytes > 0) ws = at::empty({int64_t(bytes)}, q->options().dtype(at::kByte));
    ws_p = bytes > 0 ? ws.data_ptr() : nullptr;
    q_r = rows(q), out_r = rows(&out);
    lens_p = address(lens), cuq_p = address(cu_q), cuk_p = address(cu_k), pre_p = address(pre);
    slopes_p = address(sh.slopes);
  } catch (const std::exception&) {
    return declined();
  }
  int rc;
  {
    Unlocked unlocked;
    rc = p_scored(q_r.p, q_r.s0, q_r.s1, tokens, heads, kc_p, vc_p, pages, page, kvh, 128, k_r.p,
                  k_r.s0, k_r.s1, v_r.p, v_r.s0, v_r.s1, fresh, static_cast<int32_t*>(bt_p),
                  bt_stride, blocks, decode_rows, static_cast<int32_t*>(lens_p), prefill,
                  static_cast<int32_t*>(cuq_p), static_cast<int32_t*>(cuk_p), max_q,
                  static_cast<int32_t*>(pre_p), static_cast<float*>(slopes_p), sh.cap, sh.window,
                  sh.scale, out_r.p, out_r.s0, out_r.s1, ws_p, bytes, stream);
  }
  if (rc != KVC_OK) return fail(rc, "kvc_scored_attention");
  return wrap(std::move(out));
}

// tree(q, k_cache, v_cache, block_tables, context_lens, tree_mask, scale,
//      cu_seqlens_q or None, max_seqlen_q or None, softcap, alibi_slopes,
//      window, stream)
PyObject* tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13) {
    PyErr_SetString(PyExc_TypeError, "tree takes 13 arguments");
    return nullptr;
  }
  at::Tensor out, ws;
  Rows q_r, out_r;
  void *kc_p, *vc_p, *bt_p, *lens_p, *cuq_p, *mask_p, *slopes_p, *ws_p, *stream;
  int64_t tokens, heads, kvh, pages, page, bt_stride, blocks, batch, max_q, words;
  size_t bytes;
  Shape sh;
  try {
    const at::Tensor *q = tensor(a[0]), *kc = tensor(a[1]), *vc = tensor(a[2]),
                     *bt = tensor(a[3]), *lens = tensor(a[4]), *mask = tensor(a[5]);
    if (q == nullptr || !q->defined() || !plain(q, at::kBFloat16, 3, *q) ||
        !shaped_shapes(*q, kc, vc, bt) || !plain(mask, at::kLong, 2, *q))
      Py_RETURN_NONE;
    tokens = q->size(0), heads = q->size(1), kvh = kc->size(2), batch = bt->size(0);
    if (batch == 0 || !ints(lens, batch, *q) || mask->size(0) != tokens ||
        !mask->is_contiguous() || !shape_args(a[9], a[10], a[11], a[6], *q, sh))
      Py_RETURN_NONE;
    const at::Tensor* cu_q = nullptr;
    if (a[7] != Py_None) {
      if (!ints(cu_q = tensor(a[7]), batch + 1, *q) || !PyLong_CheckExact(a[8])) Py_RETURN_NONE;
      max_q = PyLong_AsLongLong(a[8]);
      if (max_q < 0) {
        PyErr_Clear();
        Py_RETURN_NONE;
      }
    } else {
      if (tokens % batch != 0) Py_RETURN_NONE;
      max_q = tokens / batch;
    }
    words = mask->size(1);
    if (words < (max_q + 63) / 64) Py_RETURN_NONE;
    stream = PyLong_AsVoidPtr(a[12]);
    if (PyErr_Occurred()) return nullptr;
    pages = kc->size(0), page = kc->size(1), bt_stride = bt->stride(0), blocks = bt->size(1);
    out = at::empty({tokens, heads, 128}, q->options());
    bytes = p_tree_workspace(tokens, heads, kvh, batch, max_q);
    if (bytes > 0) ws = at::empty({int64_t(bytes)}, q->options().dtype(at::kByte));
    ws_p = bytes > 0 ? ws.data_ptr() : nullptr;
    q_r = rows(q), out_r = rows(&out);
    kc_p = address(kc), vc_p = address(vc), bt_p = address(bt), lens_p = address(lens);
    cuq_p = address(cu_q), mask_p = address(mask), slopes_p = address(sh.slopes);
  } catch (const std::exception&) {
    return declined();
  }
  int rc;
  {
    Unlocked unlocked;
    rc = p_tree(q_r.p, q_r.s0, q_r.s1, tokens, heads, kc_p, vc_p, pages, page, kvh, 128,
                static_cast<int32_t*>(bt_p), bt_stride, blocks, batch,
                static_cast<int32_t*>(lens_p), static_cast<int32_t*>(cuq_p), max_q,
                static_cast<int64_t*>(mask_p), words, static_cast<float*>(slopes_p), sh.cap,
                sh.window, sh.scale, out_r.p, out_r.s0, out_r.s1, ws_p, bytes, stream);
  }
  if (rc != KVC_OK) return fail(rc, "kvc_tree_attention");
  return wrap(std::move(out));
}

// mrope(q, k, v or None, positions, cos_sin, pair_axes' address, axes,
//       q_weight or None, k_weight or None, eps, k_cache or None, v_cache,
//       slot_mapping, return_k, stream)
PyObject* mrope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 15) {
    PyErr_SetString(PyExc_TypeError, "mrope takes 15 arguments");
    return nullptr;
  }
  at::Tensor q_out, k_out;
  Rows q_r, k_r, v_r, qo_r, ko_r;
  void *pos_p, *cs_p, *axes_p, *qw_p, *kw_p, *kc_p, *vc_p, *slots_p, *stream;
  int64_t tokens, heads, kvh, max_position, num_slots = 0, pos_stride, axes;
  int pb, sb = 4;
  float eps;
  try {
    const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *pos = tensor(a[3]),
                     *cs = tensor(a[4]);
    if (q == nullptr || !q->defined() || !plain(q, at::kBFloat16, 3, *q) ||
        !plain(k, at::kBFloat16, 3, *q) || !plain(cs, at::kFloat, 2, *q) ||
        !PyLong_CheckExact(a[6]) || pos == nullptr || !pos->defined())
      Py_RETURN_NONE;
    axes = PyLong_AsLongLong(a[6]);
    tokens = q->size(0), heads = q->size(1), kvh = k->size(1);
    pb = pos->scalar_type() == at::kLong ? 8 : 4;
    if (!plain(pos, pb == 8 ? at::kLong : at::kInt, 2, *q) || pos->size(0) != axes ||
        pos->size(1) != tokens || pos->stride(1) != 1 || tokens == 0 || q->size(2) != 128 ||
        k->size(0) != tokens || k->size(2) != 128 || kvh == 0 || heads == 0 ||
        q->stride(2) != 1 || k->stride(2) != 1 || cs->size(1) != 128 || !cs->is_contiguous() ||
        !PyFloat_CheckExact(a[9]) || (a[13] != Py_True && a[13] != Py_False))
      Py_RETURN_NONE;
    const at::Tensor* w[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; ++i) {
      if (a[7 + i] == Py_None) continue;
      w[i] = tensor(a[7 + i]);
      if (!plain(w[i], at::kBFloat16, 1, *q) || w[i]->size(0) != 128 || !w[i]->is_contiguous())
        Py_RETURN_NONE;
    }
    const at::Tensor* v = nullptr;
    if (a[2] != Py_None) {
      v = tensor(a[2]);
      if (!plain(v, at::kBFloat16, 3, *q) || v->sizes() != k->sizes() || v->stride(2) != 1)
        Py_RETURN_NONE;
    }
    const at::Tensor *kc = nullptr, *vc = nullptr, *slots = nullptr;
    if (a[10] != Py_None) {
      kc = tensor(a[10]);
      vc = tensor(a[11]);
      slots = tensor(a[12]);
      if (v == nullptr || !plain(kc, at::kBFloat16, 4, *q) || !plain(vc, at::kBFloat16, 4, *q) ||
          kc->sizes() != vc->sizes() || kc->size(2) != kvh || kc->size(3) != 128 ||
          !kc->is_contiguous() || !vc->is_contiguous() || !is_index(slots, tokens, *q, &sb))
        Py_RETURN_NONE;
      num_slots = kc->numel() / (kvh * 128);
    } else if (a[11] != Py_None) {
      Py_RETURN_NONE;  // a v pool alone is refused
    }
    axes_p = PyLong_AsVoidPtr(a[5]);
    stream = PyLong_AsVoidPtr(a[14]);
    if (PyErr_Occurred()) return nullptr;
    eps = float(PyFloat_AS_DOUBLE(a[9]));
    max_position = cs->size(0);
    pos_stride = pos->stride(0);
    q_out = at::empty({tokens, heads, 128}, q->options());
    if (a[13] == Py_True) k_out = at::empty({tokens, kvh, 128}, k->options());
    q_r = rows(q), k_r = rows(k), v_r = rows(v), qo_r = rows(&q_out), ko_r = rows(&k_out);
    pos_p = address(pos), cs_p = address(cs), qw_p = address(w[0]), kw_p = address(w[1]);
    kc_p = address(kc), vc_p = address(vc), slots_p = address(slots);
  } catch (const std::exception&) {
    return declined();
  }
  int rc;
  {
    Unlocked unlocked;
    rc = p_mrope(q_r.p, q_r.s0, q_r.s1, k_r.p, k_r.s0, k_r.s1, v_r.p, v_r.s0, v_r.s1, tokens,
                 heads, kvh, 128, pos_p, pos_stride, pb, axes,
                 static_cast<const int32_t*>(axes_p), qw_p, kw_p, eps,
                 static_cast<const float*>(cs_p), max_position, qo_r.p, qo_r.s0, qo_r.s1, ko_r.p,
                 ko_r.s0, ko_r.s1, kc_p, vc_p, num_slots, slots_p, sb, stream);
  }
  if (rc != KVC_OK) return fail(rc, "kvc_qk_norm_mrope_store");
  PyObject* r = PyTuple_New(2);
  if (r == nullptr) return nullptr;
  PyObject* q_py = wrap(std::move(q_out));
  PyObject* k_py = nullptr;
  if (ko_r.p != nullptr) {
    k_py = wrap(std::move(k_out));
  } else {
    Py_INCREF(Py_None);
    k_py = Py_None;
  }
  PyTuple_SET_ITEM(r, 0, q_py);
  PyTuple_SET_ITEM(r, 1, k_py);
  if (q_py != nullptr && k_py != nullptr) return r;
  Py_DECREF(r);
  return nullptr;
}

// commit(kv_cache, block_tables, context_lens, paths, path_lens, stream):
// True, or None.
PyObject* commit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "commit takes 6 arguments");
    return nullptr;
  }
  void *kv_p, *bt_p, *lens_p, *paths_p, *n_p, *stream;
  int64_t planes, plane, blocks, page, bt_stride, width, path_stride, most, batch;
  try {
    const at::Tensor *kv = tensor(a[0]), *bt = tensor(a[1]), *lens = tensor(a[2]),
                     *paths = tensor(a[3]), *count = tensor(a[4]);
    if (kv == nullptr || !kv->defined() || kv->dim() < 4 ||
        !plain(kv, kv->scalar_type(), kv->dim(), *kv) || !kv->is_contiguous() ||
        kv->numel() == 0 || !plain(bt, at::kInt, 2, *kv) || !plain(paths, at::kInt, 2, *kv))
      Py_RETURN_NONE;
    batch = bt->size(0), width = bt->size(1), most = paths->size(1);
    if (batch == 0 || paths->size(0) != batch || bt->stride(1) != 1 || paths->stride(1) != 1 ||
        !ints(lens, batch, *kv) || !ints(count, batch, *kv))
      Py_RETURN_NONE;
    stream = PyLong_AsVoidPtr(a[5]);
    if (PyErr_Occurred()) return nullptr;
    planes = kv->size(0) * kv->size(1), blocks = kv->size(2), page = kv->size(3);
    plane = kv->numel() / planes * int64_t(kv->element_size());
    bt_stride = bt->stride(0), path_stride = paths->stride(0);
    kv_p = address(kv), bt_p = address(bt), lens_p = address(lens), paths_p = address(paths);
    n_p = address(count);
  } catch (const std::exception&) {
    return declined();
  }
  int rc;
  {
    Unlocked unlocked;
    rc = p_commit(kv_p, planes, plane, blocks, page, plane / (blocks * page),
                  static_cast<int32_t*>(bt_p), bt_stride, width, static_cast<int32_t*>(lens_p),
                  static_cast<int32_t*>(paths_p), path_stride, most, static_cast<int32_t*>(n_p),
                  batch, stream);
  }
  if (rc != KVC_OK) return fail(rc, "kvc_commit_rows");
  Py_RETURN_TRUE;
}

template <typename F>
bool resolve(void* lib, const char* name, F& fn) {
  fn = reinterpret_cast<F>(dlsym(lib, name));
  if (fn == nullptr) PyErr_Format(PyExc_RuntimeError, "%s is not in the kvc library", name);
  return fn != nullptr;
}

// bind(path): the library at `path` (already loaded by _native).
PyObject* bind(PyObject*, PyObject* path) {
  const char* p = PyUnicode_AsUTF8(path);
  if (p == nullptr) return nullptr;
  void* lib = dlopen(p, RTLD_NOW);
  if (lib == nullptr) {
    PyErr_Format(PyExc_RuntimeError, "cannot open %s: %s", p, dlerror());
    return nullptr;
  }
  if (!resolve(lib, "kvc_last_error", p_last_error) ||
      !resolve(lib, "kvc_paged_decode_workspace_bytes", p_workspace) ||
      !resolve(lib, "kvc_paged_decode", p_decode) ||
      !resolve(lib, "kvc_paged_decode_append", p_decode_append) ||
      !resolve(lib, "kvc_qk_norm_rope_store", p_rope) ||
      !resolve(lib, "kvc_scored_workspace_bytes", p_scored_workspace) ||
      !resolve(lib, "kvc_scored_attention", p_scored) ||
      !resolve(lib, "kvc_tree_workspace_bytes", p_tree_workspace) ||
      !resolve(lib, "kvc_tree_attention", p_tree) ||
      !resolve(lib, "kvc_qk_norm_mrope_store", p_mrope) ||
      !resolve(lib, "kvc_commit_rows", p_commit))
    return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, "bind(path): resolve the kvc entry points"},
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL,
     "one paged decode (with the step's append when a key is given), or None"},
    {"rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope)), METH_FASTCALL,
     "the fused norm, rotary and append, or None"},
    {"scored", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scored)), METH_FASTCALL,
     "attention with shaped scores, or None"},
    {"tree", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(tree)), METH_FASTCALL,
     "attention of drafted trees, or None"},
    {"mrope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(mrope)), METH_FASTCALL,
     "the fused norm, multi-axis rotary and append, or None"},
    {"commit", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(commit)), METH_FASTCALL,
     "accepted tree paths moved, or None"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kvc_host", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kvc_host() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
