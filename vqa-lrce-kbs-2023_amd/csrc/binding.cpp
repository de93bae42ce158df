// The host side of an operator call without an interpreter's share in it: argument test, allocation, descriptor and launch
// of the attention, norm + rotation and embedding operators for the plain case (strides and alignment as the kernels read
// them, the tensors' device current).  A call of these on single tokens is host-bound: 12 us each from Python with its
// descriptor packed there, 6.5 us from here.  Everything else - other layouts, other devices, wrong arguments, errors -
// returns None, and lrce/kernels.py takes the call, words the refusal or makes the copies.  The launches go through the
// C ABI, whose addresses bind() gets from the library that Python loaded.
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/lrce_hip.h"

namespace {

decltype(&lrce_attn_fwd) attn_fwd;
decltype(&lrce_attn_bwd) attn_bwd;
decltype(&lrce_attn_fwd_workspace) attn_fwd_ws;
decltype(&lrce_attn_bwd_workspace) attn_bwd_ws;
decltype(&lrce_qk_norm_rope_fwd) rope_fwd;
decltype(&lrce_qk_norm_rope_bwd) rope_bwd;
decltype(&lrce_qk_norm_rope_bwd_workspace) rope_bwd_ws;
decltype(&lrce_embedding_fwd) embed_fwd;
decltype(&lrce_embedding_bwd) embed_bwd;
decltype(&lrce_embedding_bwd_workspace) embed_bwd_ws;

// a tensor argument (no subclass) on a device, or null
const at::Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}

// the call's last two arguments: the current device, which has to be the tensors', and its current stream
bool where(PyObject* const* a, const at::Tensor* t, void** stream) {
  const long dev = PyLong_AsLong(a[0]);
  *stream = PyLong_AsVoidPtr(a[1]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return t->get_device() == dev;
}

// batch / row / head strides of [B, L, H, D] with a contiguous last axis (0 for an axis of length 1)
bool head_strides(const at::Tensor& t, int64_t* s, bool vec16) {
  if (t.dim() != 4 || (t.stride(3) != 1 && t.size(3) > 1)) return false;
  for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
  if (!vec16) return true;
  return !((s[0] | s[1] | s[2]) & 7) && s[1] < (1 << 23) && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15);
}
void plain_strides(int64_t* s, int64_t L, int64_t H, int64_t D) {
  s[0] = L * H * D;
  s[1] = H * D;
  s[2] = D;
}

int type_code(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : t == at::kFloat ? 2 : -1; }
int int_bytes(at::ScalarType t) { return t == at::kLong ? 8 : t == at::kInt ? 4 : 0; }

// q, k, v, key_mask, scale -> d; false: not the plain case
bool attn_args(PyObject* const* a, LrceAttnDesc& d, const at::Tensor*& q, const at::Tensor*& k) {
  q = tensor(a[0]);
  k = tensor(a[1]);
  const at::Tensor* v = tensor(a[2]);
  if (!q || !k || !v) return false;
  const auto dt = q->scalar_type();
  const auto dev = q->device();
  if ((dt != at::kBFloat16 && dt != at::kHalf) || k->scalar_type() != dt || v->scalar_type() != dt || k->device() != dev || v->device() != dev)
    return false;
  d = LrceAttnDesc{};
  if (!head_strides(*q, d.q_stride, true) || !head_strides(*k, d.k_stride, true) || !head_strides(*v, d.v_stride, true)) return false;
  const int64_t B = q->size(0), Lq = q->size(1), H = q->size(2), D = q->size(3), Lk = k->size(1), Hk = k->size(2);
  if (k->size(0) != B || k->size(3) != D || !k->sizes().equals(v->sizes()) || (D != 32 && D != 64 && D != 96 && D != 128) || Hk < 1 || H < 1 ||
      H % Hk || B > INT32_MAX || Lq > INT32_MAX || Lk > INT32_MAX || H > INT32_MAX)
    return false;
  if (a[3] != Py_None) {
    const at::Tensor* m = tensor(a[3]);
    if (!m || m->device() != dev || m->dim() != 2 || m->size(0) != B || m->size(1) != Lk || (Lk > 1 && m->stride(1) != 1)) return false;
    switch (m->scalar_type()) {
      case at::kBool: case at::kByte: case at::kChar: d.mask_bytes = 1; break;
      case at::kInt: d.mask_bytes = 4; break;
      case at::kLong: d.mask_bytes = 8; break;
      default: return false;
    }
    d.key_mask = m->data_ptr();
    d.mask_stride = B > 1 ? m->stride(0) : 0;
  }
  const int causal = PyObject_IsTrue(a[4]);
  if (causal < 0) { PyErr_Clear(); return false; }
  d.causal = causal;
  if (a[5] == Py_None) {
    d.scale = (float)(1.0 / std::sqrt((double)D));
  } else {
    const double s = PyFloat_AsDouble(a[5]);
    if (s == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    d.scale = (float)s;
    if (!(s > 0.0) || !std::isfinite(s)) return false;
  }
  d.q = q->data_ptr(); d.k = k->data_ptr(); d.v = v->data_ptr();
  d.B = (int32_t)B; d.H = (int32_t)H; d.Hk = (int32_t)Hk; d.Lq = (int32_t)Lq; d.Lk = (int32_t)Lk; d.D = (int32_t)D;
  d.f16 = dt == at::kHalf;
  return true;
}

bool workspace(at::Tensor& ws, int64_t n, const at::Tensor& like, float*& p, int64_t& elems) {
  if (n < 0) return false;
  if (n > 0) {
    ws = at::empty({n}, like.options().dtype(at::kFloat));
    p = static_cast<float*>(ws.data_ptr());
    elems = n;
  }
  return true;
}

PyObject* pack(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// Allocations and launches may wait (a full queue, the allocator's lock): other threads run meanwhile
template <typename F>
bool unlocked(F&& f) {
  struct NoGil {
    PyThreadState* state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
  } no_gil;
  at::AutoDispatchBelowADInplaceOrView no_grad;
  return f();
}

// No C++ exception leaves a call: what throws here (an allocation that fails) is for the Python path to meet and report
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// attention(q, k, v, key_mask, causal, scale, device, stream)
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    LrceAttnDesc d;
    const at::Tensor *q, *k;
    void* stream;
    if (n != 8 || !attn_args(a, d, q, k) || !where(a + 6, q, &stream)) Py_RETURN_NONE;
    at::Tensor out, lse;
    const bool ok = unlocked([&] {
      at::Tensor ws;
      out = at::empty({d.B, d.Lq, d.H, d.D}, q->options());
      lse = at::empty({d.B, d.H, d.Lq}, q->options().dtype(at::kFloat));
      d.out = out.data_ptr();
      d.lse = static_cast<float*>(lse.data_ptr());
      plain_strides(d.o_stride, d.Lq, d.H, d.D);
      return workspace(ws, attn_fwd_ws(&d), *q, d.workspace, d.workspace_elems) && attn_fwd(&d, stream) == LRCE_OK;
    });
    if (!ok) Py_RETURN_NONE;
    return pack({out, lse});
  });
}

// attention_bwd(q, k, v, key_mask, causal, scale, dout, out, lse, device, stream)
PyObject* py_attention_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    LrceAttnDesc d;
    const at::Tensor *q, *k;
    void* stream;
    if (n != 11 || !attn_args(a, d, q, k) || !where(a + 9, q, &stream)) Py_RETURN_NONE;
    const at::Tensor *g = tensor(a[6]), *out = tensor(a[7]), *lse = tensor(a[8]);
    if (!g || !out || !lse || g->scalar_type() != q->scalar_type() || out->scalar_type() != q->scalar_type() || lse->scalar_type() != at::kFloat ||
        g->device() != q->device() || out->device() != q->device() || lse->device() != q->device() || !g->sizes().equals(q->sizes()) ||
        !out->sizes().equals(q->sizes()) || lse->dim() != 3 || lse->size(0) != d.B || lse->size(1) != d.H || lse->size(2) != d.Lq ||
        !lse->is_contiguous() || !head_strides(*g, d.g_stride, true) || !head_strides(*out, d.o_stride, true))
      Py_RETURN_NONE;
    at::Tensor dq, dk, dv;
    const bool ok = unlocked([&] {
      at::Tensor ws;
      dq = at::empty({d.B, d.Lq, d.H, d.D}, q->options());
      dk = at::empty({d.B, d.Lk, d.Hk, d.D}, q->options());
      dv = at::empty({d.B, d.Lk, d.Hk, d.D}, q->options());
      d.out = out->data_ptr();
      d.lse = static_cast<float*>(lse->data_ptr());
      d.dout = g->data_ptr();
      d.dq = dq.data_ptr();
      d.dk = dk.data_ptr();
      d.dv = dv.data_ptr();
      plain_strides(d.dq_stride, d.Lq, d.H, d.D);
      plain_strides(d.dk_stride, d.Lk, d.Hk, d.D);
      plain_strides(d.dv_stride, d.Lk, d.Hk, d.D);
      return workspace(ws, attn_bwd_ws(&d), *q, d.workspace, d.workspace_elems) && attn_bwd(&d, stream) == LRCE_OK;
    });
    if (!ok) Py_RETURN_NONE;
    return pack({dq, dk, dv});
  });
}

// q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved -> d; false: not the plain case
bool rope_args(PyObject* const* a, LrceRopeDesc& d, const at::Tensor*& q, const at::Tensor*& k) {
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i) {
    t[i] = tensor(a[i]);
    if (!t[i] || t[i]->device() != t[0]->device()) return false;
  }
  q = t[0];
  k = t[1];
  d = LrceRopeDesc{};
  d.dtype = type_code(q->scalar_type());
  if (d.dtype < 0 || k->scalar_type() != q->scalar_type() || !head_strides(*q, d.q_stride, false) || !head_strides(*k, d.k_stride, false)) return false;
  const int64_t B = q->size(0), L = q->size(1), H = q->size(2), D = q->size(3), Hk = k->size(2);
  if (k->size(0) != B || k->size(1) != L || k->size(3) != D || H < 1 || Hk < 1 || D < 8 || D > 256 || D % 8 || B > INT32_MAX || L > INT32_MAX ||
      H > INT32_MAX || Hk > INT32_MAX)
    return false;
  for (int i = 2; i < 4; ++i)
    if (t[i]->scalar_type() != at::kFloat || t[i]->dim() != 1 || t[i]->size(0) != D || !t[i]->is_contiguous()) return false;
  if (t[5]->scalar_type() != at::kFloat || t[5]->dim() != 1 || !t[5]->is_contiguous() || t[5]->size(0) < 1 || 2 * t[5]->size(0) > D) return false;
  const at::Tensor& pos = *t[4];
  d.pos_bytes = int_bytes(pos.scalar_type());
  if (!d.pos_bytes || !pos.is_contiguous() || !((pos.dim() == 2 && pos.size(0) == B && pos.size(1) == L) || (pos.dim() == 1 && pos.size(0) == L))) return false;
  const double eps = PyFloat_AsDouble(a[6]);
  if ((eps == -1.0 && PyErr_Occurred()) || !(eps >= 0.0) || !std::isfinite(eps)) { PyErr_Clear(); return false; }
  const int inter = PyObject_IsTrue(a[7]);
  if (inter < 0) { PyErr_Clear(); return false; }
  d.q = q->data_ptr(); d.k = k->data_ptr();
  d.q_weight = static_cast<float*>(t[2]->data_ptr()); d.k_weight = static_cast<float*>(t[3]->data_ptr());
  d.positions = pos.data_ptr(); d.inv_freq = static_cast<float*>(t[5]->data_ptr());
  d.pos_stride = pos.dim() == 2 ? L : 0;
  d.B = (int32_t)B; d.L = (int32_t)L; d.H = (int32_t)H; d.Hk = (int32_t)Hk; d.D = (int32_t)D; d.R = (int32_t)(2 * t[5]->size(0));
  d.interleaved = inter; d.eps = (float)eps;
  plain_strides(d.qo_stride, L, H, D);
  plain_strides(d.ko_stride, L, Hk, D);
  return true;
}

// qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved, device, stream)
PyObject* py_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    LrceRopeDesc d;
    const at::Tensor *q, *k;
    void* stream;
    if (n != 10 || !rope_args(a, d, q, k) || !where(a + 8, q, &stream)) Py_RETURN_NONE;
    at::Tensor qo, ko;
    const bool ok = unlocked([&] {
      qo = at::empty({d.B, d.L, d.H, d.D}, q->options());
      ko = at::empty({d.B, d.L, d.Hk, d.D}, q->options());
      d.q_out = qo.data_ptr();
      d.k_out = ko.data_ptr();
      return rope_fwd(&d, stream) == LRCE_OK;
    });
    if (!ok) Py_RETURN_NONE;
    return pack({qo, ko});
  });
}

// qk_norm_rope_bwd(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved, dq_out, dk_out, device, stream)
PyObject* py_rope_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    LrceRopeDesc d;
    const at::Tensor *q, *k;
    void* stream;
    if (n != 12 || !rope_args(a, d, q, k) || !where(a + 10, q, &stream)) Py_RETURN_NONE;
    const at::Tensor *gq = tensor(a[8]), *gk = tensor(a[9]);
    if (!gq || !gk || gq->scalar_type() != q->scalar_type() || gk->scalar_type() != q->scalar_type() || gq->device() != q->device() ||
        gk->device() != q->device() || !gq->sizes().equals(q->sizes()) || !gk->sizes().equals(k->sizes()) ||
        !head_strides(*gq, d.gq_stride, false) || !head_strides(*gk, d.gk_stride, false))
      Py_RETURN_NONE;
    at::Tensor dq, dk, dqw, dkw;
    const bool ok = unlocked([&] {
      const auto f32 = q->options().dtype(at::kFloat);
      at::Tensor ws;
      dq = at::empty({d.B, d.L, d.H, d.D}, q->options());
      dk = at::empty({d.B, d.L, d.Hk, d.D}, q->options());
      dqw = at::empty({d.D}, f32);
      dkw = at::empty({d.D}, f32);
      d.gq = gq->data_ptr();
      d.gk = gk->data_ptr();
      d.q_out = dq.data_ptr();
      d.k_out = dk.data_ptr();
      d.dq_weight = static_cast<float*>(dqw.data_ptr());
      d.dk_weight = static_cast<float*>(dkw.data_ptr());
      return workspace(ws, rope_bwd_ws((int64_t)d.B * d.L, d.D), *q, d.workspace, d.workspace_elems) && rope_bwd(&d, stream) == LRCE_OK;
    });
    if (!ok) Py_RETURN_NONE;
    return pack({dq, dk, dqw, dkw});
  });
}

// a float argument; false: none
bool number(PyObject* o, float* x) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *x = (float)v;
  return true;
}

// embedding(ids, weight, scale, out_dtype, device, stream)
PyObject* py_embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    void* stream;
    float scale;
    if (n != 6) Py_RETURN_NONE;
    const at::Tensor *ids = tensor(a[0]), *w = tensor(a[1]);
    if (!ids || !w || !where(a + 4, w, &stream) || ids->device() != w->device() || !number(a[2], &scale)) Py_RETURN_NONE;
    const int bytes = int_bytes(ids->scalar_type()), wt = type_code(w->scalar_type());
    auto out = w->scalar_type();
    if (a[3] != Py_None) {
      if (!THPDtype_Check(a[3])) Py_RETURN_NONE;
      out = reinterpret_cast<THPDtype*>(a[3])->scalar_type;
    }
    const int yt = type_code(out);
    if (!bytes || wt < 0 || yt < 0 || (wt != 2 && yt != wt) || !ids->is_contiguous() || w->dim() != 2 || !w->is_contiguous() || w->size(0) < 1 ||
        w->size(1) < 1 || w->size(1) > INT32_MAX)
      Py_RETURN_NONE;
    at::Tensor y;
    const bool ok = unlocked([&] {
      at::DimVector shape(ids->sizes().begin(), ids->sizes().end());
      shape.push_back(w->size(1));
      y = at::empty(shape, w->options().dtype(out));
      return embed_fwd(ids->data_ptr(), bytes, ids->numel(), w->data_ptr(), w->size(1), w->size(0), (int)w->size(1), wt, y.data_ptr(), yt,
                       scale, stream) == LRCE_OK;
    });
    if (!ok) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
  });
}

// embedding_bwd(dy, ids, rows, scale, padding_idx, device, stream): into a new tensor
PyObject* py_embedding_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    void* stream;
    float scale;
    if (n != 7) Py_RETURN_NONE;
    const at::Tensor *dy = tensor(a[0]), *ids = tensor(a[1]);
    if (!ids || !dy || !where(a + 5, dy, &stream) || ids->device() != dy->device() || !number(a[3], &scale)) Py_RETURN_NONE;
    const int64_t rows = PyLong_AsLongLong(a[2]), pad = PyLong_AsLongLong(a[4]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    const int bytes = int_bytes(ids->scalar_type()), yt = type_code(dy->scalar_type());
    if (!bytes || yt < 0 || rows < 1 || !ids->is_contiguous() || !dy->is_contiguous() || dy->dim() != ids->dim() + 1 ||
        dy->sizes().slice(0, ids->dim()) != ids->sizes() || dy->size(-1) < 1 || dy->size(-1) > INT32_MAX)
      Py_RETURN_NONE;
    const int cols = (int)dy->size(-1);
    at::Tensor dw;
    const bool ok = unlocked([&] {
      at::Tensor ws;
      float* p = nullptr;
      int64_t elems = 0;
      dw = at::empty({rows, cols}, dy->options().dtype(at::kFloat));
      return workspace(ws, embed_bwd_ws(ids->numel(), rows, cols), *dy, p, elems) &&
             embed_bwd(ids->data_ptr(), bytes, ids->numel(), dy->data_ptr(), yt, static_cast<float*>(dw.data_ptr()), rows, cols, scale, pad, 0,
                       p, elems, stream) == LRCE_OK;
    });
    if (!ok) Py_RETURN_NONE;
    return THPVariable_Wrap(dw);
  });
}

// bind(...): the entry points' addresses, in this order
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) {
    PyErr_SetString(PyExc_TypeError, "bind: 10 addresses");
    return nullptr;
  }
  void* p[10];
  for (int i = 0; i < 10; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: a null address");
      return nullptr;
    }
  }
  attn_fwd = reinterpret_cast<decltype(attn_fwd)>(p[0]);
  attn_bwd = reinterpret_cast<decltype(attn_bwd)>(p[1]);
  attn_fwd_ws = reinterpret_cast<decltype(attn_fwd_ws)>(p[2]);
  attn_bwd_ws = reinterpret_cast<decltype(attn_bwd_ws)>(p[3]);
  rope_fwd = reinterpret_cast<decltype(rope_fwd)>(p[4]);
  rope_bwd = reinterpret_cast<decltype(rope_bwd)>(p[5]);
  rope_bwd_ws = reinterpret_cast<decltype(rope_bwd_ws)>(p[6]);
  embed_fwd = reinterpret_cast<decltype(embed_fwd)>(p[7]);
  embed_bwd = reinterpret_cast<decltype(embed_bwd)>(p[8]);
  embed_bwd_ws = reinterpret_cast<decltype(embed_bwd_ws)>(p[9]);
  Py_RETURN_NONE;
}

#define LRCE_FN(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef METHODS[] = {
    {"bind", LRCE_FN(py_bind), METH_FASTCALL, nullptr},
    {"attention", LRCE_FN(py_attention), METH_FASTCALL, nullptr},
    {"attention_bwd", LRCE_FN(py_attention_bwd), METH_FASTCALL, nullptr},
    {"qk_norm_rope", LRCE_FN(py_rope), METH_FASTCALL, nullptr},
    {"qk_norm_rope_bwd", LRCE_FN(py_rope_bwd), METH_FASTCALL, nullptr},
    {"embedding", LRCE_FN(py_embedding), METH_FASTCALL, nullptr},
    {"embedding_bwd", LRCE_FN(py_embedding_bwd), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&MODULE); }
