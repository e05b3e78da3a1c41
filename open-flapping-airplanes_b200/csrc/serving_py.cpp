// The torch view's way from tensors to the C entry points of the serving operators, as a CPython extension: it looks at tensors in place, makes results and workspaces and calls the
// entry points, whose addresses bind() hands in. Whatever is not plainly right is not judged here: the function returns None, and the Python code beside it says what is wrong.
// A small call is bound by the host: asking ten tensors for their shapes and addresses through Python's object protocol took 4 us of logits_process' 9.5, making a result 1 us more.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/Functions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <stdint.h>
#include "../../include/ofa_b200.h"

namespace {

typedef int (*Move)(const ofa_kv_cache*, const ofa_kv_batch*, void*, void*, int, long long, long long, long long, long long, void*);
typedef int (*Attend)(const ofa_kv_cache*, const ofa_kv_batch*, const ofa_paged_attention_args*, void*);
typedef size_t (*Workspace)(const ofa_kv_cache*, const ofa_kv_batch*, int, int);
typedef int (*Process)(const ofa_logits_args*, void*);
Move g_append = nullptr, g_read = nullptr;
Attend g_attend = nullptr;
Workspace g_workspace = nullptr;
Process g_process = nullptr;

constexpr long long INT_END = 1ll << 31;

// A dense-strided CUDA tensor of this type and number of axes, the last of them dense; nullptr: something else (a subclass, another type, device or layout)
const at::Tensor* look(PyObject* o, at::ScalarType type, int dim, long device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.scalar_type() != type || t.dim() != dim || (device >= 0 && t.get_device() != device)) return nullptr;
  if (t.size(dim - 1) > 1 && t.stride(dim - 1) != 1) return nullptr;
  for (int i = 0; i < dim; i++) if (t.size(i) >= INT_END) return nullptr;
  return &t;
}
// bf16 rows [rows][heads][dim]
const at::Tensor* rows_of(PyObject* o, long device, long long rows, long long heads, long long dim) {
  const at::Tensor* t = look(o, at::kBFloat16, 3, device);
  return t && (rows < 0 || t->size(0) == rows) && (heads < 0 || t->size(1) == heads) && t->size(2) == dim && t->stride(2) == 1 ? t : nullptr;
}
// an array [n]; None is a null pointer
template <class T> bool array(PyObject* o, at::ScalarType type, long device, long long n, const T*& ptr) {
  ptr = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = look(o, type, 1, device);
  if (!t || t->size(0) != n) return false;
  ptr = static_cast<const T*>(t->data_ptr());
  return true;
}
// [rows][n]; n < 0: any
template <class T> bool table(PyObject* o, at::ScalarType type, long device, long long rows, long long& n, const T*& ptr, long long& row) {
  ptr = nullptr; row = 0;
  if (o == Py_None) { n = 0; return true; }
  const at::Tensor* t = look(o, type, 2, device);
  if (!t || t->size(0) != rows || (n >= 0 && t->size(1) != n)) return false;
  n = t->size(1); ptr = static_cast<const T*>(t->data_ptr()); row = t->stride(0);
  return true;
}
template <class T> const T* at_address(PyObject* o) { return reinterpret_cast<const T*>((uintptr_t)PyLong_AsUnsignedLongLong(o)); }
void* stream_of(long device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// move(read, cache, batch, device, n_rows or -1, k, v): the entry point's code; with read and no k and v (k, v) in their place
PyObject* move(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !g_append) Py_RETURN_NONE;
  const bool read = PyObject_IsTrue(a[0]);
  const ofa_kv_cache* cache = at_address<ofa_kv_cache>(a[1]);
  const long device = PyLong_AsLong(a[3]);
  const long long rows = PyLong_AsLongLong(a[4]);
  if (PyErr_Occurred() || rows >= INT_END) { PyErr_Clear(); Py_RETURN_NONE; }
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  const bool make = read && a[5] == Py_None && a[6] == Py_None;
  at::Tensor mk, mv;
  const at::Tensor *k = &mk, *v = &mv;
  if (make) {
    if (rows < 0) Py_RETURN_NONE;
    const auto how = at::TensorOptions().dtype(at::kBFloat16).device(at::kCUDA, (c10::DeviceIndex)device);
    mk = at::empty({rows, cache->n_kv_heads, cache->head_dim}, how);
    mv = at::empty({rows, cache->n_kv_heads, cache->head_dim}, how);
  } else {
    k = rows_of(a[5], device, rows, cache->n_kv_heads, cache->head_dim);
    v = k ? rows_of(a[6], device, k->size(0), cache->n_kv_heads, cache->head_dim) : nullptr;
    if (!v) Py_RETURN_NONE;
  }
  const int rc = (read ? g_read : g_append)(cache, at_address<ofa_kv_batch>(a[2]), k->data_ptr(), v->data_ptr(), (int)k->size(0), k->stride(0), k->stride(1), v->stride(0), v->stride(1), stream_of(device));
  if (!make || rc) return PyLong_FromLong(rc);
  PyObject *pk = THPVariable_Wrap(std::move(mk)), *pv = pk ? THPVariable_Wrap(std::move(mv)) : nullptr, *both = pv ? PyTuple_Pack(2, pk, pv) : nullptr;
  Py_XDECREF(pk); Py_XDECREF(pv);
  return both;
  END_HANDLE_TH_ERRORS
}

// attend(cache, batch, device, q, out or None, scale, causal, window, with_lse): out or (out, lse); a code other than 0 if the entry point refused
PyObject* attend(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !g_attend) Py_RETURN_NONE;
  const ofa_kv_cache* cache = at_address<ofa_kv_cache>(p[0]);
  const ofa_kv_batch* batch = at_address<ofa_kv_batch>(p[1]);
  const long device = PyLong_AsLong(p[2]);
  ofa_paged_attention_args a = {};
  a.scale = (float)PyFloat_AsDouble(p[5]);
  a.causal = PyObject_IsTrue(p[6]);
  const long window = PyLong_AsLong(p[7]);
  const bool with_lse = PyObject_IsTrue(p[8]);
  if (PyErr_Occurred() || window != (long)(int)window) { PyErr_Clear(); Py_RETURN_NONE; }
  const at::Tensor* q = rows_of(p[3], device, -1, -1, cache->head_dim);
  if (!q) Py_RETURN_NONE;
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  at::Tensor made, lse, work;
  const at::Tensor* out = &made;
  if (p[4] != Py_None) {
    out = rows_of(p[4], device, q->size(0), q->size(1), cache->head_dim);
    if (!out) Py_RETURN_NONE;
  } else made = at::empty_like(*q);
  if (with_lse) { lse = at::empty({q->size(0), q->size(1)}, q->options().dtype(at::kFloat).requires_grad(false)); a.lse = static_cast<float*>(lse.data_ptr()); }
  a.workspace_bytes = g_workspace(cache, batch, (int)q->size(0), (int)q->size(1));
  if (a.workspace_bytes) {                                        // from torch's allocator: a graph that captures the call keeps its own
    work = at::empty({(long long)a.workspace_bytes}, q->options().dtype(at::kByte).requires_grad(false));
    a.workspace = work.data_ptr();
  }
  a.n_rows = (int)q->size(0); a.n_heads = (int)q->size(1); a.window = (int)window;
  a.q = q->data_ptr(); a.q_row_stride = q->stride(0); a.q_head_stride = q->stride(1);
  a.out = out->data_ptr(); a.out_row_stride = out->stride(0); a.out_head_stride = out->stride(1);
  const int rc = g_attend(cache, batch, &a, stream_of(device));
  if (rc) return PyLong_FromLong(rc);
  PyObject* o = p[4];
  if (o == Py_None) { o = THPVariable_Wrap(std::move(made)); if (!o) return nullptr; } else Py_INCREF(o);
  if (!with_lse) return o;
  PyObject *l = THPVariable_Wrap(std::move(lse)), *both = l ? PyTuple_Pack(2, o, l) : nullptr;
  Py_DECREF(o); Py_XDECREF(l);
  return both;
  END_HANDLE_TH_ERRORS
}

// process(logits, out, tokens, n_tokens, n_prompt, repetition, presence, frequency, bias_ids, bias, mask), the last ten or None: out; a code other than 0 if the entry point refused
PyObject* process(PyObject*, PyObject* const* p, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || !g_process) Py_RETURN_NONE;
  const at::Tensor* x = look(p[0], at::kFloat, 2, -1);
  if (!x) x = look(p[0], at::kBFloat16, 2, -1);
  if (!x) Py_RETURN_NONE;
  const long device = x->get_device();
  const long long rows = x->size(0), vocab = x->size(1);
  if (p[2] == Py_None) for (int i = 3; i < 8; i++) if (p[i] != Py_None) Py_RETURN_NONE;
  if ((p[8] == Py_None) != (p[9] == Py_None)) Py_RETURN_NONE;
  ofa_logits_args a = {};
  long long text = -1, ids = -1, bias_row = 0, words = (vocab + 31) / 32;
  const int* mask = nullptr;
  if (!table(p[2], at::kInt, device, rows, text, a.tokens, a.tokens_stride) || !array(p[3], at::kInt, device, rows, a.n_tokens) || !array(p[4], at::kInt, device, rows, a.n_prompt) ||
      !array(p[5], at::kFloat, device, rows, a.repetition) || !array(p[6], at::kFloat, device, rows, a.presence) || !array(p[7], at::kFloat, device, rows, a.frequency) ||
      !table(p[8], at::kInt, device, rows, ids, a.bias_ids, a.bias_stride) || !table(p[9], at::kFloat, device, rows, ids, a.bias, bias_row) || (rows > 1 && bias_row != a.bias_stride) ||
      !table(p[10], at::kInt, device, rows, words, mask, a.mask_stride)) Py_RETURN_NONE;
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  at::Tensor made;
  const at::Tensor* y = &made;
  if (p[1] != Py_None) {
    y = look(p[1], x->scalar_type(), 2, device);
    if (!y || y->size(0) != rows || y->size(1) != vocab) Py_RETURN_NONE;
  } else made = at::empty_like(*x);
  a.dtype = x->scalar_type() == at::kFloat ? OFA_DTYPE_F32 : OFA_DTYPE_BF16; a.n_rows = (int)rows; a.vocab = (int)vocab;
  a.in = x->data_ptr(); a.in_stride = x->stride(0); a.out = y->data_ptr(); a.out_stride = y->stride(0);
  a.max_tokens = (int)text; a.max_bias = (int)ids; a.mask = reinterpret_cast<const unsigned*>(mask);
  const int rc = g_process(&a, stream_of(device));
  if (rc) return PyLong_FromLong(rc);
  if (p[1] == Py_None) return THPVariable_Wrap(std::move(made));
  Py_INCREF(p[1]);
  return p[1];
  END_HANDLE_TH_ERRORS
}

// bind(append, read, attention, workspace, logits): the entry points' addresses
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) { PyErr_SetString(PyExc_TypeError, "bind takes five arguments"); return nullptr; }
  void* f[5];
  for (int i = 0; i < 5; i++) f[i] = (void*)(uintptr_t)PyLong_AsUnsignedLongLong(a[i]);
  if (PyErr_Occurred()) return nullptr;
  g_append = (Move)f[0]; g_read = (Move)f[1]; g_attend = (Attend)f[2]; g_workspace = (Workspace)f[3]; g_process = (Process)f[4];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
                         {"move", (PyCFunction)(void (*)(void))move, METH_FASTCALL, nullptr},
                         {"attend", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, nullptr},
                         {"process", (PyCFunction)(void (*)(void))process, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
