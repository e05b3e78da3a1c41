// The torch view's way from tensors to the C entry points of the serving operators, as a CPython extension: it looks at each tensor's type, device, shape and strides
// through the object protocol alone (no torch headers, nothing linked: the entry points' addresses are handed in by bind()), and calls the entry point. Whatever
// is not plainly right is not judged here: the function returns None, and the Python code beside it says what is wrong.
// A small call is bound by the host: logits_process with all its arrays took 14 us in Python.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>
#include "../../include/ofa_b200.h"

namespace {

typedef int (*Move)(const ofa_kv_cache*, const ofa_kv_batch*, void*, void*, int, long long, long long, long long, long long, void*);
typedef int (*Attend)(const ofa_kv_cache*, const ofa_kv_batch*, const ofa_paged_attention_args*, void*);
typedef int (*Process)(const ofa_logits_args*, void*);
Move g_append = nullptr, g_read = nullptr;
Attend g_attend = nullptr;
Process g_process = nullptr;
PyObject *g_bf16, *g_f32, *g_i32, *g_u8, *g_stream, *g_current;                    // torch's types, current stream's handle (of a device), current device
PyObject *s_dtype, *s_shape, *s_stride, *s_get_device, *s_data_ptr;

struct Tensor { PyObject* dtype; long long shape[3], stride[3]; int dim; long device; uintptr_t ptr; };

bool numbers(PyObject* t, long long* to, int n) {
  for (int i = 0; i < n; i++) {
    to[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(t, i));
    if (to[i] == -1 && PyErr_Occurred()) return false;
  }
  return true;
}
// false, with no error set, for anything that is not a tensor of at most three axes
bool look(PyObject* o, Tensor& t) {
  bool ok = false;
  PyObject *shape = nullptr, *stride = nullptr, *device = nullptr, *ptr = nullptr;
  t.dtype = PyObject_GetAttr(o, s_dtype);
  if (t.dtype) Py_DECREF(t.dtype);                                                 // torch keeps its types
  if (t.dtype && (shape = PyObject_GetAttr(o, s_shape)) && PyTuple_Check(shape) && (stride = PyObject_CallMethodNoArgs(o, s_stride)) && PyTuple_Check(stride) &&
      (device = PyObject_CallMethodNoArgs(o, s_get_device)) && (ptr = PyObject_CallMethodNoArgs(o, s_data_ptr))) {
    t.dim = (int)PyTuple_GET_SIZE(shape);
    ok = t.dim <= 3 && PyTuple_GET_SIZE(stride) == t.dim && numbers(shape, t.shape, t.dim) && numbers(stride, t.stride, t.dim);
    t.device = PyLong_AsLong(device);
    t.ptr = (uintptr_t)PyLong_AsUnsignedLongLong(ptr);
  }
  Py_XDECREF(shape); Py_XDECREF(stride); Py_XDECREF(device); Py_XDECREF(ptr);
  if (PyErr_Occurred()) { PyErr_Clear(); ok = false; }
  return ok;
}
// bf16 rows [rows][heads][dim], the last axis dense
bool rows_of(const Tensor& t, long device, long long rows, long long heads, long long dim) {
  return t.dtype == g_bf16 && t.dim == 3 && t.device == device && t.shape[0] == rows && t.shape[1] == heads && t.shape[2] == dim && t.stride[2] == 1 && rows < (1ll << 31);
}
// a dense array [n]; None is 0
bool array(PyObject* o, PyObject* dtype, long device, long long n, uintptr_t& ptr) {
  Tensor t;
  ptr = 0;
  if (o == Py_None) return true;
  if (!look(o, t) || t.dtype != dtype || t.device != device || t.dim != 1 || t.shape[0] != n || (n > 1 && t.stride[0] != 1)) return false;
  ptr = t.ptr;
  return true;
}
// [rows][n], rows dense; n < 0: any
bool table(PyObject* o, PyObject* dtype, long device, long long rows, long long& n, uintptr_t& ptr, long long& row) {
  Tensor t;
  ptr = 0; row = 0;
  if (o == Py_None) { n = 0; return true; }
  if (!look(o, t) || t.dtype != dtype || t.device != device || t.dim != 2 || t.shape[0] != rows || (n >= 0 && t.shape[1] != n) || t.shape[1] >= (1ll << 31) || (t.shape[1] > 1 && t.stride[1] != 1)) return false;
  n = t.shape[1]; ptr = t.ptr; row = t.stride[0];
  return true;
}
// the current stream of `device`, which has to be the current one
bool stream_of(long device, void*& stream) {
  PyObject* c = PyObject_CallNoArgs(g_current);
  const long current = c ? PyLong_AsLong(c) : -1;
  Py_XDECREF(c);
  PyObject *d = current == device ? PyLong_FromLong(device) : nullptr, *s = d ? PyObject_CallOneArg(g_stream, d) : nullptr;
  const bool ok = s != nullptr;
  if (s) stream = (void*)(uintptr_t)PyLong_AsUnsignedLongLong(s);
  Py_XDECREF(d); Py_XDECREF(s);
  if (PyErr_Occurred()) { PyErr_Clear(); return false; }
  return ok;
}
template <class T> const T* at(PyObject* o) { return reinterpret_cast<const T*>((uintptr_t)PyLong_AsUnsignedLongLong(o)); }

// move(read, cache, batch, n_kv_heads, head_dim, device, n_rows or -1, k, v)
PyObject* move(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9 || !g_append) Py_RETURN_NONE;
  const long heads = PyLong_AsLong(a[3]), dim = PyLong_AsLong(a[4]), device = PyLong_AsLong(a[5]);
  const long long rows = PyLong_AsLongLong(a[6]);
  Tensor k, v;
  void* stream = nullptr;
  if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  if (!look(a[7], k) || !look(a[8], v) || !rows_of(k, device, rows < 0 ? k.shape[0] : rows, heads, dim) || !rows_of(v, device, k.shape[0], heads, dim) || !stream_of(device, stream)) Py_RETURN_NONE;
  return PyLong_FromLong((PyObject_IsTrue(a[0]) ? g_read : g_append)(at<ofa_kv_cache>(a[1]), at<ofa_kv_batch>(a[2]), (void*)k.ptr, (void*)v.ptr, (int)k.shape[0], k.stride[0], k.stride[1],
                                                                      v.stride[0], v.stride[1], stream));
}

// attend(cache, batch, head_dim, device, q, out, lse or None, work or None, scale, causal, window)
PyObject* attend(PyObject*, PyObject* const* p, Py_ssize_t n) {
  if (n != 11 || !g_attend) Py_RETURN_NONE;
  const long dim = PyLong_AsLong(p[2]), device = PyLong_AsLong(p[3]);
  Tensor q, o, l, w;
  ofa_paged_attention_args a = {};
  void* stream = nullptr;
  a.scale = (float)PyFloat_AsDouble(p[8]);
  a.causal = PyObject_IsTrue(p[9]);
  const long window = PyLong_AsLong(p[10]);
  if (PyErr_Occurred() || window != (long)(int)window) { PyErr_Clear(); Py_RETURN_NONE; }
  if (!look(p[4], q) || q.dim != 3 || !look(p[5], o) || !rows_of(q, device, q.shape[0], q.shape[1], dim) || !rows_of(o, device, q.shape[0], q.shape[1], dim) || q.shape[1] >= (1ll << 31)) Py_RETURN_NONE;
  if (p[6] != Py_None) {
    if (!look(p[6], l) || l.dtype != g_f32 || l.device != device || l.dim != 2 || l.shape[0] != q.shape[0] || l.shape[1] != q.shape[1]) Py_RETURN_NONE;
    a.lse = (float*)l.ptr;
  }
  if (p[7] != Py_None) {
    if (!look(p[7], w) || w.dtype != g_u8 || w.device != device || w.dim != 1) Py_RETURN_NONE;
    a.workspace = (void*)w.ptr; a.workspace_bytes = (size_t)w.shape[0];
  }
  if (!stream_of(device, stream)) Py_RETURN_NONE;
  a.n_rows = (int)q.shape[0]; a.n_heads = (int)q.shape[1]; a.window = (int)window;
  a.q = (const void*)q.ptr; a.q_row_stride = q.stride[0]; a.q_head_stride = q.stride[1];
  a.out = (void*)o.ptr; a.out_row_stride = o.stride[0]; a.out_head_stride = o.stride[1];
  return PyLong_FromLong(g_attend(at<ofa_kv_cache>(p[0]), at<ofa_kv_batch>(p[1]), &a, stream));
}

// process(logits, out, tokens, n_tokens, n_prompt, repetition, presence, frequency, bias_ids, bias, mask), the last nine or None
PyObject* process(PyObject*, PyObject* const* p, Py_ssize_t n) {
  if (n != 11 || !g_process) Py_RETURN_NONE;
  Tensor x, y;
  if (!look(p[0], x) || x.dim != 2 || (x.dtype != g_f32 && x.dtype != g_bf16) || x.device < 0) Py_RETURN_NONE;
  const long long rows = x.shape[0], vocab = x.shape[1];
  if (!look(p[1], y) || y.dtype != x.dtype || y.device != x.device || y.dim != 2 || y.shape[0] != rows || y.shape[1] != vocab || rows >= (1ll << 31) || vocab >= (1ll << 31) ||
      (vocab > 1 && (x.stride[1] != 1 || y.stride[1] != 1))) Py_RETURN_NONE;
  if (p[2] == Py_None) for (int i = 3; i < 8; i++) if (p[i] != Py_None) Py_RETURN_NONE;
  if ((p[8] == Py_None) != (p[9] == Py_None)) Py_RETURN_NONE;
  ofa_logits_args a = {};
  uintptr_t ptr[9];
  long long text = -1, ids = -1, bias_row = 0, words = (vocab + 31) / 32;
  if (!table(p[2], g_i32, x.device, rows, text, ptr[0], a.tokens_stride) || !array(p[3], g_i32, x.device, rows, ptr[1]) || !array(p[4], g_i32, x.device, rows, ptr[2]) ||
      !array(p[5], g_f32, x.device, rows, ptr[3]) || !array(p[6], g_f32, x.device, rows, ptr[4]) || !array(p[7], g_f32, x.device, rows, ptr[5]) ||
      !table(p[8], g_i32, x.device, rows, ids, ptr[6], a.bias_stride) || !table(p[9], g_f32, x.device, rows, ids, ptr[7], bias_row) || (rows > 1 && bias_row != a.bias_stride) ||
      !table(p[10], g_i32, x.device, rows, words, ptr[8], a.mask_stride)) Py_RETURN_NONE;
  void* stream = nullptr;
  if (!stream_of(x.device, stream)) Py_RETURN_NONE;
  a.dtype = x.dtype == g_f32 ? OFA_DTYPE_F32 : OFA_DTYPE_BF16; a.n_rows = (int)rows; a.vocab = (int)vocab;
  a.in = (const void*)x.ptr; a.in_stride = x.stride[0]; a.out = (void*)y.ptr; a.out_stride = y.stride[0];
  a.tokens = (const int*)ptr[0]; a.max_tokens = (int)text; a.n_tokens = (const int*)ptr[1]; a.n_prompt = (const int*)ptr[2];
  a.repetition = (const float*)ptr[3]; a.presence = (const float*)ptr[4]; a.frequency = (const float*)ptr[5];
  a.bias_ids = (const int*)ptr[6]; a.bias = (const float*)ptr[7]; a.max_bias = (int)ids; a.mask = (const unsigned*)ptr[8];
  return PyLong_FromLong(g_process(&a, stream));
}

// bind(append, read, attention, logits: addresses; bf16, f32, i32, u8: types; stream, current: functions)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10) { PyErr_SetString(PyExc_TypeError, "bind takes ten arguments"); return nullptr; }
  void* f[4];
  for (int i = 0; i < 4; i++) f[i] = (void*)(uintptr_t)PyLong_AsUnsignedLongLong(a[i]);
  if (PyErr_Occurred()) return nullptr;
  PyObject** to[6] = {&g_bf16, &g_f32, &g_i32, &g_u8, &g_stream, &g_current};
  for (int i = 0; i < 6; i++) { Py_INCREF(a[4 + i]); Py_XDECREF(*to[i]); *to[i] = a[4 + i]; }
  g_append = (Move)f[0]; g_read = (Move)f[1]; g_attend = (Attend)f[2]; g_process = (Process)f[3];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
                         {"move", (PyCFunction)(void (*)(void))move, METH_FASTCALL, nullptr},
                         {"attend", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, nullptr},
                         {"process", (PyCFunction)(void (*)(void))process, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) {
  s_dtype = PyUnicode_InternFromString("dtype"); s_shape = PyUnicode_InternFromString("shape"); s_stride = PyUnicode_InternFromString("stride");
  s_get_device = PyUnicode_InternFromString("get_device"); s_data_ptr = PyUnicode_InternFromString("data_ptr");
  if (!s_dtype || !s_shape || !s_stride || !s_get_device || !s_data_ptr) return nullptr;
  return PyModule_Create(&module);
}
