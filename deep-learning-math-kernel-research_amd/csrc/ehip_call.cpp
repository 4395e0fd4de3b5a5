// The calls of a running model's loop -- execute, input quantization, activation reorders -- for Python, straight on the
// CPython API: a call costs 0.2 us on top of the C-ABI where ctypes takes 0.8 us (argument objects, foreign-function
// interface), against 2.6 us for the kernel launch itself.  Everything else of the C-ABI goes through ctypes.
//
// The library is not linked: the package hands the functions' addresses over (bind), so that a process keeps the one
// copy that it loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stddef.h>
#include <string.h>
#include <structmember.h>

#include "euler_hip.h"

namespace {

typedef int (*execute_t)(void *, void *, const void *, const void *, const void *, void *);
typedef int (*quantize_t)(void *, const void *, size_t, float, float, void *);
typedef int (*reorder_t)(void *, const void *, int, int, int, int, int, void *);

typedef int (*layer_t)(const void *, const void *, void *);

execute_t g_execute;
layer_t g_linear, g_experts, g_norm, g_route;
quantize_t g_quantize;
reorder_t g_to_blocked, g_to_nchw;
PyObject *g_raise;      // called with a status that is not zero, raises
PyObject *g_data_ptr;   // "data_ptr"

// device pointer of a tensor (its data_ptr()), of an int, of None
bool as_pointer(PyObject *x, void **p)
{
  if (x == Py_None) {
    *p = nullptr;
    return true;
  }
  if (PyLong_Check(x)) {
    *p = PyLong_AsVoidPtr(x);
    return !PyErr_Occurred();
  }
  PyObject *v = PyObject_CallMethodNoArgs(x, g_data_ptr);
  if (!v) return false;
  *p = PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  return !PyErr_Occurred();
}

PyObject *result(int rc)
{
  if (rc == 0) Py_RETURN_NONE;
  PyObject *r = PyObject_CallFunction(g_raise, "i", rc);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "euler_hip: call failed");
  return nullptr;
}

// The arguments of a vectorcall by name: value[i] is the argument called names[i], or null if it was not given
template <int N>
bool arguments(const char *fn, const char *const (&names)[N], int required, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames,
               PyObject *(&value)[N])
{
  for (int i = 0; i < N; ++i) value[i] = i < nargs ? args[i] : nullptr;
  if (nargs > N) {
    PyErr_Format(PyExc_TypeError, "%s() takes at most %d arguments (%zd given)", fn, N, nargs);
    return false;
  }
  const Py_ssize_t nkw = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
  for (Py_ssize_t k = 0; k < nkw; ++k) {
    PyObject *name = PyTuple_GET_ITEM(kwnames, k);
    int i = 0;
    while (i < N && PyUnicode_CompareWithASCIIString(name, names[i]) != 0) ++i;
    if (i == N) {
      PyErr_Format(PyExc_TypeError, "%s() got an unexpected keyword argument '%U'", fn, name);
      return false;
    }
    if (value[i]) {
      PyErr_Format(PyExc_TypeError, "%s() got multiple values for argument '%s'", fn, names[i]);
      return false;
    }
    value[i] = args[nargs + k];
  }
  for (int i = 0; i < required; ++i)
    if (!value[i]) {
      PyErr_Format(PyExc_TypeError, "%s() missing required argument: '%s'", fn, names[i]);
      return false;
    }
  return true;
}

bool pointer_or_null(PyObject *x, void **p)
{
  *p = nullptr;
  return !x || as_pointer(x, p);
}

// a stream: its address as an int, None or not given for the default stream.  Not a tensor: one in the stream's place (one
// positional argument too many) would hand the runtime its data as a stream.
bool stream_or_null(PyObject *x, void **p)
{
  if (x && x != Py_None && !PyLong_Check(x)) {
    PyErr_Format(PyExc_TypeError, "stream: an int or None, not %.100s", Py_TYPE(x)->tp_name);
    return false;
  }
  return pointer_or_null(x, p);
}

bool as_int(PyObject *x, int *v)
{
  const long l = PyLong_AsLong(x);
  if (l == -1 && PyErr_Occurred()) return false;
  if (l != (long)(int)l) {
    PyErr_SetString(PyExc_OverflowError, "integer argument does not fit 32 bits");
    return false;
  }
  *v = (int)l;
  return true;
}

// ---- the base class of Conv: the handle and its execute ------------------------------------------
struct ConvBase {
  PyObject_HEAD
  void *handle;
};

PyObject *conv_execute(PyObject *self, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames)
{
  static const char *const names[] = {"output", "input", "weights", "bias", "stream"};
  PyObject *v[5];
  void *p[5];
  if (!arguments("execute", names, 2, args, nargs, kwnames, v)) return nullptr;
  for (int i = 0; i < 4; ++i)
    if (!pointer_or_null(v[i], &p[i])) return nullptr;
  if (!stream_or_null(v[4], &p[4])) return nullptr;
  void *h = reinterpret_cast<ConvBase *>(self)->handle;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_execute(h, p[0], p[1], p[2], p[3], p[4]);
  Py_END_ALLOW_THREADS
  return result(rc);
}

PyObject *conv_get_h(PyObject *self, void *)
{
  void *h = reinterpret_cast<ConvBase *>(self)->handle;
  if (!h) Py_RETURN_NONE;
  return PyLong_FromVoidPtr(h);
}
int conv_set_h(PyObject *self, PyObject *v, void *)
{
  void *h = nullptr;
  if (v && !as_pointer(v, &h)) return -1;
  reinterpret_cast<ConvBase *>(self)->handle = h;
  return 0;
}

PyMethodDef conv_methods[] = {
    {"execute", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(conv_execute)), METH_FASTCALL | METH_KEYWORDS,
     "execute(output, input, weights=None, bias=None, stream=0): ehip_conv_execute; tensors, device addresses or None, and "
     "the stream's address"},
    {nullptr, nullptr, 0, nullptr}};
PyGetSetDef conv_getset[] = {{"_h", conv_get_h, conv_set_h, "address of the C handle, or None", nullptr},
                             {nullptr, nullptr, nullptr, nullptr, nullptr}};
PyTypeObject conv_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

// ---- linear, norm, route: a handle, and an execute that fills the C-ABI's argument structure --------------------
// kind of each argument by name, in the order of the structure's fields: p = pointer, q = 64-bit integer, i = 32-bit integer,
// s = the stream.  `at` maps the order of the Python arguments to that of the fields.
struct Field {
  const char *name;
  char kind;
  size_t offset;
};

// The names of keyword arguments are interned where they stand in a caller's source: mostly one comparison of pointers each
template <int N>
PyObject *layer_execute(PyObject *self, const char *fn, layer_t f, const Field (&fields)[N], PyObject *(&interned)[N], int required,
                        PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames, char *block)
{
  PyObject *v[N];
  const Py_ssize_t nkw = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
  bool plain = nargs <= N;
  if (plain) {
    for (int i = 0; i < N; ++i) v[i] = i < nargs ? args[i] : nullptr;
    int i = 0;   // (keywords mostly come in the order of the fields)
    for (Py_ssize_t k = 0; k < nkw && plain; ++k) {
      PyObject *name = PyTuple_GET_ITEM(kwnames, k);
      int looked = 0;
      for (; looked < N && interned[i] != name; ++looked) i = i + 1 < N ? i + 1 : 0;
      plain = looked < N && !v[i];
      if (plain) v[i] = args[nargs + k];
    }
    for (int r = 0; r < required; ++r) plain = plain && v[r];
  }
  if (!plain) {   // a name that is not interned, or an argument list that is wrong
    const char *names[N];
    for (int i = 0; i < N; ++i) names[i] = fields[i].name;
    if (!arguments(fn, names, required, args, nargs, kwnames, v)) return nullptr;
  }
  void *stream = nullptr;
  for (int i = 0; i < N; ++i) {
    const Field &d = fields[i];
    if (d.kind == 's') {
      if (!stream_or_null(v[i], &stream)) return nullptr;
    } else if (d.kind == 'p') {
      void *p;
      if (!pointer_or_null(v[i], &p)) return nullptr;
      memcpy(block + d.offset, &p, sizeof(p));
    } else if (v[i]) {
      PyObject *n = PyNumber_Index(v[i]);
      if (!n) return nullptr;
      const long long q = PyLong_AsLongLong(n);
      int w = 0;
      const bool ok = d.kind == 'q' ? !PyErr_Occurred() : as_int(n, &w);
      Py_DECREF(n);
      if (!ok) return nullptr;
      if (d.kind == 'q') memcpy(block + d.offset, &q, sizeof(q));
      else memcpy(block + d.offset, &w, sizeof(w));
    }
  }
  void *h = reinterpret_cast<ConvBase *>(self)->handle;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(h, block, stream);
  Py_END_ALLOW_THREADS
  return result(rc);
}

template <int N>
bool intern(const Field (&fields)[N], PyObject *(&interned)[N])
{
  for (int i = 0; i < N && !interned[N - 1]; ++i)
    if (!interned[i] && !(interned[i] = PyUnicode_InternFromString(fields[i].name))) return false;
  return true;
}

#define F(S, name, kind, field) {name, kind, offsetof(S, field)}
PyObject *linear_execute(PyObject *self, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames)
{
  typedef ehip_linear_args_t S;
  static const Field fields[] = {F(S, "output", 'p', output_dev), F(S, "input", 'p', input_dev), F(S, "rows", 'q', rows),
                                 F(S, "input_scale", 'p', input_scale_dev), F(S, "residual", 'p', residual_dev),
                                 F(S, "output_stride", 'q', output_stride), F(S, "input_stride", 'q', input_stride),
                                 F(S, "residual_stride", 'q', residual_stride), {"stream", 's', 0}};
  static PyObject *interned[sizeof(fields) / sizeof(fields[0])];
  if (!intern(fields, interned)) return nullptr;
  S block = {};
  return layer_execute(self, "execute", g_linear, fields, interned, 3, args, nargs, kwnames, reinterpret_cast<char *>(&block));
}
PyObject *experts_execute(PyObject *self, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames)
{
  typedef ehip_linear_args_t S;
  static const Field fields[] = {F(S, "output", 'p', output_dev), F(S, "input", 'p', input_dev), F(S, "slots", 'p', slots_dev),
                                 F(S, "offsets", 'p', offsets_dev), F(S, "rows", 'q', rows), F(S, "topk", 'i', topk),
                                 F(S, "input_scale", 'p', input_scale_dev), F(S, "input_rows", 'i', input_rows),
                                 F(S, "output_rows", 'i', output_rows), F(S, "output_stride", 'q', output_stride),
                                 F(S, "input_stride", 'q', input_stride), {"stream", 's', 0}};
  static PyObject *interned[sizeof(fields) / sizeof(fields[0])];
  if (!intern(fields, interned)) return nullptr;
  S block = {};
  return layer_execute(self, "execute_experts", g_experts, fields, interned, 6, args, nargs, kwnames, reinterpret_cast<char *>(&block));
}
PyObject *norm_execute(PyObject *self, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames)
{
  typedef ehip_norm_args_t S;
  static const Field fields[] = {F(S, "output", 'p', output_dev), F(S, "block", 'p', block_dev), F(S, "rows", 'q', rows),
                                 F(S, "output_scale", 'p', output_scale_dev), F(S, "sum", 'p', sum_dev), F(S, "residual", 'p', residual_dev),
                                 F(S, "gate", 'p', gate_dev), F(S, "part_weights", 'p', part_weights_dev),
                                 F(S, "post_weight", 'p', post_weight_dev), F(S, "post_bias", 'p', post_bias_dev),
                                 F(S, "pre_weight", 'p', pre_weight_dev), F(S, "pre_bias", 'p', pre_bias_dev),
                                 F(S, "output_stride", 'q', output_stride), F(S, "sum_stride", 'q', sum_stride),
                                 F(S, "block_stride", 'q', block_stride), F(S, "residual_stride", 'q', residual_stride),
                                 F(S, "gate_stride", 'q', gate_stride), {"stream", 's', 0}};
  static PyObject *interned[sizeof(fields) / sizeof(fields[0])];
  if (!intern(fields, interned)) return nullptr;
  S block = {};
  return layer_execute(self, "execute", g_norm, fields, interned, 3, args, nargs, kwnames, reinterpret_cast<char *>(&block));
}
PyObject *route_execute(PyObject *self, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames)
{
  typedef ehip_route_args_t S;
  static const Field fields[] = {F(S, "ids", 'p', ids_dev), F(S, "weights", 'p', weights_dev), F(S, "plan", 'p', plan_dev),
                                 F(S, "logits", 'p', logits_dev), F(S, "tokens", 'q', tokens), F(S, "bias", 'p', bias_dev),
                                 F(S, "logits_stride", 'q', logits_stride), {"stream", 's', 0}};
  static PyObject *interned[sizeof(fields) / sizeof(fields[0])];
  if (!intern(fields, interned)) return nullptr;
  S block = {};
  return layer_execute(self, "execute", g_route, fields, interned, 5, args, nargs, kwnames, reinterpret_cast<char *>(&block));
}
#undef F

#define EHIP_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL | METH_KEYWORDS
PyMethodDef linear_methods[] = {
    {"execute", EHIP_FAST(linear_execute),
     "execute(output, input, rows, input_scale=None, residual=None, output_stride=0, input_stride=0, residual_stride=0, stream=0): "
     "ehip_linear_execute; tensors, device addresses or None, strides in elements (0: rows without a gap), the stream's address"},
    {"execute_experts", EHIP_FAST(experts_execute),
     "execute_experts(output, input, slots, offsets, rows, topk, input_scale=None, input_rows=ROWS_SORTED, output_rows=ROWS_SORTED, "
     "output_stride=0, input_stride=0, stream=0): ehip_linear_execute_experts"},
    {nullptr, nullptr, 0, nullptr}};
PyMethodDef norm_methods[] = {
    {"execute", EHIP_FAST(norm_execute),
     "execute(output, block, rows, output_scale=None, sum=None, residual=None, gate=None, part_weights=None, post_weight=None, "
     "post_bias=None, pre_weight=None, pre_bias=None, output_stride=0, sum_stride=0, block_stride=0, residual_stride=0, gate_stride=0, "
     "stream=0): ehip_norm_execute"},
    {nullptr, nullptr, 0, nullptr}};
PyMethodDef route_methods[] = {
    {"execute", EHIP_FAST(route_execute),
     "execute(ids, weights, plan, logits, tokens, bias=None, logits_stride=0, stream=0): ehip_route_execute"},
    {nullptr, nullptr, 0, nullptr}};
PyTypeObject linear_type = {PyVarObject_HEAD_INIT(nullptr, 0)}, norm_type = {PyVarObject_HEAD_INIT(nullptr, 0)},
             route_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

// ---- functions -----------------------------------------------------------------------------------
PyObject *quantize_input_u8(PyObject *, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames)
{
  static const char *const names[] = {"dst", "src", "count", "scale", "z", "stream"};
  PyObject *v[6];
  void *dst, *src, *stream;
  if (!arguments("quantize_input_u8", names, 5, args, nargs, kwnames, v)) return nullptr;
  if (!as_pointer(v[0], &dst) || !as_pointer(v[1], &src) || !stream_or_null(v[5], &stream)) return nullptr;
  PyObject *n = PyNumber_Index(v[2]);   // (whatever converts to an int without loss, a numpy integer for instance)
  if (!n) return nullptr;
  const size_t count = PyLong_AsSize_t(n);
  Py_DECREF(n);
  if (PyErr_Occurred()) return nullptr;
  const double scale = PyFloat_AsDouble(v[3]);
  if (PyErr_Occurred()) return nullptr;
  const double z = PyFloat_AsDouble(v[4]);
  if (PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_quantize(dst, src, count, (float)scale, (float)z, stream);
  Py_END_ALLOW_THREADS
  return result(rc);
}

PyObject *reorder(const char *fn, reorder_t f, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames)
{
  static const char *const names[] = {"dst", "src", "elem_size", "n", "c", "h", "w", "stream"};
  PyObject *v[8];
  void *dst, *src, *stream;
  int d[5];
  if (!arguments(fn, names, 7, args, nargs, kwnames, v)) return nullptr;
  if (!as_pointer(v[0], &dst) || !as_pointer(v[1], &src) || !stream_or_null(v[7], &stream)) return nullptr;
  for (int i = 0; i < 5; ++i)
    if (!as_int(v[2 + i], &d[i])) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(dst, src, d[0], d[1], d[2], d[3], d[4], stream);
  Py_END_ALLOW_THREADS
  return result(rc);
}
PyObject *reorder_nchw_to_blocked(PyObject *, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames)
{
  return reorder("reorder_nchw_to_blocked", g_to_blocked, args, nargs, kwnames);
}
PyObject *reorder_blocked_to_nchw(PyObject *, PyObject *const *args, Py_ssize_t nargs, PyObject *kwnames)
{
  return reorder("reorder_blocked_to_nchw", g_to_nchw, args, nargs, kwnames);
}

// bind(execute, quantize_input_u8, reorder_nchw_to_blocked, reorder_blocked_to_nchw, linear_execute, linear_execute_experts,
// norm_execute, route_execute, raise)
PyObject *bind(PyObject *, PyObject *args)
{
  unsigned long long e, q, b, n, l, x, m, t;
  PyObject *r;
  if (!PyArg_ParseTuple(args, "KKKKKKKKO", &e, &q, &b, &n, &l, &x, &m, &t, &r)) return nullptr;
  g_execute = reinterpret_cast<execute_t>(e);
  g_quantize = reinterpret_cast<quantize_t>(q);
  g_to_blocked = reinterpret_cast<reorder_t>(b);
  g_to_nchw = reinterpret_cast<reorder_t>(n);
  g_linear = reinterpret_cast<layer_t>(l);
  g_experts = reinterpret_cast<layer_t>(x);
  g_norm = reinterpret_cast<layer_t>(m);
  g_route = reinterpret_cast<layer_t>(t);
  Py_INCREF(r);
  Py_XSETREF(g_raise, r);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "addresses of the library's functions, and what raises for a status"},
    {"quantize_input_u8", EHIP_FAST(quantize_input_u8), "quantize_input_u8(dst, src, count, scale, z, stream=0)"},
    {"reorder_nchw_to_blocked", EHIP_FAST(reorder_nchw_to_blocked), "reorder_nchw_to_blocked(dst, src, elem_size, n, c, h, w, stream=0)"},
    {"reorder_blocked_to_nchw", EHIP_FAST(reorder_blocked_to_nchw), "reorder_blocked_to_nchw(dst, src, elem_size, n, c, h, w, stream=0)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ehip_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ehip_call(void)
{
  const struct {
    PyTypeObject *type;
    const char *name;
    PyMethodDef *methods;
  } bases[] = {{&conv_type, "_ehip_call.ConvBase", conv_methods}, {&linear_type, "_ehip_call.LinearBase", linear_methods},
               {&norm_type, "_ehip_call.NormBase", norm_methods}, {&route_type, "_ehip_call.RouterBase", route_methods}};
  for (const auto &b : bases) {
    b.type->tp_name = b.name;
    b.type->tp_basicsize = sizeof(ConvBase);
    b.type->tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE;
    b.type->tp_new = PyType_GenericNew;
    b.type->tp_methods = b.methods;
    b.type->tp_getset = conv_getset;
    if (PyType_Ready(b.type) < 0) return nullptr;
  }
  g_data_ptr = PyUnicode_InternFromString("data_ptr");
  if (!g_data_ptr) return nullptr;
  PyObject *m = PyModule_Create(&module);
  if (!m) return nullptr;
  for (const auto &b : bases) {
    Py_INCREF(b.type);
    if (PyModule_AddObject(m, strrchr(b.name, '.') + 1, reinterpret_cast<PyObject *>(b.type)) < 0) {
      Py_DECREF(b.type);
      Py_DECREF(m);
      return nullptr;
    }
  }
  return m;
}
