/* The short way from Python into the C ABI, for operators whose kernels take a few microseconds: a
 * decoding step makes hundreds of calls, and filling seven lh_memref_t through ctypes costs 20 us
 * a call where this takes 3. One function, call(fn, ctx, device, scalar, operands...): reads
 * address, shape, strides, type and device of each torch tensor through its public methods,
 * calls the entry point without the interpreter lock and returns its status. ctypes remains
 * the binding of everything else (_native.py). */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/lh_b200.h"

#define MAX_OPERANDS LH_MAX_OPERANDS

static PyObject *tensor_type, *memref_type, *dtype_codes;
static PyObject *name_data_ptr, *name_get_device, *name_stride, *name_shape, *name_dtype;

static PyObject* setup(PyObject* self, PyObject* args) {
  PyObject *t, *m, *d;
  if (!PyArg_ParseTuple(args, "OOO", &t, &m, &d)) return NULL;
  Py_INCREF(t);
  Py_INCREF(m);
  Py_INCREF(d);
  Py_XSETREF(tensor_type, t);
  Py_XSETREF(memref_type, m);
  Py_XSETREF(dtype_codes, d);
  Py_RETURN_NONE;
}

/* A tuple of whole numbers into at most LH_MAX_RANK places; the length, or -1. */
static int read_tuple(PyObject* tuple, int64_t* out) {
  if (!tuple) return -1;
  if (!PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) > LH_MAX_RANK) {
    PyErr_Format(PyExc_ValueError, "operands have at most %d dimensions", LH_MAX_RANK);
    return -1;
  }
  const int n = (int)PyTuple_GET_SIZE(tuple);
  for (int i = 0; i < n; ++i) {
    out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
    if (out[i] == -1 && PyErr_Occurred()) return -1;
  }
  return n;
}

static int read_tensor(PyObject* t, long device, lh_memref_t* m) {
  PyObject* v = PyObject_CallMethodNoArgs(t, name_get_device);
  if (!v) return -1;
  const long on = PyLong_AsLong(v);
  Py_DECREF(v);
  if (on == -1 && PyErr_Occurred()) return -1;
  if (on < 0) {
    PyErr_SetString(PyExc_ValueError, "operands must be CUDA tensors: this backend has no CPU path");
    return -1;
  }
  if (on != device) {
    PyErr_Format(PyExc_ValueError, "an operand is on cuda:%ld, the context on cuda:%ld", on, device);
    return -1;
  }
  v = PyObject_GetAttr(t, name_dtype);
  if (!v) return -1;
  PyObject* code = PyDict_GetItemWithError(dtype_codes, v);
  if (!code) {
    if (!PyErr_Occurred()) PyErr_Format(PyExc_ValueError, "Unsupported dtype: %S", v);
    Py_DECREF(v);
    return -1;
  }
  Py_DECREF(v);
  m->dtype = (int32_t)PyLong_AsLong(code);
  v = PyObject_GetAttr(t, name_shape);
  m->rank = read_tuple(v, m->shape);
  Py_XDECREF(v);
  if (m->rank < 0) return -1;
  v = PyObject_CallMethodNoArgs(t, name_stride);
  const int strides = read_tuple(v, m->strides);
  Py_XDECREF(v);
  if (strides != m->rank) return -1;
  v = PyObject_CallMethodNoArgs(t, name_data_ptr);
  if (!v) return -1;
  m->allocated = m->aligned = PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  if (!m->aligned && PyErr_Occurred()) return -1;
  m->offset = 0;
  return 0;
}

typedef const lh_memref_t* M;
typedef int (*Call7)(void*, M, M, M, M, M, M, M, float);
typedef int (*Call8)(void*, M, M, M, M, M, M, M, M);

/* call(fn, ctx, device, scalar, *operands): seven operands and a float, or eight and None. */
static PyObject* call(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  const Py_ssize_t n = nargs - 4;
  if (!tensor_type || nargs < 4 || !(args[3] == Py_None ? n == 8 : n == 7)) {
    PyErr_SetString(PyExc_TypeError, "call(fn, ctx, device, scalar, operands): seven operands and a number, or eight and None");
    return NULL;
  }
  void* fn = PyLong_AsVoidPtr(args[0]);
  if (!fn) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no entry point");
    return NULL;
  }
  void* ctx = args[1] == Py_None ? NULL : PyLong_AsVoidPtr(args[1]);
  if (!ctx && PyErr_Occurred()) return NULL;
  const long device = PyLong_AsLong(args[2]);
  if (device == -1 && PyErr_Occurred()) return NULL;
  float scalar = 0.f;
  if (args[3] != Py_None) {
    const double d = PyFloat_AsDouble(args[3]);
    if (d == -1.0 && PyErr_Occurred()) return NULL;
    scalar = (float)d;
  }
  lh_memref_t m[MAX_OPERANDS];
  M p[MAX_OPERANDS];
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* t = args[4 + i];
    p[i] = NULL;
    if (t == Py_None) continue;
    memset(&m[i], 0, sizeof(m[i]));
    if ((PyObject*)Py_TYPE(t) == memref_type) {
      Py_buffer view;
      if (PyObject_GetBuffer(t, &view, PyBUF_SIMPLE)) return NULL;
      const int fits = view.len == (Py_ssize_t)sizeof(lh_memref_t);
      if (fits) memcpy(&m[i], view.buf, sizeof(lh_memref_t));
      PyBuffer_Release(&view);
      if (!fits) {
        PyErr_SetString(PyExc_TypeError, "a MemRef of another size");
        return NULL;
      }
    } else {
      const int is = PyObject_IsInstance(t, tensor_type);
      if (is < 0) return NULL;
      if (!is) {
        PyErr_Format(PyExc_TypeError, "operands are torch tensors or MemRefs, not %.100s", Py_TYPE(t)->tp_name);
        return NULL;
      }
      if (read_tensor(t, device, &m[i])) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an operand's shape and strides differ in length");
        return NULL;
      }
    }
    p[i] = &m[i];
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (n == 7) rc = ((Call7)fn)(ctx, p[0], p[1], p[2], p[3], p[4], p[5], p[6], scalar);
  else rc = ((Call8)fn)(ctx, p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyMethodDef methods[] = {
  {"setup", setup, METH_VARARGS, "setup(Tensor, MemRef, {torch dtype: lh_dtype_t})"},
  {"call", (PyCFunction)(void (*)(void))call, METH_FASTCALL, "call(fn, ctx, device, scalar, *operands) -> status"},
  {NULL, NULL, 0, NULL},
};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "lh_binding", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit_lh_binding(void) {
  name_data_ptr = PyUnicode_InternFromString("data_ptr");
  name_get_device = PyUnicode_InternFromString("get_device");
  name_stride = PyUnicode_InternFromString("stride");
  name_shape = PyUnicode_InternFromString("shape");
  name_dtype = PyUnicode_InternFromString("dtype");
  if (!name_data_ptr || !name_get_device || !name_stride || !name_shape || !name_dtype) return NULL;
  return PyModule_Create(&module);
}
