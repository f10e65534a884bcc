/* The calls of the Python mirror that a program makes many of, as native callables: borrowing an array, giving one
 * back, describing it (__cuda_array_interface__), and entry points with their results.  A call through ctypes converts its
 * arguments one object at a time, which at the smallest sizes takes longer than the entry point itself.
 *
 *   Fn("new_raw", addr)                       (ctx, devptr, dim0[, dim1[, dim2]]) -> array
 *   Fn("free", addr)                          (ctx, array) -> status
 *   Fn("interface", shape, raw, rank, typestr)  (ctx, array) -> dict
 *   Fn("array", entry, float_first)           (ctx, args...) -> array, or the negative status
 *   Fn("record", entry, float_first, free, project_0, ...)   (ctx, args...) -> tuple of arrays, or the negative status
 *
 * Arrays and contexts are addresses as Python integers.  Functions are addresses in libfuthark_b200.so. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

enum { K_NEW_RAW, K_FREE, K_INTERFACE, K_ARRAY, K_RECORD };
#define MAX_ARGS 6
#define MAX_FIELDS 4

typedef struct {
  PyObject_HEAD
  vectorcallfunc call;
  int kind, float_first, rank, fields;
  void *fn, *fn2;                 /* the function; values_raw / the record's free */
  void *project[MAX_FIELDS];
  PyObject *typestr;
} Fn;

static PyObject *s_shape, *s_typestr, *s_data, *s_version, *s_two;

static void *as_ptr(PyObject *o) { return PyLong_AsVoidPtr(o); }

static PyObject *interface(Fn *f, void *ctx, void *arr) {
  const int64_t *shape = ((const int64_t *(*)(void *, void *))f->fn)(ctx, arr);
  const uint64_t raw = ((uint64_t (*)(void *, void *))f->fn2)(ctx, arr);
  PyObject *dims = PyTuple_New(f->rank), *data = NULL, *d = NULL, *addr = NULL;
  if (dims == NULL) return NULL;
  for (int i = 0; i < f->rank; i++) {
    PyObject *n = PyLong_FromLongLong(shape[i]);
    if (n == NULL) goto done;
    PyTuple_SET_ITEM(dims, i, n);
  }
  addr = PyLong_FromUnsignedLongLong(raw);
  if (addr == NULL) goto done;
  data = PyTuple_Pack(2, addr, Py_False);
  d = PyDict_New();
  if (data == NULL || d == NULL || PyDict_SetItem(d, s_shape, dims) || PyDict_SetItem(d, s_typestr, f->typestr) ||
      PyDict_SetItem(d, s_data, data) || PyDict_SetItem(d, s_version, s_two))
    Py_CLEAR(d);
done:
  Py_XDECREF(addr);
  Py_XDECREF(data);
  Py_DECREF(dims);
  return d;
}

typedef void *P;
/* an entry point: (ctx, &out, [float,] arrays...) */
static int enter(Fn *f, P ctx, P *out, float x, const P *a, int n) {
#define T1 P
#define T2 T1, P
#define T3 T2, P
#define T4 T3, P
#define T5 T4, P
#define T6 T5, P
#define A1 a[0]
#define A2 A1, a[1]
#define A3 A2, a[2]
#define A4 A3, a[3]
#define A5 A4, a[4]
#define A6 A5, a[5]
#define CASE(N)                                                                                     \
  case N:                                                                                           \
    return f->float_first ? ((int (*)(P, P *, float, T##N))f->fn)(ctx, out, x, A##N)                \
                          : ((int (*)(P, P *, T##N))f->fn)(ctx, out, A##N);
  switch (n) {
    CASE(1) CASE(2) CASE(3) CASE(4) CASE(5) CASE(6)
  }
  return -1;
}

static PyObject *fn_call(PyObject *self, PyObject *const *args, size_t nargsf, PyObject *kwnames) {
  Fn *f = (Fn *)self;
  const Py_ssize_t n = PyVectorcall_NARGS(nargsf);
  if (kwnames != NULL && PyTuple_GET_SIZE(kwnames) > 0) { PyErr_SetString(PyExc_TypeError, "no keywords"); return NULL; }
  if (n < 2) { PyErr_SetString(PyExc_TypeError, "a context and at least one argument are wanted"); return NULL; }
  P ctx = as_ptr(args[0]);
  if (ctx == NULL) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "the context is closed");
    return NULL;
  }
  if (f->kind == K_NEW_RAW) {
    if (n < 3 || n > 5) { PyErr_SetString(PyExc_TypeError, "an address and one to three dimensions are wanted"); return NULL; }
    if (n - 2 != f->rank) { PyErr_Format(PyExc_TypeError, "%d dimensions are wanted, got %zd", f->rank, n - 2); return NULL; }
    const uint64_t dev = PyLong_AsUnsignedLongLong(args[1]);
    int64_t d[3] = {0, 0, 0};
    for (int i = 0; i < f->rank; i++) d[i] = PyLong_AsLongLong(args[2 + i]);
    if (PyErr_Occurred()) return NULL;
    P r;
    if (f->rank == 1) r = ((P (*)(P, uint64_t, int64_t))f->fn)(ctx, dev, d[0]);
    else if (f->rank == 2) r = ((P (*)(P, uint64_t, int64_t, int64_t))f->fn)(ctx, dev, d[0], d[1]);
    else r = ((P (*)(P, uint64_t, int64_t, int64_t, int64_t))f->fn)(ctx, dev, d[0], d[1], d[2]);
    return PyLong_FromVoidPtr(r);
  }
  if (f->kind == K_FREE || f->kind == K_INTERFACE) {
    if (n != 2) { PyErr_SetString(PyExc_TypeError, "a context and an array are wanted"); return NULL; }
    P arr = as_ptr(args[1]);
    if (arr == NULL) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "the array has been freed");
      return NULL;
    }
    if (f->kind == K_INTERFACE) return interface(f, ctx, arr);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = ((int (*)(P, P))f->fn)(ctx, arr);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  }
  /* entry points */
  P a[MAX_ARGS], out = NULL, parts[MAX_FIELDS] = {NULL, NULL, NULL, NULL};
  float x = 0.f;
  Py_ssize_t k = 1;
  if (f->float_first) x = (float)PyFloat_AsDouble(args[k++]);
  if (n - k > MAX_ARGS) { PyErr_SetString(PyExc_TypeError, "too many arguments"); return NULL; }
  int m = 0;
  for (; k < n; k++) {
    a[m] = as_ptr(args[k]);
    if (a[m] == NULL && !PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an array has been freed");
    if (PyErr_Occurred()) return NULL;
    m++;
  }
  if (m == 0 && !PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "an array is wanted");
  if (PyErr_Occurred()) return NULL;
  int rc, bad = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = enter(f, ctx, &out, x, a, m);
  if (rc == 0 && f->kind == K_RECORD) {
    for (int i = 0; i < f->fields; i++) bad |= ((int (*)(P, P *, P))f->project[i])(ctx, &parts[i], out);
    ((int (*)(P, P))f->fn2)(ctx, out);
  }
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(-(long)(rc < 0 ? -rc : rc));
  if (f->kind == K_ARRAY) return PyLong_FromVoidPtr(out);
  if (bad) { PyErr_NoMemory(); return NULL; }
  PyObject *t = PyTuple_New(f->fields);
  for (int i = 0; t != NULL && i < f->fields; i++) {
    PyObject *p = PyLong_FromVoidPtr(parts[i]);
    if (p == NULL) Py_CLEAR(t);
    else PyTuple_SET_ITEM(t, i, p);
  }
  return t;
}

static PyObject *fn_new(PyTypeObject *type, PyObject *args, PyObject *kw) {
  (void)kw;
  const Py_ssize_t n = PyTuple_GET_SIZE(args);
  if (n < 2 || !PyUnicode_Check(PyTuple_GET_ITEM(args, 0))) { PyErr_SetString(PyExc_TypeError, "a kind and an address are wanted"); return NULL; }
  const char *kind = PyUnicode_AsUTF8(PyTuple_GET_ITEM(args, 0));
  Fn *f = (Fn *)type->tp_alloc(type, 0);
  if (f == NULL) return NULL;
  f->call = fn_call;
  f->fn = as_ptr(PyTuple_GET_ITEM(args, 1));
#define ARG(i) PyTuple_GET_ITEM(args, i)
  if (strcmp(kind, "new_raw") == 0 && n == 3) {
    f->kind = K_NEW_RAW;
    f->rank = (int)PyLong_AsLong(ARG(2));
    if (f->rank < 1 || f->rank > 3) goto bad;
  } else if (strcmp(kind, "free") == 0 && n == 2) {
    f->kind = K_FREE;
  } else if (strcmp(kind, "interface") == 0 && n == 5) {
    f->kind = K_INTERFACE;
    f->fn2 = as_ptr(ARG(2));
    f->rank = (int)PyLong_AsLong(ARG(3));
    f->typestr = Py_NewRef(ARG(4));
  } else if (strcmp(kind, "array") == 0 && n == 3) {
    f->kind = K_ARRAY;
    f->float_first = PyObject_IsTrue(ARG(2));
  } else if (strcmp(kind, "record") == 0 && n >= 5 && n - 4 <= MAX_FIELDS) {
    f->kind = K_RECORD;
    f->float_first = PyObject_IsTrue(ARG(2));
    f->fn2 = as_ptr(ARG(3));
    f->fields = (int)(n - 4);
    for (int i = 0; i < f->fields; i++) f->project[i] = as_ptr(ARG(4 + i));
  } else {
  bad:
    PyErr_Format(PyExc_TypeError, "no function of kind %s with %zd arguments", kind, n);
  }
#undef ARG
  if (!PyErr_Occurred() && f->fn == NULL) PyErr_SetString(PyExc_ValueError, "no address");
  if (PyErr_Occurred()) { Py_DECREF(f); return NULL; }
  return (PyObject *)f;
}

static void fn_dealloc(PyObject *self) {
  Py_XDECREF(((Fn *)self)->typestr);
  Py_TYPE(self)->tp_free(self);
}

static PyTypeObject FnType = {
    PyVarObject_HEAD_INIT(NULL, 0).tp_name = "futhark_b200._mirror.Fn",
    .tp_basicsize = sizeof(Fn),
    .tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL,
    .tp_vectorcall_offset = offsetof(Fn, call),
    .tp_call = PyVectorcall_Call,
    .tp_new = fn_new,
    .tp_dealloc = fn_dealloc,
    .tp_doc = "A function of libfuthark_b200.so",
};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mirror", "Native callables of the Python mirror", -1, NULL, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__mirror(void) {
  if (PyType_Ready(&FnType) < 0) return NULL;
  s_shape = PyUnicode_InternFromString("shape");
  s_typestr = PyUnicode_InternFromString("typestr");
  s_data = PyUnicode_InternFromString("data");
  s_version = PyUnicode_InternFromString("version");
  s_two = PyLong_FromLong(2);
  PyObject *m = PyModule_Create(&module);
  if (m == NULL || PyModule_AddObjectRef(m, "Fn", (PyObject *)&FnType) < 0) return NULL;
  return m;
}
