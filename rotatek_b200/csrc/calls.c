/* Python module rotatek_b200._calls: the entry points whose calls are a few
 * microseconds on the GPU, without ctypes.
 *
 * A ctypes call spends ~1.7 us on every tensor's descriptor (a struct filled from
 * Python), 26 us for the fifteen tensors of a shared decode whose kernels take 14 us.
 * Here the descriptors are filled in C, through DLPack's C exchange API, or where a tensor
 * has none from its attributes (get_device, data_ptr, dtype, shape, stride: ~0.3 us each),
 * and the C ABI function, found in the already loaded librotatek_b200.so, is called directly.
 *
 * Each function takes the C ABI's tensors in its order (None for a nullable one), then
 * its integers (addresses as integers), and returns the status code, or -1 when a
 * tensor is not on a CUDA device or two are on different ones -- the caller then raises. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <dlfcn.h>
#include <string.h>

#include "../../include/rotatek_b200.h"

/* The exchange API came with version 1.3 of dlpack.h. */
#if defined(__has_include)
#if __has_include(<ATen/dlpack.h>)
#include <ATen/dlpack.h>
#endif
#endif
#if defined(DLPACK_MAJOR_VERSION) && \
    (DLPACK_MAJOR_VERSION > 1 || (DLPACK_MAJOR_VERSION == 1 && DLPACK_MINOR_VERSION >= 3))
#define HAVE_EXCHANGE 1
#else
#define HAVE_EXCHANGE 0
#endif

#define MAX_TENSORS 16
#define MAX_DTYPES 16

static PyObject *s_get_device, *s_data_ptr, *s_dtype, *s_shape, *s_stride;
static PyObject *dtypes[MAX_DTYPES];
static int dtype_codes[MAX_DTYPES], n_dtypes;

static int (*f_shared_decode)(const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, const rtk_tensor *,
                              const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, const rtk_tensor *,
                              const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, const rtk_tensor *,
                              const rtk_tensor *, int64_t, const rtk_tensor *, void *, size_t, void *, void *);
static int (*f_append_text)(const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, const rtk_tensor *,
                            const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, void *);
static int (*f_read_text)(const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, const rtk_tensor *,
                          const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, void *);
static int (*f_verify_drafts)(const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, const rtk_tensor *,
                              const rtk_tensor *, const rtk_tensor *, const rtk_tensor *, const rtk_tensor *,
                              const rtk_tensor *, void *, size_t, void *);

static int as_int(PyObject *o, int64_t *out) {
  *out = (int64_t)PyLong_AsLongLong(o);
  return !(*out == -1 && PyErr_Occurred());
}

static int dims_of(PyObject *tuple, int64_t *out, int32_t *ndim) {
  if (tuple == NULL || !PyTuple_Check(tuple)) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "a tensor's shape and stride must be tuples");
    return 0;
  }
  const Py_ssize_t n = PyTuple_GET_SIZE(tuple);
  if (n > 4) {
    PyErr_SetString(PyExc_ValueError, "tensors of more than 4 dimensions are not supported");
    return 0;
  }
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!as_int(PyTuple_GET_ITEM(tuple, i), &out[i])) return 0;
  *ndim = (int32_t)n;
  return 1;
}

#if HAVE_EXCHANGE
/* DLPack's C exchange API of torch.Tensor: a tensor's address, type, shape and strides as one
 * C call that makes no Python object (the attributes below take seven).  NULL where this torch
 * has none. */
static const DLPackExchangeAPI *exchange;
static PyTypeObject *tensor_type;

static int dtype_of(DLDataType t) {
  if (t.lanes != 1) return -1;
  if (t.code == kDLFloat) return t.bits == 32 ? RTK_F32 : t.bits == 16 ? RTK_F16 : -1;
  if (t.code == kDLBfloat) return t.bits == 16 ? RTK_BF16 : -1;
  if (t.code == kDLInt) return t.bits == 32 ? RTK_I32 : t.bits == 64 ? RTK_I64 : -1;
  if (t.code == kDLUInt) return t.bits == 8 ? RTK_U8 : -1;
  return -1;
}

/* Descriptor by the exchange API: 1 done, 0 not possible this way (no exception is set). */
static int describe_fast(PyObject *t, rtk_tensor *d, int64_t *device) {
  DLTensor x;
  if (exchange == NULL || Py_TYPE(t) != tensor_type) return 0;
  if (exchange->dltensor_from_py_object_no_sync(t, &x) != 0) {
    PyErr_Clear();
    return 0;
  }
  if (x.ndim > 4 || (x.ndim > 0 && (x.shape == NULL || x.strides == NULL))) return 0;
  if (x.device.device_type != kDLCUDA || (*device != -2 && x.device.device_id != *device)) {
    *device = -1;
    return 1;
  }
  *device = x.device.device_id;
  d->data = (char *)x.data + x.byte_offset;
  d->dtype = dtype_of(x.dtype);
  d->ndim = x.ndim;
  for (int i = 0; i < x.ndim; ++i) {
    d->shape[i] = x.shape[i];
    d->stride[i] = x.strides[i];
  }
  return 1;
}

static void find_exchange(PyObject *type) {
  PyObject *capsule = PyObject_GetAttrString(type, "__dlpack_c_exchange_api__");
  const DLPackExchangeAPI *api =
      capsule != NULL ? (const DLPackExchangeAPI *)PyCapsule_GetPointer(capsule, "dlpack_exchange_api") : NULL;
  Py_XDECREF(capsule);                          /* the type keeps it */
  PyErr_Clear();
  if (api != NULL && api->header.version.major == DLPACK_MAJOR_VERSION) {
    Py_INCREF(type);
    tensor_type = (PyTypeObject *)type;
    exchange = api;
  }
}
#else
static int describe_fast(PyObject *t, rtk_tensor *d, int64_t *device) { return 0; }
static void find_exchange(PyObject *type) {}
#endif

/* Descriptor of tensor t; *device is the tensors' common device so far (-2: none yet, -1:
 * not one CUDA device).  Returns 0 with an exception set on failure. */
static int describe(PyObject *t, rtk_tensor *d, int64_t *device) {
  PyObject *o = PyObject_CallMethodNoArgs(t, s_get_device);
  int64_t dev = -1, ptr = 0;
  int32_t nd = 0;
  int ok = o != NULL && as_int(o, &dev);
  Py_XDECREF(o);
  if (!ok) return 0;
  if (dev < 0 || (*device != -2 && dev != *device)) dev = -1;
  *device = dev;
  if (dev < 0) return 1;
  o = PyObject_CallMethodNoArgs(t, s_data_ptr);
  if (o == NULL) return 0;
  ptr = (int64_t)PyLong_AsUnsignedLongLong(o);
  Py_DECREF(o);
  if (PyErr_Occurred()) return 0;
  d->data = (void *)(uintptr_t)ptr;
  o = PyObject_GetAttr(t, s_dtype);
  if (o == NULL) return 0;
  d->dtype = -1;
  for (int i = 0; i < n_dtypes; ++i)
    if (dtypes[i] == o) d->dtype = dtype_codes[i];
  Py_DECREF(o);
  o = PyObject_GetAttr(t, s_shape);
  ok = dims_of(o, d->shape, &nd);
  Py_XDECREF(o);
  if (!ok) return 0;
  o = PyObject_CallMethodNoArgs(t, s_stride);
  ok = dims_of(o, d->stride, &d->ndim);
  Py_XDECREF(o);
  if (ok && d->ndim != nd) {
    PyErr_SetString(PyExc_ValueError, "a tensor's shape and stride differ in length");
    return 0;
  }
  return ok;
}

/* Parse nt tensors and ni integers; 1 ready, 0 exception, -1 not one CUDA device. */
static int parse(PyObject *const *args, Py_ssize_t nargs, int nt, int ni, rtk_tensor *mem, const rtk_tensor **t,
                 int64_t *ints) {
  if (nargs != nt + ni) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", nt + ni, nargs);
    return 0;
  }
  int64_t device = -2;
  for (int i = 0; i < nt; ++i) {
    t[i] = NULL;
    if (args[i] == Py_None) continue;
    memset(&mem[i], 0, sizeof(mem[i]));
    if (!describe_fast(args[i], &mem[i], &device) && !describe(args[i], &mem[i], &device)) return 0;
    if (device < 0) return -1;
    t[i] = &mem[i];
  }
  for (int i = 0; i < ni; ++i)
    if (!as_int(args[nt + i], &ints[i])) return 0;
  return 1;
}

#define PROLOGUE(f, nt, ni)                                            \
  rtk_tensor mem[MAX_TENSORS];                                         \
  const rtk_tensor *t[MAX_TENSORS];                                    \
  int64_t v[5];                                                        \
  int code;                                                            \
  if (f == NULL) {                                                     \
    PyErr_SetString(PyExc_RuntimeError, "rotatek_b200._calls is not bound"); \
    return NULL;                                                       \
  }                                                                    \
  const int ready = parse(args, nargs, nt, ni, mem, t, v);             \
  if (ready == 0) return NULL;                                         \
  if (ready < 0) return PyLong_FromLong(-1);

static PyObject *py_shared_decode(PyObject *self, PyObject *const *args, Py_ssize_t nargs) {
  /* tensors: the first thirteen, out; integers: groups, workspace, bytes, status, stream */
  PROLOGUE(f_shared_decode, 14, 5)
  Py_BEGIN_ALLOW_THREADS
  code = f_shared_decode(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], t[9], t[10], t[11], t[12], v[0], t[13],
                         (void *)(uintptr_t)v[1], (size_t)v[2], (void *)(uintptr_t)v[3], (void *)(uintptr_t)v[4]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(code);
}

static PyObject *py_append_text(PyObject *self, PyObject *const *args, Py_ssize_t nargs) {
  PROLOGUE(f_append_text, 8, 1)
  Py_BEGIN_ALLOW_THREADS
  code = f_append_text(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], (void *)(uintptr_t)v[0]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(code);
}

static PyObject *py_read_text(PyObject *self, PyObject *const *args, Py_ssize_t nargs) {
  PROLOGUE(f_read_text, 7, 1)
  Py_BEGIN_ALLOW_THREADS
  code = f_read_text(t[0], t[1], t[2], t[3], t[4], t[5], t[6], (void *)(uintptr_t)v[0]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(code);
}

static PyObject *py_verify_drafts(PyObject *self, PyObject *const *args, Py_ssize_t nargs) {
  /* integers: workspace, bytes, stream */
  PROLOGUE(f_verify_drafts, 9, 3)
  Py_BEGIN_ALLOW_THREADS
  code = f_verify_drafts(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], (void *)(uintptr_t)v[0], (size_t)v[1],
                         (void *)(uintptr_t)v[2]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(code);
}

static int find(void *lib, const char *name, void *slot) {
  void *f = dlsym(lib, name);
  if (f == NULL) {
    PyErr_Format(PyExc_RuntimeError, "%s is not in the library", name);
    return 0;
  }
  memcpy(slot, &f, sizeof(f));
  return 1;
}

static PyObject *py_bind(PyObject *self, PyObject *args) {
  const char *path;
  PyObject *codes, *key, *value, *type;
  Py_ssize_t pos = 0;
  if (!PyArg_ParseTuple(args, "sO!O!", &path, &PyDict_Type, &codes, &PyType_Type, &type)) return NULL;
  void *lib = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (lib == NULL) {
    PyErr_SetString(PyExc_RuntimeError, dlerror());
    return NULL;
  }
  n_dtypes = 0;
  while (PyDict_Next(codes, &pos, &key, &value) && n_dtypes < MAX_DTYPES) {
    int64_t code;
    if (!as_int(value, &code)) return NULL;
    Py_INCREF(key);
    dtypes[n_dtypes] = key;
    dtype_codes[n_dtypes++] = (int)code;
  }
  if (!find(lib, "rtk_shared_decode", &f_shared_decode) || !find(lib, "rtk_append_text", &f_append_text) ||
      !find(lib, "rtk_read_text", &f_read_text) || !find(lib, "rtk_verify_drafts", &f_verify_drafts))
    return NULL;
  find_exchange(type);
  Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, "bind(path of librotatek_b200.so, {torch dtype: rtk_dtype}, torch.Tensor)"},
    {"shared_decode", (PyCFunction)(void (*)(void))py_shared_decode, METH_FASTCALL, "rtk_shared_decode"},
    {"append_text", (PyCFunction)(void (*)(void))py_append_text, METH_FASTCALL, "rtk_append_text"},
    {"read_text", (PyCFunction)(void (*)(void))py_read_text, METH_FASTCALL, "rtk_read_text"},
    {"verify_drafts", (PyCFunction)(void (*)(void))py_verify_drafts, METH_FASTCALL, "rtk_verify_drafts"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Direct calls of librotatek_b200.so.", -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__calls(void) {
  s_get_device = PyUnicode_InternFromString("get_device");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_dtype = PyUnicode_InternFromString("dtype");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  if (!s_get_device || !s_data_ptr || !s_dtype || !s_shape || !s_stride) return NULL;
  return PyModule_Create(&module);
}
