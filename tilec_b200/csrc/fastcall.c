/* fastcall.c -- CPython entry points for the per-call path of tilec_b200.ext.
 *
 * The same two C ABI calls the ctypes binding makes for every matrix_mul
 * (tilec_mm_workspace_bytes, tilec_mm_f32; include/tilec_mm.h), without ctypes' per-argument
 * conversion, which costs about 1.4 us of the binding's per-call time.  The functions are
 * not linked: tilec_b200._native hands over the addresses of the ones in the already
 * loaded libtilec_mm.so (install()), so both bindings drive the same library instance.
 *
 *   install(addr_mm_f32, addr_workspace_bytes) -> None
 *   mm(a, b, c, M, N, K, lda, ldb, ldc, variant, split_k, flags, ws, ws_bytes, stream) -> int
 *   ws_bytes(a, b, c, M, N, K, lda, ldb, ldc, variant, split_k, flags) -> int
 *   install_lm(addr_mm_w4, addr_ce_forward, addr_ce_backward) -> None
 *   w4(x, dtype, M, ldx, weight, scale_dtype, N, K, group, bias, out, ldo, ws, ws_bytes, stream) -> int
 *   ce_forward(x, w, target, dtype, T, V, D, ldx, ldw, ignore_index, reduction, loss, stats, ws, ws_bytes,
 *              stream) -> int
 *   ce_backward(x, w, target, dtype, T, V, D, ldx, ldw, ignore_index, reduction, stats, grad, dx, dw, ws,
 *               ws_bytes, stream) -> int
 *
 * Pointers (a, b, c, ws, stream) are Python ints (0 or None for NULL); the rest are ints.
 * Return values are the C ABI's status codes and byte counts, unchanged.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "../../include/tilec_mm.h"

typedef int (*mm_f32_fn)(const float*, const float*, float*, int64_t, int64_t, int64_t, int64_t, int64_t,
                         int64_t, const tilec_mm_cfg*, void*, size_t, void*);
typedef size_t (*ws_bytes_fn)(const float*, const float*, const float*, int64_t, int64_t, int64_t, int64_t,
                              int64_t, int64_t, const tilec_mm_cfg*);

static mm_f32_fn g_mm = NULL;
static ws_bytes_fn g_ws = NULL;

static int as_ptr(PyObject* o, void** out) {
  if (o == Py_None) {
    *out = NULL;
    return 0;
  }
  const unsigned long long v = PyLong_AsUnsignedLongLong(o);
  if (v == (unsigned long long)-1 && PyErr_Occurred()) return -1;
  *out = (void*)(uintptr_t)v;
  return 0;
}

static int as_i64(PyObject* o, int64_t* out) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) return -1;
  *out = (int64_t)v;
  return 0;
}

/* Parses the 12 leading arguments shared by mm() and ws_bytes(). */
static int parse_problem(PyObject* const* args, void** p, int64_t* d, tilec_mm_cfg* cfg) {
  for (int i = 0; i < 3; ++i)
    if (as_ptr(args[i], &p[i])) return -1;
  for (int i = 0; i < 6; ++i)
    if (as_i64(args[3 + i], &d[i])) return -1;
  int64_t v[3];
  for (int i = 0; i < 3; ++i)
    if (as_i64(args[9 + i], &v[i])) return -1;
  cfg->variant = (int32_t)v[0];
  cfg->split_k = (int32_t)v[1];
  cfg->flags = (int32_t)v[2];
  cfg->activation = 0;
  for (int i = 0; i < 4; ++i) cfg->reserved[i] = 0;
  return 0;
}

static PyObject* py_install(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "install(addr_mm_f32, addr_workspace_bytes)");
    return NULL;
  }
  void* a = NULL;
  void* b = NULL;
  if (as_ptr(args[0], &a) || as_ptr(args[1], &b)) return NULL;
  if (a == NULL || b == NULL) {
    PyErr_SetString(PyExc_ValueError, "install: null function address");
    return NULL;
  }
  g_mm = (mm_f32_fn)a;
  g_ws = (ws_bytes_fn)b;
  Py_RETURN_NONE;
}

static PyObject* py_mm(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 15) {
    PyErr_SetString(PyExc_TypeError, "mm() takes 15 arguments");
    return NULL;
  }
  if (g_mm == NULL) {
    PyErr_SetString(PyExc_RuntimeError, "tilec fastcall: install() was not called");
    return NULL;
  }
  void* p[3];
  int64_t d[6];
  tilec_mm_cfg cfg;
  if (parse_problem(args, p, d, &cfg)) return NULL;
  void* ws = NULL;
  void* stream = NULL;
  int64_t ws_bytes = 0;
  if (as_ptr(args[12], &ws) || as_i64(args[13], &ws_bytes) || as_ptr(args[14], &stream)) return NULL;
  if (ws_bytes < 0) {
    PyErr_SetString(PyExc_ValueError, "mm: negative workspace size");
    return NULL;
  }
  int rc;
  /* The GIL is released around the launch, as ctypes does, so other host threads run. */
  Py_BEGIN_ALLOW_THREADS
  rc = g_mm((const float*)p[0], (const float*)p[1], (float*)p[2], d[0], d[1], d[2], d[3], d[4], d[5], &cfg, ws,
            (size_t)ws_bytes, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyObject* py_ws_bytes(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 12) {
    PyErr_SetString(PyExc_TypeError, "ws_bytes() takes 12 arguments");
    return NULL;
  }
  if (g_ws == NULL) {
    PyErr_SetString(PyExc_RuntimeError, "tilec fastcall: install() was not called");
    return NULL;
  }
  void* p[3];
  int64_t d[6];
  tilec_mm_cfg cfg;
  if (parse_problem(args, p, d, &cfg)) return NULL;
  const size_t n = g_ws((const float*)p[0], (const float*)p[1], (const float*)p[2], d[0], d[1], d[2], d[3], d[4],
                        d[5], &cfg);
  return PyLong_FromSize_t(n);
}

typedef int (*mm_w4_fn)(const void*, int32_t, int64_t, int64_t, const void*, int32_t, int64_t, int64_t, int64_t,
                        const void*, void*, int64_t, void*, size_t, void*);
typedef int (*ce_forward_fn)(const void*, const void*, const int64_t*, int32_t, int64_t, int64_t, int64_t, int64_t,
                             int64_t, int64_t, int32_t, float*, float*, void*, size_t, void*);
typedef int (*ce_backward_fn)(const void*, const void*, const int64_t*, int32_t, int64_t, int64_t, int64_t, int64_t,
                              int64_t, int64_t, int32_t, const float*, const float*, void*, void*, void*, size_t,
                              void*);
static mm_w4_fn g_w4 = NULL;
static ce_forward_fn g_ce_forward = NULL;
static ce_backward_fn g_ce_backward = NULL;

static PyObject* py_install_lm(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void* p[3] = {NULL, NULL, NULL};
  if (nargs != 3) {
    PyErr_SetString(PyExc_TypeError, "install_lm(addr_mm_w4, addr_ce_forward, addr_ce_backward)");
    return NULL;
  }
  for (int i = 0; i < 3; ++i)
    if (as_ptr(args[i], &p[i])) return NULL;
  if (p[0] == NULL || p[1] == NULL || p[2] == NULL) {
    PyErr_SetString(PyExc_ValueError, "install_lm: null function address");
    return NULL;
  }
  g_w4 = (mm_w4_fn)p[0];
  g_ce_forward = (ce_forward_fn)p[1];
  g_ce_backward = (ce_backward_fn)p[2];
  Py_RETURN_NONE;
}

/* Parses args[at[i]] as pointers or integers. */
static int parse_at(PyObject* const* args, const int* ptr_at, int nptr, void** p, const int* int_at, int nint,
                    int64_t* v) {
  for (int i = 0; i < nptr; ++i)
    if (as_ptr(args[ptr_at[i]], &p[i])) return -1;
  for (int i = 0; i < nint; ++i)
    if (as_i64(args[int_at[i]], &v[i])) return -1;
  if (v[nint - 1] < 0) { /* the last integer is the workspace's size */
    PyErr_SetString(PyExc_ValueError, "negative workspace size");
    return -1;
  }
  return 0;
}

static PyObject* py_ce_forward(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 16 || g_ce_forward == NULL) {
    PyErr_SetString(nargs != 16 ? PyExc_TypeError : PyExc_RuntimeError,
                    nargs != 16 ? "ce_forward() takes 16 arguments" : "tilec fastcall: install_lm() was not called");
    return NULL;
  }
  static const int kPtr[7] = {0, 1, 2, 11, 12, 13, 15}, kInt[9] = {3, 4, 5, 6, 7, 8, 9, 10, 14};
  void* p[7];
  int64_t v[9];
  if (parse_at(args, kPtr, 7, p, kInt, 9, v)) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ce_forward(p[0], p[1], (const int64_t*)p[2], (int32_t)v[0], v[1], v[2], v[3], v[4], v[5], v[6],
                    (int32_t)v[7], (float*)p[3], (float*)p[4], p[5], (size_t)v[8], p[6]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyObject* py_ce_backward(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 18 || g_ce_backward == NULL) {
    PyErr_SetString(nargs != 18 ? PyExc_TypeError : PyExc_RuntimeError,
                    nargs != 18 ? "ce_backward() takes 18 arguments" : "tilec fastcall: install_lm() was not called");
    return NULL;
  }
  static const int kPtr[9] = {0, 1, 2, 11, 12, 13, 14, 15, 17}, kInt[9] = {3, 4, 5, 6, 7, 8, 9, 10, 16};
  void* p[9];
  int64_t v[9];
  if (parse_at(args, kPtr, 9, p, kInt, 9, v)) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ce_backward(p[0], p[1], (const int64_t*)p[2], (int32_t)v[0], v[1], v[2], v[3], v[4], v[5], v[6],
                     (int32_t)v[7], (const float*)p[3], (const float*)p[4], p[5], p[6], p[7], (size_t)v[8], p[8]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyObject* py_w4(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 15) {
    PyErr_SetString(PyExc_TypeError, "w4() takes 15 arguments");
    return NULL;
  }
  if (g_w4 == NULL) {
    PyErr_SetString(PyExc_RuntimeError, "tilec fastcall: install_lm() was not called");
    return NULL;
  }
  /* x, weight, bias, out, ws, stream; dtype, M, ldx, scale_dtype, N, K, group, ldo, ws_bytes */
  static const int kPtr[6] = {0, 4, 9, 10, 12, 14}, kInt[9] = {1, 2, 3, 5, 6, 7, 8, 11, 13};
  void* p[6];
  int64_t v[9];
  if (parse_at(args, kPtr, 6, p, kInt, 9, v)) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_w4(p[0], (int32_t)v[0], v[1], v[2], p[1], (int32_t)v[3], v[4], v[5], v[6], p[2], p[3], v[7], p[4],
            (size_t)v[8], p[5]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyMethodDef kMethods[] = {
    {"install", (PyCFunction)(void (*)(void))py_install, METH_FASTCALL, "install(addr_mm_f32, addr_workspace_bytes)"},
    {"mm", (PyCFunction)(void (*)(void))py_mm, METH_FASTCALL,
     "mm(a, b, c, M, N, K, lda, ldb, ldc, variant, split_k, flags, ws, ws_bytes, stream) -> status"},
    {"ws_bytes", (PyCFunction)(void (*)(void))py_ws_bytes, METH_FASTCALL,
     "ws_bytes(a, b, c, M, N, K, lda, ldb, ldc, variant, split_k, flags) -> bytes"},
    {"install_lm", (PyCFunction)(void (*)(void))py_install_lm, METH_FASTCALL,
     "install_lm(addr_mm_w4, addr_ce_forward, addr_ce_backward)"},
    {"ce_forward", (PyCFunction)(void (*)(void))py_ce_forward, METH_FASTCALL,
     "ce_forward(x, w, target, dtype, T, V, D, ldx, ldw, ignore_index, reduction, loss, stats, ws, ws_bytes, "
     "stream) -> status"},
    {"ce_backward", (PyCFunction)(void (*)(void))py_ce_backward, METH_FASTCALL,
     "ce_backward(x, w, target, dtype, T, V, D, ldx, ldw, ignore_index, reduction, stats, grad, dx, dw, ws, ws_bytes, "
     "stream) -> status"},
    {"w4", (PyCFunction)(void (*)(void))py_w4, METH_FASTCALL,
     "w4(x, dtype, M, ldx, weight, scale_dtype, N, K, group, bias, out, ldo, ws, ws_bytes, stream) -> status"},
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tilec_fast", NULL, -1, kMethods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__tilec_fast(void) { return PyModule_Create(&kModule); }
