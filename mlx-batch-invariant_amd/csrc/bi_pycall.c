/* bi_pycall.c — a CPython binding of the most frequently called C-ABI entry
 * points (bi_quantized_matmul, bi_matmul, bi_rms_norm, and the operators of a
 * paged serving step: bi_paged_slots, bi_rope_paged_cache, bi_rope_quantized_cache,
 * bi_read_quantized_cache, bi_attn_scored, bi_attn_pages, bi_residual_rms_norm) for
 * eager callers.
 *
 * ctypes converts every argument through its argtypes on each call (about
 * 3 us for the 15 arguments of bi_quantized_matmul); here the arguments are
 * read with one PyLong_AsLongLong each. The entry points are reached through
 * addresses the Python layer passes in once (bind), taken from its ctypes
 * handle of libbi_kernels.so, so this module has no link-time dependency on
 * the kernel library and calls exactly the functions ctypes would. Arguments
 * keep the C ABI's order and meaning (include/bi_kernels.h); None stands for
 * a NULL pointer, and what the ABI takes as a host array or struct comes as its
 * values one by one. The functions return the ABI's status code.
 *
 * The GIL is released for the library call, as ctypes does: the call can block
 * on host work (first-use code-object load, a full launch queue), and
 * bi_last_error is thread-local, so the message stays with the calling thread.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include "../../include/bi_kernels.h"

typedef int (*qmm_fn)(const void*, int64_t, const uint32_t*, const void*, const void*, void*, int64_t, int64_t,
                      int64_t, int, int, int, void*, size_t, void*);
typedef int (*mm_fn)(const void*, int64_t, const void*, int64_t, void*, int64_t, int64_t, int64_t, int, void*,
                     size_t, void*);
typedef int (*rms_fn)(const void*, int64_t, const void*, void*, int64_t, int64_t, float, int, void*);

static qmm_fn g_qmm;
static mm_fn g_mm;
static rms_fn g_rms;
static __typeof__(&bi_paged_slots) g_slots;
static __typeof__(&bi_rope_paged_cache) g_rope;
static __typeof__(&bi_attn_scored) g_scored;
static __typeof__(&bi_residual_rms_norm) g_resnorm;
static __typeof__(&bi_rope_quantized_cache) g_ropeq;
static __typeof__(&bi_read_quantized_cache) g_readq;
static __typeof__(&bi_attn_pages) g_pages;

#define PTR(v) ((void*)(intptr_t)(v))

/* Reads n integer arguments (None -> 0) into v, skipping index `skip`. */
static int read_i64(PyObject* const* args, Py_ssize_t n, Py_ssize_t want, Py_ssize_t skip, int64_t* v,
                    const char* name) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%s: %zd arguments, expected %zd", name, n, want);
    return -1;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (i == skip) continue;
    if (args[i] == Py_None) {
      v[i] = 0;
      continue;
    }
    v[i] = PyLong_AsLongLong(args[i]);
    if (v[i] == -1 && PyErr_Occurred()) return -1;
  }
  return 0;
}

static PyObject* py_bind(PyObject* self, PyObject* args) {
  unsigned long long a[10];
  (void)self;
  if (!PyArg_ParseTuple(args, "KKKKKKKKKK", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &a[7], &a[8], &a[9]))
    return NULL;
  for (int i = 0; i < 10; ++i) {
    if (!a[i]) {
      PyErr_SetString(PyExc_ValueError, "bind: null entry point");
      return NULL;
    }
  }
  g_qmm = (qmm_fn)(uintptr_t)a[0];
  g_mm = (mm_fn)(uintptr_t)a[1];
  g_rms = (rms_fn)(uintptr_t)a[2];
  g_slots = (__typeof__(g_slots))(uintptr_t)a[3];
  g_rope = (__typeof__(g_rope))(uintptr_t)a[4];
  g_scored = (__typeof__(g_scored))(uintptr_t)a[5];
  g_resnorm = (__typeof__(g_resnorm))(uintptr_t)a[6];
  g_ropeq = (__typeof__(g_ropeq))(uintptr_t)a[7];
  g_readq = (__typeof__(g_readq))(uintptr_t)a[8];
  g_pages = (__typeof__(g_pages))(uintptr_t)a[9];
  Py_RETURN_NONE;
}

static PyObject* py_quantized_matmul(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[15];
  int rc;
  (void)self;
  if (!g_qmm) {
    PyErr_SetString(PyExc_RuntimeError, "quantized_matmul: entry points not bound");
    return NULL;
  }
  if (read_i64(args, n, 15, -1, v, "quantized_matmul")) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = g_qmm(PTR(v[0]), v[1], (const uint32_t*)PTR(v[2]), PTR(v[3]), PTR(v[4]), PTR(v[5]), v[6], v[7], v[8],
             (int)v[9], (int)v[10], (int)v[11], PTR(v[12]), (size_t)v[13], PTR(v[14]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyObject* py_matmul(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[12];
  int rc;
  (void)self;
  if (!g_mm) {
    PyErr_SetString(PyExc_RuntimeError, "matmul: entry points not bound");
    return NULL;
  }
  if (read_i64(args, n, 12, -1, v, "matmul")) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = g_mm(PTR(v[0]), v[1], PTR(v[2]), v[3], PTR(v[4]), v[5], v[6], v[7], (int)v[8], PTR(v[9]), (size_t)v[10],
            PTR(v[11]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyObject* py_rms_norm(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[9];
  double eps;
  int rc;
  (void)self;
  if (!g_rms) {
    PyErr_SetString(PyExc_RuntimeError, "rms_norm: entry points not bound");
    return NULL;
  }
  if (read_i64(args, n, 9, 6, v, "rms_norm")) return NULL;
  eps = PyFloat_AsDouble(args[6]);
  if (eps == -1.0 && PyErr_Occurred()) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = g_rms(PTR(v[0]), v[1], PTR(v[2]), PTR(v[3]), v[4], v[5], (float)eps, (int)v[7], PTR(v[8]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* Arguments by the letters of `kinds`: i an integer or None into v, f a number into d. */
static int read_mixed(PyObject* const* args, Py_ssize_t n, const char* kinds, int64_t* v, double* d,
                      const char* name) {
  Py_ssize_t i = 0;
  for (; i < n && kinds[i]; ++i) {
    if (kinds[i] == 'f') {
      d[i] = PyFloat_AsDouble(args[i]);
      if (d[i] == -1.0 && PyErr_Occurred()) return -1;
    } else if (args[i] == Py_None) {
      v[i] = 0;
    } else {
      v[i] = PyLong_AsLongLong(args[i]);
      if (v[i] == -1 && PyErr_Occurred()) return -1;
    }
  }
  if (i < n || kinds[i]) {
    PyErr_Format(PyExc_TypeError, "%s: %zd arguments, expected %zd", name, n, (Py_ssize_t)strlen(kinds));
    return -1;
  }
  return 0;
}

#define NEED(fn, name)                                                           \
  if (!(fn)) {                                                                   \
    PyErr_SetString(PyExc_RuntimeError, name ": entry points not bound");        \
    return NULL;                                                                 \
  }

static PyObject* py_paged_slots(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[16];
  int rc;
  (void)self;
  NEED(g_slots, "paged_slots")
  if (read_mixed(args, n, "iiiiiiiiiiiiiiii", v, NULL, "paged_slots")) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = g_slots(PTR(v[0]), PTR(v[1]), PTR(v[2]), v[3], v[4], PTR(v[5]), v[6], PTR(v[7]), PTR(v[8]), PTR(v[9]),
               PTR(v[10]), PTR(v[11]), v[12], v[13], v[14], PTR(v[15]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* ... positions, axes, its 4 sections, slots, ... D, the 6 strides, dtype, stream */
static PyObject* py_rope_paged_cache(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[35];
  int rc;
  (void)self;
  NEED(g_rope, "rope_paged_cache")
  if (read_mixed(args, n, "iiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiii", v, NULL, "rope_paged_cache")) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = g_rope(PTR(v[0]), v[1], PTR(v[2]), v[3], PTR(v[4]), v[5], PTR(v[6]), PTR(v[7]), v[8], (int)v[9], PTR(v[10]),
              &v[12], v[11], PTR(v[16]), PTR(v[17]), PTR(v[18]), PTR(v[19]), v[20], v[21], v[22], v[23], v[24],
              v[25], v[26], &v[27], (int)v[33], PTR(v[34]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* ... D, the 9 strides, causal, scale, the 5 fields of bi_score_mod, dtype, ... */
static PyObject* py_attn_scored(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[35];
  double d[35];
  int rc;
  (void)self;
  NEED(g_scored, "attn_scored")
  if (read_mixed(args, n, "iiiiiiiiiiiiiiiiiiiiiiiiiffiiiiiiii", v, d, "attn_scored")) return NULL;
  bi_score_mod mod = {(float)d[26], PTR(v[27]), PTR(v[28]), v[29], PTR(v[30])};
  Py_BEGIN_ALLOW_THREADS
  rc = g_scored(PTR(v[0]), PTR(v[1]), PTR(v[2]), PTR(v[3]), v[4], v[5], v[6], PTR(v[7]), PTR(v[8]), v[9], v[10],
                v[11], v[12], v[13], v[14], &v[15], (int)v[24], (float)d[25], &mod, (int)v[31], PTR(v[32]),
                (size_t)v[33], PTR(v[34]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyObject* py_residual_rms_norm(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[19];
  double d[19];
  int rc;
  (void)self;
  NEED(g_resnorm, "residual_rms_norm")
  if (read_mixed(args, n, "iiiiiiiiiiiiiffiiii", v, d, "residual_rms_norm")) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = g_resnorm(PTR(v[0]), v[1], PTR(v[2]), v[3], PTR(v[4]), v[5], v[6], PTR(v[7]), PTR(v[8]), PTR(v[9]), PTR(v[10]),
                 v[11], v[12], (float)d[13], (float)d[14], (int)v[15], (int)v[16], (int)v[17], PTR(v[18]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* ... positions, axes, its 4 sections, slots, ... D, bits, group size, the 12 strides, dtype, stream */
static PyObject* py_rope_quantized_cache(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[45];
  int rc;
  (void)self;
  NEED(g_ropeq, "rope_quantized_cache")
  if (read_mixed(args, n, "iiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiii", v, NULL, "rope_quantized_cache")) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = g_ropeq(PTR(v[0]), v[1], PTR(v[2]), v[3], PTR(v[4]), v[5], PTR(v[6]), PTR(v[7]), v[8], (int)v[9], PTR(v[10]),
               &v[12], v[11], PTR(v[16]), PTR(v[17]), PTR(v[18]), PTR(v[19]), PTR(v[20]), PTR(v[21]), v[22], v[23],
               v[24], v[25], v[26], v[27], v[28], (int)v[29], v[30], &v[31], (int)v[43], PTR(v[44]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* the 4 pools, the 12 strides, block_table, ... */
static PyObject* py_read_quantized_cache(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[32];
  int rc;
  (void)self;
  NEED(g_readq, "read_quantized_cache")
  if (read_mixed(args, n, "iiiiiiiiiiiiiiiiiiiiiiiiiiiiiiii", v, NULL, "read_quantized_cache")) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = g_readq(PTR(v[0]), PTR(v[1]), PTR(v[2]), PTR(v[3]), &v[4], PTR(v[16]), v[17], v[18], v[19], PTR(v[20]),
               PTR(v[21]), PTR(v[22]), v[23], v[24], v[25], v[26], (int)v[27], v[28], (int)v[29], (int)v[30],
               PTR(v[31]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* ... L, D, the 15 strides, causal, scale, dtype, ... */
static PyObject* py_attn_pages(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  int64_t v[44];
  double d[44];
  int rc;
  (void)self;
  NEED(g_pages, "attn_pages")
  if (read_mixed(args, n, "iiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiiifiiii", v, d, "attn_pages")) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = g_pages(PTR(v[0]), PTR(v[1]), PTR(v[2]), PTR(v[3]), PTR(v[4]), (int)v[5], v[6], PTR(v[7]), v[8], v[9], v[10],
               PTR(v[11]), PTR(v[12]), PTR(v[13]), v[14], v[15], PTR(v[16]), v[17], v[18], v[19], v[20], v[21], v[22],
               &v[23], (int)v[38], (float)d[39], (int)v[40], PTR(v[41]), (size_t)v[42], PTR(v[43]));
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyMethodDef methods[] = {
    {"bind", py_bind, METH_VARARGS, "bind(...): addresses of the C-ABI entry points, in the order below"},
    {"quantized_matmul", (PyCFunction)(void (*)(void))py_quantized_matmul, METH_FASTCALL,
     "bi_quantized_matmul with the C ABI's arguments"},
    {"matmul", (PyCFunction)(void (*)(void))py_matmul, METH_FASTCALL, "bi_matmul with the C ABI's arguments"},
    {"rms_norm", (PyCFunction)(void (*)(void))py_rms_norm, METH_FASTCALL, "bi_rms_norm with the C ABI's arguments"},
    {"paged_slots", (PyCFunction)(void (*)(void))py_paged_slots, METH_FASTCALL,
     "bi_paged_slots with the C ABI's arguments"},
    {"rope_paged_cache", (PyCFunction)(void (*)(void))py_rope_paged_cache, METH_FASTCALL,
     "bi_rope_paged_cache: axes before its 4 sections, and the 6 strides, one by one"},
    {"attn_scored", (PyCFunction)(void (*)(void))py_attn_scored, METH_FASTCALL,
     "bi_attn_scored: the 9 strides and the 5 fields of bi_score_mod one by one"},
    {"residual_rms_norm", (PyCFunction)(void (*)(void))py_residual_rms_norm, METH_FASTCALL,
     "bi_residual_rms_norm with the C ABI's arguments"},
    {"rope_quantized_cache", (PyCFunction)(void (*)(void))py_rope_quantized_cache, METH_FASTCALL,
     "bi_rope_quantized_cache: axes before its 4 sections, and the 12 strides, one by one"},
    {"read_quantized_cache", (PyCFunction)(void (*)(void))py_read_quantized_cache, METH_FASTCALL,
     "bi_read_quantized_cache: the 12 strides one by one"},
    {"attn_pages", (PyCFunction)(void (*)(void))py_attn_pages, METH_FASTCALL,
     "bi_attn_pages: the 15 strides one by one"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bi_pycall", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__bi_pycall(void) { return PyModule_Create(&module); }
