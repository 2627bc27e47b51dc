/*
 * chol_pyext.c — CPython fast-call binding of the hot C-ABI entry point, used by the
 * Python drop-in (linalg_kernels_b200/cholesky.py) instead of ctypes: one call with eight
 * integer arguments costs ~0.3 us here against several us of ctypes marshalling, which
 * matters when a whole batch of n = 32 matrices factors in ~10 us.
 *
 *   potrf_ws(A, L, batch, n, info, ws, ws_bytes, queue) -> status
 *     all arguments are Python ints (device addresses, sizes; 0 for NULL)
 *
 * The entry points of linalg_b200.h the same way, a matrix as four ints (data, ld, stride,
 * type) and the coefficients as a buffer of 3 * steps floats:
 *   orthogonalize(x[4], out[4], batch, m, n, steps, precision, ws, ws_bytes, queue, eps, coef)
 *   muon_update(param[4], grad[4], momentum[4], batch, m, n, nesterov, steps, precision, ws,
 *               ws_bytes, queue, beta, decay, rate, eps, coef)
 *   grouped_matmul(x[4], w[4], y[4], w_rows_k, offsets, offsets64, groups, rows, k, n, fill,
 *                  queue)
 *   grouped_outer(a[4], b[4], dw[4], offsets, offsets64, groups, rows, k, n, queue)
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <float.h>
#include <stdint.h>

#include "../../include/linalg_b200.h"

static PyObject* potrf_ws(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 8) {
    PyErr_SetString(PyExc_TypeError, "potrf_ws expects 8 integer arguments");
    return NULL;
  }
  unsigned long long v[8];
  for (int i = 0; i < 8; ++i) {
    v[i] = PyLong_AsUnsignedLongLongMask(args[i]);
    if (v[i] == (unsigned long long)-1 && PyErr_Occurred()) return NULL;
  }
  int st = chol_potrf_batched_ws_f32((const float*)(uintptr_t)v[0], (float*)(uintptr_t)v[1],
                                     (int64_t)v[2], (int64_t)v[3], (int*)(uintptr_t)v[4],
                                     (void*)(uintptr_t)v[5], (size_t)v[6], (void*)(uintptr_t)v[7]);
  return PyLong_FromLong(st);
}

/* args[0 .. count) as integers; args[count .. count + floats) as doubles; an optional buffer of
   coefficients after them. */
static int parse(PyObject* const* args, Py_ssize_t nargs, int count, int floats, int buffer,
                 int64_t* v, double* f, Py_buffer* coef) {
  if (nargs != count + floats + buffer) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return 0;
  }
  for (int i = 0; i < count; ++i) {
    const unsigned long long x = PyLong_AsUnsignedLongLongMask(args[i]);
    if (x == (unsigned long long)-1 && PyErr_Occurred()) return 0;
    v[i] = (int64_t)x;
  }
  for (int i = 0; i < floats; ++i) {
    f[i] = PyFloat_AsDouble(args[count + i]);
    if (f[i] == -1.0 && PyErr_Occurred()) return 0;
  }
  return !buffer || PyObject_GetBuffer(args[count + floats], coef, PyBUF_SIMPLE) == 0;
}

static linalg_matrix matrix(const int64_t* v) {
  const linalg_matrix x = {(void*)(uintptr_t)v[0], v[1], v[2], (int)v[3]};
  return x;
}
/* A positive eps stays positive: below the smallest FP32 number it would turn 0, and the zero matrix's
   0 / (0 + eps) into NaN. */
static float positive(double eps) {
  const float e = (float)eps;
  return e == 0.0f && eps > 0.0 ? FLT_TRUE_MIN : e;
}
/* The buffer holds what the call reads. */
static int enough(const Py_buffer* coef, int64_t steps) {
  return steps >= 0 && steps <= LINALG_MAX_STEPS &&
         coef->len >= (Py_ssize_t)(3 * steps * (int64_t)sizeof(float));
}

static PyObject* orthogonalize(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  int64_t v[16];
  double f[1];
  Py_buffer coef;
  (void)self;
  if (!parse(args, nargs, 16, 1, 1, v, f, &coef)) return NULL;
  const linalg_matrix x = matrix(v), out = matrix(v + 4);
  int st = CHOL_ERR_INVALID_ARG;
  if (enough(&coef, v[11]))
    st = linalg_orthogonalize(&x, &out, v[8], v[9], v[10], (int)v[11], (const float*)coef.buf,
                              positive(f[0]), (int)v[12], (void*)(uintptr_t)v[13], (size_t)v[14],
                              (void*)(uintptr_t)v[15]);
  PyBuffer_Release(&coef);
  return PyLong_FromLong(st);
}

static PyObject* muon_update(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  int64_t v[21];
  double f[4];
  Py_buffer coef;
  (void)self;
  if (!parse(args, nargs, 21, 4, 1, v, f, &coef)) return NULL;
  const linalg_matrix param = matrix(v), grad = matrix(v + 4), momentum = matrix(v + 8);
  int st = CHOL_ERR_INVALID_ARG;
  if (enough(&coef, v[16]))
    st = linalg_muon_update(&param, &grad, &momentum, v[12], v[13], v[14], f[0], (int)v[15],
                            (float)f[1], (float)f[2], (int)v[16], (const float*)coef.buf,
                            positive(f[3]), (int)v[17], (void*)(uintptr_t)v[18], (size_t)v[19],
                            (void*)(uintptr_t)v[20]);
  PyBuffer_Release(&coef);
  return PyLong_FromLong(st);
}

static PyObject* grouped_matmul(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  int64_t v[21];
  (void)self;
  if (!parse(args, nargs, 21, 0, 0, v, NULL, NULL)) return NULL;
  const linalg_matrix x = matrix(v), w = matrix(v + 4), y = matrix(v + 8);
  return PyLong_FromLong(linalg_grouped_matmul(
      &x, &w, (int)v[12], &y, (const void*)(uintptr_t)v[13], (int)v[14], v[15], v[16], v[17],
      v[18], (int)v[19], (void*)(uintptr_t)v[20]));
}

static PyObject* grouped_outer(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  int64_t v[19];
  (void)self;
  if (!parse(args, nargs, 19, 0, 0, v, NULL, NULL)) return NULL;
  const linalg_matrix a = matrix(v), b = matrix(v + 4), dw = matrix(v + 8);
  return PyLong_FromLong(linalg_grouped_outer(&a, &b, &dw, (const void*)(uintptr_t)v[12],
                                              (int)v[13], v[14], v[15], v[16], v[17],
                                              (void*)(uintptr_t)v[18]));
}

static PyMethodDef methods[] = {
    {"orthogonalize", (PyCFunction)(void (*)(void))orthogonalize, METH_FASTCALL,
     "linalg_orthogonalize with integer arguments"},
    {"muon_update", (PyCFunction)(void (*)(void))muon_update, METH_FASTCALL,
     "linalg_muon_update with integer arguments"},
    {"grouped_matmul", (PyCFunction)(void (*)(void))grouped_matmul, METH_FASTCALL,
     "linalg_grouped_matmul with integer arguments"},
    {"grouped_outer", (PyCFunction)(void (*)(void))grouped_outer, METH_FASTCALL,
     "linalg_grouped_outer with integer arguments"},
    {"potrf_ws", (PyCFunction)(void (*)(void))potrf_ws, METH_FASTCALL,
     "chol_potrf_batched_ws_f32 with integer arguments"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_cholpy", NULL, -1, methods};

PyMODINIT_FUNC PyInit__cholpy(void) { return PyModule_Create(&module); }
