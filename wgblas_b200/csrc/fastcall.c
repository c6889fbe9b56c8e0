/*
 * _fast: the checks and calls of the resident grouped and microscaled products
 * for Python, without the interpreter's and ctypes' cost per argument (about 10
 * microseconds a call, more than the smallest products take on the GPU).
 *
 * Each function handles the ordinary call: plain ints and floats, a live device
 * that does not report times, GpuArray or contiguous CUDA tensor operands that
 * pass every check. It returns the wg_status of the call then, and None for
 * anything else, without having called the library: the Python function of the
 * same name (grouped.py, mx.py) then goes through the same checks one by one and
 * raises or calls. Nothing is accepted here that is refused there. The package does
 * without this file where it was not built for the running interpreter.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#if PY_VERSION_HEX < 0x030C0000
#include <structmember.h>
#define Py_T_OBJECT_EX T_OBJECT_EX
#endif
#include <stdint.h>

#include "wgblas.h"

/* Set once by setup(): the classes, and the type names of foreign dtype objects. */
static PyObject *t_device, *t_array, *t_mx, *foreign;
/* Interned attribute and method names. */
static PyObject *n_handle, *n_value, *n_benchmark, *n_ordinal, *n_dtype, *n_is_cuda, *n_data_ptr, *n_get_device,
    *n_is_contiguous, *n_numel;
/* Where GpuArray and GpuMxMatrix objects keep their __slots__ (asked of the classes by
 * setup(): an attribute lookup for each of a matrix's nine costs 0.3 microseconds). */
static Py_ssize_t a_device, a_ptr, a_length, a_dtype, m_device, m_rows, m_cols, m_batch, m_groups, m_codes, m_scales,
    m_pcodes, m_pscales;

enum { T_F32 = WG_TYPE_F32, T_BF16 = WG_TYPE_BF16, T_F16 = WG_TYPE_F16, T_I32 = 3, T_U8 = 4 };
static const int item_bytes[] = {4, 2, 2, 4, 1};

typedef struct {
  uintptr_t p;
  int64_t n;
  int type;
} operand;

typedef struct {
  PyObject *obj;
  wg_device *handle;
  int64_t ordinal;
} device;

/* ---- reading Python objects: 1 on success, 0 (no exception set) otherwise ---- */

static int get_i64(PyObject *x, int64_t *out) {
  if (!x || !PyLong_CheckExact(x)) return 0;
  int over = 0;
  *out = PyLong_AsLongLongAndOverflow(x, &over);
  return !over;
}

static int attr_i64(PyObject *x, PyObject *name, int64_t *out) {
  PyObject *v = PyObject_GetAttr(x, name);
  int ok = get_i64(v, out);
  Py_XDECREF(v);
  if (!v) PyErr_Clear();
  return ok;
}

static int get_ptr(PyObject *v, uintptr_t *out) {
  if (!v || !PyLong_CheckExact(v)) return 0;
  *out = (uintptr_t)PyLong_AsUnsignedLongLong(v);
  if (*out != (uintptr_t)-1 || !PyErr_Occurred()) return 1;
  PyErr_Clear();
  return 0;
}

static int attr_ptr(PyObject *x, PyObject *name, uintptr_t *out) {
  PyObject *v = PyObject_GetAttr(x, name);
  int ok = get_ptr(v, out);
  Py_XDECREF(v);
  PyErr_Clear();
  return ok;
}

/* A slot's object (borrowed; NULL when it was never set). */
static PyObject *slot(PyObject *x, Py_ssize_t at) { return *(PyObject **)((char *)x + at); }

static int call_i64(PyObject *x, PyObject *method, int64_t *out) {
  PyObject *v = PyObject_CallMethodNoArgs(x, method);
  int ok = get_i64(v, out);
  Py_XDECREF(v);
  if (!v) PyErr_Clear();
  return ok;
}

static int is_true(PyObject *v) { /* steals v */
  int ok = v == Py_True;
  Py_XDECREF(v);
  if (!v) PyErr_Clear();
  return ok;
}

/* A finite Python float (alpha, beta). */
static int get_scalar(PyObject *x, float *out) {
  if (!PyFloat_CheckExact(x)) return 0;
  const double v = PyFloat_AS_DOUBLE(x);
  *out = (float)v;
  return v - v == 0.0;
}

static int get_trans(PyObject *x, int *out) {
  if (!PyUnicode_CheckExact(x)) return 0;
  if (PyUnicode_CompareWithASCIIString(x, "transpose") == 0) *out = 1;
  else if (PyUnicode_CompareWithASCIIString(x, "no-transpose") == 0) *out = 0;
  else return 0;
  return 1;
}

static int type_of(PyObject *name) {
  if (!name || !PyUnicode_CheckExact(name)) return -1;
  static const char *const names[] = {"float32", "bfloat16", "float16", "int32", "uint8"};
  for (int i = 0; i < 5; i++)
    if (PyUnicode_CompareWithASCIIString(name, names[i]) == 0) return i;
  return -1;
}

/* A live device that init() made without benchmark=True. */
static int get_device(PyObject *x, device *out) {
  if (!t_device || (PyObject *)Py_TYPE(x) != t_device) return 0;
  PyObject *b = PyObject_GetAttr(x, n_benchmark);
  Py_XDECREF(b);
  if (b != Py_False) {
    PyErr_Clear();
    return 0;
  }
  PyObject *h = PyObject_GetAttr(x, n_handle);
  uintptr_t p = 0;
  int ok = h && h != Py_None && attr_ptr(h, n_value, &p) && p;
  Py_XDECREF(h);
  PyErr_Clear();
  if (!ok || !attr_i64(x, n_ordinal, &out->ordinal)) return 0;
  out->obj = x;
  out->handle = (wg_device *)p;
  return 1;
}

static int get_operand(const device *d, PyObject *x, operand *out) {
  if ((PyObject *)Py_TYPE(x) == t_array) {
    out->type = type_of(slot(x, a_dtype));
    return slot(x, a_device) == d->obj && out->type >= 0 && get_ptr(slot(x, a_ptr), &out->p) && out->p &&
           get_i64(slot(x, a_length), &out->n);
  }
  if (!is_true(PyObject_GetAttr(x, n_is_cuda))) return 0;
  PyObject *dtype = PyObject_GetAttr(x, n_dtype);
  if (!dtype) {
    PyErr_Clear();
    return 0;
  }
  out->type = type_of(PyDict_GetItem(foreign, dtype)); /* (borrowed; absent: the Python path meets it first) */
  Py_DECREF(dtype);
  int64_t at, dev;
  if (out->type < 0 || !call_i64(x, n_get_device, &dev) || dev != d->ordinal || !call_i64(x, n_data_ptr, &at) ||
      !call_i64(x, n_numel, &out->n))
    return 0;
  out->p = (uintptr_t)at;
  return is_true(PyObject_CallMethodNoArgs(x, n_is_contiguous));
}

typedef struct {
  int64_t rows, cols, batch, groups;
  uintptr_t codes, scales;
} mx;

static int live(PyObject *x) { /* a GpuArray that was not destroyed, or another's tensor */
  uintptr_t p = 0;
  return x && ((PyObject *)Py_TYPE(x) != t_array || (get_ptr(slot(x, a_ptr), &p) && p));
}

static int get_mx(const device *d, PyObject *x, mx *out) {
  return (PyObject *)Py_TYPE(x) == t_mx && slot(x, m_device) == d->obj && get_i64(slot(x, m_rows), &out->rows) &&
         get_i64(slot(x, m_cols), &out->cols) && get_i64(slot(x, m_batch), &out->batch) &&
         get_i64(slot(x, m_groups), &out->groups) && get_ptr(slot(x, m_pcodes), &out->codes) &&
         get_ptr(slot(x, m_pscales), &out->scales) && live(slot(x, m_codes)) && live(slot(x, m_scales));
}

/* ---- sizes ------------------------------------------------------------------ */

/* Sizes and strides a call may have, so that the products below stay in 64 bits
 * (larger ones take the Python path, whose integers do not overflow). */
static int small(int64_t v) { return v >= 0 && v < ((int64_t)1 << 31); }
static int stride_ok(int64_t v) { return v >= 0 && v < ((int64_t)1 << 40); }

/* Elements from a matrix's first to its last; -1 when that leaves 62 bits. */
static int64_t span(int64_t rows, int64_t cols, int64_t ld) {
  if (rows <= 0 || cols <= 0) return 0;
  const __int128 v = (__int128)(rows - 1) * ld + cols;
  return v < ((__int128)1 << 61) ? (int64_t)v : -1;
}
static int64_t plus(int64_t a, int64_t count, int64_t stride) {
  if (a < 0) return -1;
  const __int128 v = (__int128)a + (__int128)count * stride;
  return v < ((__int128)1 << 61) ? (int64_t)v : -1;
}
static int apart(uintptr_t p, int64_t bytes, uintptr_t q, int64_t qbytes) {
  return !(p < q + (uintptr_t)qbytes && q < p + (uintptr_t)bytes);
}
/* No offsets, or none of them in the range: CTAs read them at different times. */
static int apart_offsets(uintptr_t p, int64_t bytes, const int *offsets, int64_t groups) {
  return !offsets || apart(p, bytes, (uintptr_t)offsets, (groups + 1) * 4);
}
static int64_t codes_size(int64_t rows, int64_t cols, int64_t batch) {
  const __int128 v = (__int128)batch * rows * ((cols + 31) / 32 * 16);
  return v < ((__int128)1 << 61) ? (int64_t)v : -1;
}
static int64_t scales_size(int64_t rows, int64_t cols, int64_t batch, int64_t groups) {
  const __int128 v = ((__int128)batch * ((rows + 127) / 128) + groups) * ((cols + 127) / 128) * 512;
  return v < ((__int128)1 << 61) ? (int64_t)v : -1;
}

static PyObject *status(wg_status st) { return PyLong_FromLong((long)st); }

/* ---- the calls ------------------------------------------------------------------ */

/* (device, transB, groups, m, n, k, alpha, A, lda, B, ldb, strideB, offsets, beta, C, ldc) */
static PyObject *gemm_grouped(PyObject *self, PyObject *const *v, Py_ssize_t nv) {
  (void)self;
  device d;
  operand A, B, C, O;
  int trans;
  float alpha, beta;
  int64_t groups, m, n, k, lda, ldb, strideB, ldc;
  if (nv != 16 || !get_device(v[0], &d) || !get_trans(v[1], &trans) || !get_i64(v[2], &groups) || !get_i64(v[3], &m) ||
      !get_i64(v[4], &n) || !get_i64(v[5], &k) || !get_scalar(v[6], &alpha) || !get_i64(v[8], &lda) ||
      !get_i64(v[10], &ldb) || !get_i64(v[11], &strideB) || !get_scalar(v[13], &beta) || !get_i64(v[15], &ldc))
    Py_RETURN_NONE;
  if (groups < 1 || groups > WG_MAX_GROUPS || m < 1 || n < 1 || !small(m) || !small(n) || !small(k) ||
      !stride_ok(lda) || !stride_ok(ldb) || !stride_ok(strideB) || !stride_ok(ldc) || alpha == 0.0f)
    Py_RETURN_NONE;
  if (!get_operand(&d, v[7], &A) || !get_operand(&d, v[9], &B) || !get_operand(&d, v[12], &O) ||
      !get_operand(&d, v[14], &C))
    Py_RETURN_NONE;
  const int64_t brows = trans ? n : k, bcols = trans ? k : n;
  const int64_t ua = span(m, k, lda), ub = plus(span(brows, bcols, ldb), k > 0 ? groups - 1 : 0, strideB),
                uc = span(m, n, ldc);
  if ((A.type != T_BF16 && A.type != T_F16) || B.type != A.type || (C.type != A.type && C.type != T_F32) ||
      O.type != T_I32 || lda < 1 || ldb < 1 || lda < k || ldb < bcols || ldc < n || ua < 0 || ub < 0 || uc < 0 ||
      A.n < ua || B.n < ub || C.n < uc || O.n < groups + 1)
    Py_RETURN_NONE;
  const int64_t cb = uc * item_bytes[C.type];
  if (!apart(C.p, cb, A.p, ua * 2) || !apart(C.p, cb, B.p, ub * 2) || !apart_offsets(C.p, cb, (const int *)O.p, groups))
    Py_RETURN_NONE;
  wg_status st;
  Py_BEGIN_ALLOW_THREADS
  st = wg_gemm_grouped_dev(d.handle, A.type, C.type, trans, groups, m, n, k, alpha, (const void *)A.p, lda,
                           (const void *)B.p, ldb, strideB, (const int *)O.p, beta, (void *)C.p, ldc, NULL);
  Py_END_ALLOW_THREADS
  return status(st);
}

/* (device, groups, m, n, k, alpha, A, lda, B, ldb, offsets, beta, C, ldc, strideC) */
static PyObject *gemm_grouped_inner(PyObject *self, PyObject *const *v, Py_ssize_t nv) {
  (void)self;
  device d;
  operand A, B, C, O;
  float alpha, beta;
  int64_t groups, m, n, k, lda, ldb, ldc, strideC;
  if (nv != 15 || !get_device(v[0], &d) || !get_i64(v[1], &groups) || !get_i64(v[2], &m) || !get_i64(v[3], &n) ||
      !get_i64(v[4], &k) || !get_scalar(v[5], &alpha) || !get_i64(v[7], &lda) || !get_i64(v[9], &ldb) ||
      !get_scalar(v[11], &beta) || !get_i64(v[13], &ldc) || !get_i64(v[14], &strideC))
    Py_RETURN_NONE;
  if (groups < 1 || groups > WG_MAX_GROUPS || m < 1 || n < 1 || !small(m) || !small(n) || !small(k) ||
      !stride_ok(lda) || !stride_ok(ldb) || !stride_ok(ldc) || !stride_ok(strideC) || alpha == 0.0f)
    Py_RETURN_NONE;
  if (!get_operand(&d, v[6], &A) || !get_operand(&d, v[8], &B) || !get_operand(&d, v[10], &O) ||
      !get_operand(&d, v[12], &C))
    Py_RETURN_NONE;
  const int64_t ua = span(k, m, lda), ub = span(k, n, ldb), one = span(m, n, ldc), uc = plus(one, groups - 1, strideC);
  if ((A.type != T_BF16 && A.type != T_F16) || B.type != A.type || (C.type != A.type && C.type != T_F32) ||
      O.type != T_I32 || lda < m || ldb < n || ldc < n || ua < 0 || ub < 0 || one < 0 || uc < 0 ||
      (groups > 1 && strideC < one) || A.n < ua || B.n < ub || C.n < uc || O.n < groups + 1)
    Py_RETURN_NONE;
  const int64_t cb = uc * item_bytes[C.type];
  if (!apart(C.p, cb, A.p, ua * 2) || !apart(C.p, cb, B.p, ub * 2) || !apart_offsets(C.p, cb, (const int *)O.p, groups))
    Py_RETURN_NONE;
  wg_status st;
  Py_BEGIN_ALLOW_THREADS
  st = wg_gemm_grouped_inner_dev(d.handle, A.type, C.type, groups, m, n, k, alpha, (const void *)A.p, lda,
                                 (const void *)B.p, ldb, (const int *)O.p, beta, (void *)C.p, ldc, strideC, NULL);
  Py_END_ALLOW_THREADS
  return status(st);
}

/* The address of offsets for a matrix with grouped rows (NULL for one without); 0 when it must be refused. */
static int get_grouping(const device *d, int64_t groups, PyObject *x, const int **out) {
  *out = NULL;
  if (groups == 0) return x == Py_None;
  operand o;
  if (x == Py_None || !get_operand(d, x, &o) || o.type != T_I32 || o.n < groups + 1) return 0;
  *out = (const int *)o.p;
  return 1;
}

/* (device, trans, rows, cols, X, ldx, out, offsets, strideX) */
static PyObject *mx_quantize(PyObject *self, PyObject *const *v, Py_ssize_t nv) {
  (void)self;
  device d;
  operand X;
  mx out;
  int trans;
  const int *off;
  int64_t rows, cols, ldx, strideX;
  if (nv != 9 || !get_device(v[0], &d) || !get_trans(v[1], &trans) || !get_i64(v[2], &rows) || !get_i64(v[3], &cols) ||
      !get_i64(v[5], &ldx) || !get_i64(v[8], &strideX))
    Py_RETURN_NONE;
  if (rows < 1 || cols < 1 || !small(rows) || !small(cols) || !stride_ok(ldx) || !stride_ok(strideX)) Py_RETURN_NONE;
  if (!get_mx(&d, v[6], &out) || out.rows != rows || out.cols != cols || out.batch < 1 || (trans && out.groups) ||
      !get_operand(&d, v[4], &X) || X.type > T_F16 || !get_grouping(&d, out.groups, v[7], &off))
    Py_RETURN_NONE;
  const int64_t srows = trans ? cols : rows, scols = trans ? rows : cols;
  if (!strideX && out.batch > 1) {
    if (ldx && srows > ((int64_t)1 << 39) / ldx) Py_RETURN_NONE;
    strideX = srows * ldx;
  }
  const int64_t used = plus(span(srows, scols, ldx), out.batch - 1, strideX);
  const int64_t nc = codes_size(rows, cols, out.batch), ns = scales_size(rows, cols, out.batch, out.groups);
  if (ldx < scols || used < 0 || X.n < used || nc < 0 || ns < 0) Py_RETURN_NONE;
  if (!apart(out.codes, nc, X.p, used * item_bytes[X.type]) || !apart(out.scales, ns, X.p, used * item_bytes[X.type]) ||
      !apart_offsets(out.codes, nc, off, out.groups) || !apart_offsets(out.scales, ns, off, out.groups))
    Py_RETURN_NONE;
  wg_status st;
  Py_BEGIN_ALLOW_THREADS
  st = wg_mx_quantize_dev(d.handle, X.type, trans, out.batch, rows, cols, (const void *)X.p, ldx, strideX, out.groups,
                          off, (void *)out.codes, (void *)out.scales, NULL);
  Py_END_ALLOW_THREADS
  return status(st);
}

/* (device, x, out, ldo, offsets, strideO) */
static PyObject *mx_dequantize(PyObject *self, PyObject *const *v, Py_ssize_t nv) {
  (void)self;
  device d;
  operand O;
  mx x;
  const int *off;
  int64_t ldo, strideO;
  if (nv != 6 || !get_device(v[0], &d) || !get_mx(&d, v[1], &x) || !get_i64(v[3], &ldo) || !get_i64(v[5], &strideO))
    Py_RETURN_NONE;
  if (x.rows < 1 || x.cols < 1 || x.batch < 1 || !small(x.rows) || !small(x.cols) || !stride_ok(ldo) ||
      !stride_ok(strideO) || ldo < x.cols)
    Py_RETURN_NONE;
  if (!get_operand(&d, v[2], &O) || O.type > T_F16 || !get_grouping(&d, x.groups, v[4], &off)) Py_RETURN_NONE;
  if (!strideO && x.batch > 1) {
    if (x.rows > ((int64_t)1 << 39) / ldo) Py_RETURN_NONE;
    strideO = x.rows * ldo;
  }
  const int64_t one = span(x.rows, x.cols, ldo), used = plus(one, x.batch - 1, strideO);
  const int64_t nc = codes_size(x.rows, x.cols, x.batch), ns = scales_size(x.rows, x.cols, x.batch, x.groups);
  if (one < 0 || used < 0 || nc < 0 || ns < 0 || (x.batch > 1 && strideO < one) || O.n < used) Py_RETURN_NONE;
  const int64_t ob = used * item_bytes[O.type];
  if (!apart(O.p, ob, x.codes, nc) || !apart(O.p, ob, x.scales, ns) || !apart_offsets(O.p, ob, off, x.groups))
    Py_RETURN_NONE;
  wg_status st;
  Py_BEGIN_ALLOW_THREADS
  st = wg_mx_dequantize_dev(d.handle, O.type, x.batch, x.rows, x.cols, (const void *)x.codes, (const void *)x.scales,
                            x.groups, off, (void *)O.p, ldo, strideO, NULL);
  Py_END_ALLOW_THREADS
  return status(st);
}

/* (device, groups, m, n, k, alpha, A, B, offsets, beta, C, ldc); groups 0 and offsets None: mxGemm */
static PyObject *mx_gemm(PyObject *self, PyObject *const *v, Py_ssize_t nv) {
  (void)self;
  device d;
  operand C;
  mx A, B;
  const int *off;
  float alpha, beta;
  int64_t groups, m, n, k, ldc;
  if (nv != 12 || !get_device(v[0], &d) || !get_i64(v[1], &groups) || !get_i64(v[2], &m) || !get_i64(v[3], &n) ||
      !get_i64(v[4], &k) || !get_scalar(v[5], &alpha) || !get_scalar(v[9], &beta) || !get_i64(v[11], &ldc))
    Py_RETURN_NONE;
  if (groups < 0 || groups > WG_MAX_GROUPS || m < 1 || n < 1 || !small(m) || !small(n) || !small(k) ||
      !stride_ok(ldc) || ldc < n)
    Py_RETURN_NONE;
  if (!get_mx(&d, v[6], &A) || !get_mx(&d, v[7], &B) || !get_grouping(&d, groups, v[8], &off) ||
      !get_operand(&d, v[10], &C) || C.type > T_F16)
    Py_RETURN_NONE;
  if (A.rows != m || A.cols != k || B.rows != n || B.cols != k || A.batch != 1 || A.groups != groups || B.groups != 0 ||
      B.batch != (groups ? groups : 1))
    Py_RETURN_NONE;
  const int64_t used = span(m, n, ldc);
  const int64_t ca = codes_size(m, k, 1), cb = codes_size(n, k, B.batch), sa = scales_size(m, k, 1, groups),
                sb = scales_size(n, k, B.batch, 0);
  if (used < 0 || C.n < used || ca < 0 || cb < 0 || sa < 0 || sb < 0) Py_RETURN_NONE;
  const int64_t bytes = used * item_bytes[C.type];
  if (!apart(C.p, bytes, A.codes, ca) || !apart(C.p, bytes, B.codes, cb) || !apart(C.p, bytes, A.scales, sa) ||
      !apart(C.p, bytes, B.scales, sb) || !apart_offsets(C.p, bytes, off, groups))
    Py_RETURN_NONE;
  wg_status st;
  Py_BEGIN_ALLOW_THREADS
  if (groups)
    st = wg_mx_gemm_grouped_dev(d.handle, C.type, groups, m, n, k, alpha, (const void *)A.codes, (const void *)A.scales,
                                (const void *)B.codes, (const void *)B.scales, off, beta, (void *)C.p, ldc, NULL);
  else
    st = wg_mx_gemm_dev(d.handle, C.type, m, n, k, alpha, (const void *)A.codes, (const void *)A.scales,
                        (const void *)B.codes, (const void *)B.scales, beta, (void *)C.p, ldc, NULL);
  Py_END_ALLOW_THREADS
  return status(st);
}

/* (device, codes, scales, rows, cols, batch, groups) -> a GpuMxMatrix over them, or None */
static PyObject *mx_wrap(PyObject *self, PyObject *const *v, Py_ssize_t nv) {
  (void)self;
  device d;
  operand c, s;
  int64_t rows, cols, batch, groups;
  if (nv != 7 || !get_device(v[0], &d) || !get_i64(v[3], &rows) || !get_i64(v[4], &cols) || !get_i64(v[5], &batch) ||
      !get_i64(v[6], &groups) || !small(rows) || !small(cols) || !small(batch) || groups < 0 ||
      groups > WG_MAX_GROUPS || (groups && batch != 1) || !get_operand(&d, v[1], &c) || !get_operand(&d, v[2], &s))
    Py_RETURN_NONE;
  const int64_t nc = codes_size(rows, cols, batch), ns = scales_size(rows, cols, batch, groups);
  if (c.type != T_U8 || s.type != T_U8 || nc < 0 || ns < 0 || c.n < nc || s.n < ns || ((c.p | s.p) & 15) ||
      !apart(c.p, nc, s.p, ns))
    Py_RETURN_NONE;
  PyTypeObject *t = (PyTypeObject *)t_mx;
  PyObject *x = t->tp_alloc(t, 0);
  if (!x) return NULL;
  PyObject *pc = PyLong_FromUnsignedLongLong(c.p), *ps = PyLong_FromUnsignedLongLong(s.p);
  if (!pc || !ps) {
    Py_XDECREF(pc);
    Py_XDECREF(ps);
    Py_DECREF(x);
    return NULL;
  }
  PyObject *const value[] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], pc, ps};
  const Py_ssize_t at[] = {m_device, m_codes, m_scales, m_rows, m_cols, m_batch, m_groups, m_pcodes, m_pscales};
  for (int i = 0; i < 9; i++) {
    if (i < 7) Py_INCREF(value[i]); /* (pc and ps are new) */
    *(PyObject **)((char *)x + at[i]) = value[i];
  }
  return x;
}

/* Where the class keeps its slot `name`; -1 with an exception set. */
static Py_ssize_t slot_of(PyObject *type, const char *name) {
  PyObject *v = PyObject_GetAttrString(type, name);
  if (!v) return -1;
  Py_ssize_t at = -1;
  if (Py_TYPE(v) == &PyMemberDescr_Type && ((PyMemberDescrObject *)v)->d_member->type == Py_T_OBJECT_EX)
    at = ((PyMemberDescrObject *)v)->d_member->offset;
  else PyErr_Format(PyExc_TypeError, "%s is not a slot", name);
  Py_DECREF(v);
  return at;
}

/* setup(Device, GpuArray, GpuMxMatrix, foreign type names) */
static PyObject *setup(PyObject *self, PyObject *args) {
  (void)self;
  PyObject *d, *a, *m, *f;
  if (!PyArg_ParseTuple(args, "O!O!O!O!", &PyType_Type, &d, &PyType_Type, &a, &PyType_Type, &m, &PyDict_Type, &f))
    return NULL;
  const struct {
    PyObject *type;
    Py_ssize_t *at;
    const char *name;
  } slots[] = {{a, &a_device, "device"}, {a, &a_ptr, "ptr"}, {a, &a_length, "length"}, {a, &a_dtype, "dtype"},
               {m, &m_device, "device"}, {m, &m_rows, "rows"}, {m, &m_cols, "cols"}, {m, &m_batch, "batch"},
               {m, &m_groups, "groups"}, {m, &m_codes, "codes"}, {m, &m_scales, "scales"}, {m, &m_pcodes, "_codes"},
               {m, &m_pscales, "_scales"}};
  for (size_t i = 0; i < sizeof slots / sizeof slots[0]; i++)
    if ((*slots[i].at = slot_of(slots[i].type, slots[i].name)) < 0) return NULL;
  Py_INCREF(d);
  Py_INCREF(a);
  Py_INCREF(m);
  Py_INCREF(f);
  t_device = d;
  t_array = a;
  t_mx = m;
  foreign = f;
  Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {FAST(gemm_grouped), FAST(gemm_grouped_inner), FAST(mx_quantize), FAST(mx_dequantize),
                                FAST(mx_gemm), FAST(mx_wrap), {"setup", setup, METH_VARARGS, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fast(void) {
  static struct {
    PyObject **at;
    const char *name;
  } const table[] = {{&n_handle, "_handle"}, {&n_value, "value"}, {&n_benchmark, "benchmark"}, {&n_ordinal, "ordinal"},
                     {&n_dtype, "dtype"}, {&n_is_cuda, "is_cuda"}, {&n_data_ptr, "data_ptr"},
                     {&n_get_device, "get_device"}, {&n_is_contiguous, "is_contiguous"}, {&n_numel, "numel"}};
  for (size_t i = 0; i < sizeof table / sizeof table[0]; i++)
    if (!(*table[i].at = PyUnicode_InternFromString(table[i].name))) return NULL;
  return PyModule_Create(&module);
}
