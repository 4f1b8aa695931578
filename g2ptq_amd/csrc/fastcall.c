/*
 * _fastcall: CPython fast-call bindings of the C-ABI entry points that are
 * called once per batch or token: the calibration hooks' g2ptq_hessian_stage,
 * for callers that deliver many small batches (an MoE block's routed tokens:
 * thousands of add_batch calls per layer), and what a decoding step calls for
 * every layer (8-bit linears, the paged cache and attention over it), where
 * ctypes' conversions cost more than a small launch.  Each function takes the same arguments as
 * the entry point, as Python integers (pointers and streams as addresses),
 * and returns its status; the caller raises on a nonzero status exactly as
 * for the ctypes binding.  It calls the entry point of libg2ptq_hip.so
 * (linked, resolved next to this module) and adds no logic of its own.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/g2ptq_hip.h"

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

/* hessian_stage(stream, X, T, C, ldx, XT, ldt, t_off) -> status */
static PyObject* hessian_stage(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 8) {
    PyErr_SetString(PyExc_TypeError, "hessian_stage takes 8 arguments");
    return NULL;
  }
  void *stream, *X, *XT;
  int64_t T, C, ldx, ldt, t_off;
  if (as_ptr(args[0], &stream) || as_ptr(args[1], &X) || as_i64(args[2], &T) ||
      as_i64(args[3], &C) || as_i64(args[4], &ldx) || as_ptr(args[5], &XT) ||
      as_i64(args[6], &ldt) || as_i64(args[7], &t_off))
    return NULL;
  const int status = g2ptq_hessian_stage(stream, (const uint16_t*)X, T, C, ldx, (uint16_t*)XT,
                                         ldt, t_off);
  return PyLong_FromLong(status);
}

static int as_int(PyObject* o, int* out) {
  int64_t v;
  if (as_i64(o, &v)) return -1;
  *out = (int)v;
  return 0;
}

static int as_f32(PyObject* o, float* out) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) return -1;
  *out = (float)v;
  return 0;
}

static int count(Py_ssize_t nargs, Py_ssize_t want, const char* name) {
  if (nargs == want) return 0;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, want);
  return -1;
}

/* int8_linear(stream, x, dtype, T, K, ldx, sym, W, ldw, wscale, wsum, bias, N, out, ldo, ws,
 * ws_bytes) -> status */
static PyObject* int8_linear(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *x, *W, *wscale, *wsum, *bias, *out, *ws;
  int64_t T, K, ldx, ldw, N, ldo, ws_bytes;
  int dtype, sym;
  if (count(nargs, 17, "int8_linear") || as_ptr(a[0], &stream) || as_ptr(a[1], &x) ||
      as_int(a[2], &dtype) || as_i64(a[3], &T) || as_i64(a[4], &K) || as_i64(a[5], &ldx) ||
      as_int(a[6], &sym) || as_ptr(a[7], &W) || as_i64(a[8], &ldw) || as_ptr(a[9], &wscale) ||
      as_ptr(a[10], &wsum) || as_ptr(a[11], &bias) || as_i64(a[12], &N) || as_ptr(a[13], &out) ||
      as_i64(a[14], &ldo) || as_ptr(a[15], &ws) || as_i64(a[16], &ws_bytes))
    return NULL;
  return PyLong_FromLong(g2ptq_int8_linear(stream, x, dtype, T, K, ldx, sym, (const int8_t*)W, ldw,
                                           (const float*)wscale, (const int32_t*)wsum,
                                           (const float*)bias, N, out, ldo, ws,
                                           (size_t)ws_bytes));
}

/* int8_linear_workspace(T, N, K) -> bytes, or a negative status */
static PyObject* int8_linear_workspace(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  int64_t T, N, K;
  size_t bytes = 0;
  if (count(nargs, 3, "int8_linear_workspace") || as_i64(a[0], &T) || as_i64(a[1], &N) ||
      as_i64(a[2], &K))
    return NULL;
  const int status = g2ptq_int8_linear_workspace(T, N, K, &bytes);
  return PyLong_FromLongLong(status ? status : (long long)bytes);
}

/* kv_write(stream, cache, k, k_token, k_head, v, v_token, v_head, dtype, T, slots) -> status */
static PyObject* kv_write(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *cache, *k, *v, *slots;
  int64_t kt, kh, vt, vh, T;
  int dtype;
  if (count(nargs, 11, "kv_write") || as_ptr(a[0], &stream) || as_ptr(a[1], &cache) ||
      as_ptr(a[2], &k) || as_i64(a[3], &kt) || as_i64(a[4], &kh) || as_ptr(a[5], &v) ||
      as_i64(a[6], &vt) || as_i64(a[7], &vh) || as_int(a[8], &dtype) || as_i64(a[9], &T) ||
      as_ptr(a[10], &slots))
    return NULL;
  return PyLong_FromLong(g2ptq_kv_write(stream, (const g2ptq_kv_cache*)cache, k, kt, kh, v, vt, vh,
                                        dtype, T, (const int64_t*)slots));
}

/* kv_read(stream, cache, table, ldt, B, width, cu, total, k, v, dtype) -> status */
static PyObject* kv_read(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *cache, *table, *cu, *k, *v;
  int64_t ldt, B, width, total;
  int dtype;
  if (count(nargs, 11, "kv_read") || as_ptr(a[0], &stream) || as_ptr(a[1], &cache) ||
      as_ptr(a[2], &table) || as_i64(a[3], &ldt) || as_i64(a[4], &B) || as_i64(a[5], &width) ||
      as_ptr(a[6], &cu) || as_i64(a[7], &total) || as_ptr(a[8], &k) || as_ptr(a[9], &v) ||
      as_int(a[10], &dtype))
    return NULL;
  return PyLong_FromLong(g2ptq_kv_read(stream, (const g2ptq_kv_cache*)cache, (const int32_t*)table,
                                       ldt, B, width, (const int32_t*)cu, total, k, v, dtype));
}

/* paged_attention(stream, cache, q, q_token, q_head, dtype, T, Hq, table, ldt, B, width, cu_q,
 * kv_lens, max_q, max_kv, scale, out, ws, ws_bytes) -> status */
static PyObject* paged_attention(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *cache, *q, *table, *cu, *kv, *out, *ws;
  int64_t qt, qh, T, Hq, ldt, B, width, max_q, max_kv, ws_bytes;
  int dtype;
  float scale;
  if (count(nargs, 20, "paged_attention") || as_ptr(a[0], &stream) || as_ptr(a[1], &cache) ||
      as_ptr(a[2], &q) || as_i64(a[3], &qt) || as_i64(a[4], &qh) || as_int(a[5], &dtype) ||
      as_i64(a[6], &T) || as_i64(a[7], &Hq) || as_ptr(a[8], &table) || as_i64(a[9], &ldt) ||
      as_i64(a[10], &B) || as_i64(a[11], &width) || as_ptr(a[12], &cu) || as_ptr(a[13], &kv) ||
      as_i64(a[14], &max_q) || as_i64(a[15], &max_kv) || as_f32(a[16], &scale) ||
      as_ptr(a[17], &out) || as_ptr(a[18], &ws) || as_i64(a[19], &ws_bytes))
    return NULL;
  return PyLong_FromLong(g2ptq_paged_attention(
      stream, (const g2ptq_kv_cache*)cache, q, qt, qh, dtype, T, Hq, (const int32_t*)table, ldt, B,
      width, (const int32_t*)cu, (const int32_t*)kv, max_q, max_kv, scale, out, ws,
      (size_t)ws_bytes));
}

/* paged_attention_workspace(T, Hq, kv_heads, dim, B, max_q, max_kv) -> bytes, or a negative
 * status */
static PyObject* paged_attention_workspace(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  int64_t v[7];
  size_t bytes = 0;
  if (count(nargs, 7, "paged_attention_workspace")) return NULL;
  for (int i = 0; i < 7; ++i)
    if (as_i64(a[i], &v[i])) return NULL;
  const int status =
      g2ptq_paged_attention_workspace(v[0], v[1], v[2], v[3], v[4], v[5], v[6], &bytes);
  return PyLong_FromLongLong(status ? status : (long long)bytes);
}

/* rms_norm(stream, x, x_outer, x_inner, r, r_outer, r_inner, dtype, w, wtype, rows, inner, C, eps,
 * y, sum, sym, codes, ldc, scale, zero) -> status */
static PyObject* rms_norm(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *x, *r, *w, *y, *sum, *codes, *scale, *zero;
  int64_t xo, xi, ro, ri, rows, inner, C, ldc;
  int dtype, wtype, sym;
  float eps;
  if (count(nargs, 21, "rms_norm") || as_ptr(a[0], &stream) || as_ptr(a[1], &x) ||
      as_i64(a[2], &xo) || as_i64(a[3], &xi) || as_ptr(a[4], &r) || as_i64(a[5], &ro) ||
      as_i64(a[6], &ri) || as_int(a[7], &dtype) || as_ptr(a[8], &w) || as_int(a[9], &wtype) ||
      as_i64(a[10], &rows) || as_i64(a[11], &inner) || as_i64(a[12], &C) || as_f32(a[13], &eps) ||
      as_ptr(a[14], &y) || as_ptr(a[15], &sum) || as_int(a[16], &sym) || as_ptr(a[17], &codes) ||
      as_i64(a[18], &ldc) || as_ptr(a[19], &scale) || as_ptr(a[20], &zero))
    return NULL;
  return PyLong_FromLong(g2ptq_rms_norm(stream, x, xo, xi, r, ro, ri, dtype, w, wtype, rows, inner,
                                        C, eps, y, sum, sym, (int8_t*)codes, ldc, (float*)scale,
                                        (float*)zero));
}

/* dequantize_tokens(stream, codes, ldc, scale, zero, T, K, out, dtype) -> status */
static PyObject* dequantize_tokens(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *codes, *scale, *zero, *out;
  int64_t ldc, T, K;
  int dtype;
  if (count(nargs, 9, "dequantize_tokens") || as_ptr(a[0], &stream) || as_ptr(a[1], &codes) ||
      as_i64(a[2], &ldc) || as_ptr(a[3], &scale) || as_ptr(a[4], &zero) || as_i64(a[5], &T) ||
      as_i64(a[6], &K) || as_ptr(a[7], &out) || as_int(a[8], &dtype))
    return NULL;
  return PyLong_FromLong(g2ptq_dequantize_tokens(stream, (const int8_t*)codes, ldc,
                                                 (const float*)scale, (const float*)zero, T, K,
                                                 out, dtype));
}

/* rotary(stream, q, q_token, q_head, q_heads, k, k_token, k_head, k_heads, dtype, T, dim, n,
 * interleaved, positions, freq, factor, q_out, k_out) -> status */
static PyObject* rotary(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *q, *k, *positions, *freq, *q_out, *k_out;
  int64_t qt, qh, Hq, kt, kh, Hk, T, dim, n;
  int dtype, interleaved;
  float factor;
  if (count(nargs, 19, "rotary") || as_ptr(a[0], &stream) || as_ptr(a[1], &q) ||
      as_i64(a[2], &qt) || as_i64(a[3], &qh) || as_i64(a[4], &Hq) || as_ptr(a[5], &k) ||
      as_i64(a[6], &kt) || as_i64(a[7], &kh) || as_i64(a[8], &Hk) || as_int(a[9], &dtype) ||
      as_i64(a[10], &T) || as_i64(a[11], &dim) || as_i64(a[12], &n) ||
      as_int(a[13], &interleaved) || as_ptr(a[14], &positions) || as_ptr(a[15], &freq) ||
      as_f32(a[16], &factor) || as_ptr(a[17], &q_out) || as_ptr(a[18], &k_out))
    return NULL;
  return PyLong_FromLong(g2ptq_rotary(stream, q, qt, qh, Hq, k, kt, kh, Hk, dtype, T, dim, n,
                                      interleaved, (const int64_t*)positions, (const double*)freq,
                                      factor, q_out, k_out));
}

/* pages_workspace(B) -> bytes, or a negative status */
static PyObject* pages_workspace(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  int64_t B;
  size_t bytes = 0;
  if (count(nargs, 1, "pages_workspace") || as_i64(a[0], &B)) return NULL;
  const int status = g2ptq_pages_workspace(B, &bytes);
  return PyLong_FromLongLong(status ? status : (long long)bytes);
}

/* pages_extend(stream, tables, rows, counts, B, total, table, cu, kv_lens, slots, positions, ws,
 * ws_bytes) -> status */
static PyObject* pages_extend(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *tables, *rows, *counts, *table, *cu, *kv, *slots, *positions, *ws;
  int64_t B, total, ws_bytes;
  if (count(nargs, 13, "pages_extend") || as_ptr(a[0], &stream) || as_ptr(a[1], &tables) ||
      as_ptr(a[2], &rows) || as_ptr(a[3], &counts) || as_i64(a[4], &B) || as_i64(a[5], &total) ||
      as_ptr(a[6], &table) || as_ptr(a[7], &cu) || as_ptr(a[8], &kv) || as_ptr(a[9], &slots) ||
      as_ptr(a[10], &positions) || as_ptr(a[11], &ws) || as_i64(a[12], &ws_bytes))
    return NULL;
  return PyLong_FromLong(g2ptq_pages_extend(
      stream, (const g2ptq_page_tables*)tables, (const int32_t*)rows, (const int32_t*)counts, B,
      total, (int32_t*)table, (int32_t*)cu, (int32_t*)kv, (int64_t*)slots, (int64_t*)positions, ws,
      (size_t)ws_bytes));
}

/* pages_release(stream, tables, rows, keep, B, ws, ws_bytes) -> status */
static PyObject* pages_release(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *tables, *rows, *keep, *ws;
  int64_t B, ws_bytes;
  if (count(nargs, 7, "pages_release") || as_ptr(a[0], &stream) || as_ptr(a[1], &tables) ||
      as_ptr(a[2], &rows) || as_ptr(a[3], &keep) || as_i64(a[4], &B) || as_ptr(a[5], &ws) ||
      as_i64(a[6], &ws_bytes))
    return NULL;
  return PyLong_FromLong(g2ptq_pages_release(stream, (const g2ptq_page_tables*)tables,
                                             (const int32_t*)rows, (const int32_t*)keep, B, ws,
                                             (size_t)ws_bytes));
}

/* adapters_workspace(T, K, n, R) -> bytes, or a negative status */
static PyObject* adapters_workspace(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  int64_t T, K, n, R;
  size_t bytes = 0;
  if (count(nargs, 4, "adapters_workspace") || as_i64(a[0], &T) || as_i64(a[1], &K) ||
      as_i64(a[2], &n) || as_i64(a[3], &R))
    return NULL;
  const int status = g2ptq_adapters_workspace(T, K, n, R, &bytes);
  return PyLong_FromLongLong(status ? status : (long long)bytes);
}

/* adapters(stream, set, x, ldx, index, T, base, ldb, out, ldo, ws, ws_bytes) -> status */
static PyObject* adapters(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  (void)self;
  void *stream, *set, *x, *index, *base, *out, *ws;
  int64_t ldx, T, ldb, ldo, ws_bytes;
  if (count(nargs, 12, "adapters") || as_ptr(a[0], &stream) || as_ptr(a[1], &set) ||
      as_ptr(a[2], &x) || as_i64(a[3], &ldx) || as_ptr(a[4], &index) || as_i64(a[5], &T) ||
      as_ptr(a[6], &base) || as_i64(a[7], &ldb) || as_ptr(a[8], &out) || as_i64(a[9], &ldo) ||
      as_ptr(a[10], &ws) || as_i64(a[11], &ws_bytes))
    return NULL;
  return PyLong_FromLong(g2ptq_adapters(stream, (const g2ptq_adapter_set*)set, x, ldx,
                                        (const int32_t*)index, T, base, ldb, out, ldo, ws,
                                        (size_t)ws_bytes));
}

#define FAST(name, doc) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, doc}
static PyMethodDef methods[] = {
    FAST(int8_linear, "g2ptq_int8_linear(...) -> status"),
    FAST(int8_linear_workspace, "g2ptq_int8_linear_workspace(T, N, K) -> bytes"),
    FAST(kv_write, "g2ptq_kv_write(...) -> status"),
    FAST(kv_read, "g2ptq_kv_read(...) -> status"),
    FAST(paged_attention, "g2ptq_paged_attention(...) -> status"),
    FAST(paged_attention_workspace, "g2ptq_paged_attention_workspace(...) -> bytes"),
    FAST(rms_norm, "g2ptq_rms_norm(...) -> status"),
    FAST(dequantize_tokens, "g2ptq_dequantize_tokens(...) -> status"),
    FAST(rotary, "g2ptq_rotary(...) -> status"),
    FAST(pages_workspace, "g2ptq_pages_workspace(B) -> bytes"),
    FAST(pages_extend, "g2ptq_pages_extend(...) -> status"),
    FAST(pages_release, "g2ptq_pages_release(...) -> status"),
    FAST(adapters_workspace, "g2ptq_adapters_workspace(T, K, n, R) -> bytes"),
    FAST(adapters, "g2ptq_adapters(...) -> status"),
    {"hessian_stage", (PyCFunction)(void (*)(void))hessian_stage, METH_FASTCALL,
     "g2ptq_hessian_stage(stream, X, T, C, ldx, XT, ldt, t_off) -> status"},
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", NULL, -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&module); }
