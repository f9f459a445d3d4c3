// CPython entry to the calls of attention over prompts and over the 8-bit key / value cache, made once per layer: as pycall.c, which
// says why, and a module of its own because it imports other functions of the library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "tpb200.h"

static void *ptr(PyObject *o) {
    return o == Py_None ? NULL : PyLong_AsVoidPtr(o);
}
static int64_t i64(PyObject *o) { return (int64_t)PyLong_AsLongLong(o); }
static int i32(PyObject *o) { return (int)PyLong_AsLong(o); }
static float f32(PyObject *o) { return (float)PyFloat_AsDouble(o); }

// argument i as a pointer, a 64-bit or 32-bit integer, a float
#define P(i) ptr(a[i])
#define L(i) i64(a[i])
#define I(i) i32(a[i])
#define F(i) f32(a[i])
#define CHECK_ARGS(name, want)                                                                  \
    if (n != (want)) {                                                                          \
        PyErr_Format(PyExc_TypeError, name " takes %d arguments (%zd given)", (want), n);       \
        return NULL;                                                                            \
    }
#define CALL(expr)                        \
    int rc;                               \
    if (PyErr_Occurred()) return NULL;    \
    Py_BEGIN_ALLOW_THREADS                \
    rc = (expr);                          \
    Py_END_ALLOW_THREADS                  \
    return PyLong_FromLong(rc)

static PyObject *attention_packed(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    CHECK_ARGS("tpb_attention_packed", 18);
    tpb_handle_t h = (tpb_handle_t)P(0);
    void *st = P(1), *out = P(2), *q = P(4), *k = P(6), *v = P(8), *cu = P(11);
    int64_t ld_out = L(3), ld_q = L(5), ld_k = L(7), ld_v = L(9), tokens = L(13);
    int dt = I(10), n_seqs = I(12), heads = I(14), kv_heads = I(15), hd = I(16);
    float scale = F(17);
    CALL(tpb_attention_packed(h, st, out, ld_out, q, ld_q, k, ld_k, v, ld_v, dt, (const int32_t *)cu, n_seqs, tokens, heads, kv_heads, hd,
                              scale));
}

static PyObject *kv_append(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    CHECK_ARGS("tpb_kv_append", 13);
    tpb_handle_t h = (tpb_handle_t)P(0);
    void *st = P(1), *c = P(2), *k = P(4), *v = P(6), *seqs = P(9), *cu = P(10);
    int layer = I(3), dt = I(8), n_seqs = I(11);
    int64_t ld_k = L(5), ld_v = L(7), rows = L(12);
    CALL(tpb_kv_append(h, st, (const tpb_kv_cache *)c, layer, k, ld_k, v, ld_v, dt, (const int32_t *)seqs, (const int32_t *)cu, n_seqs,
                       rows));
}

static PyObject *kv_read(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    CHECK_ARGS("tpb_kv_read", 14);
    tpb_handle_t h = (tpb_handle_t)P(0);
    void *st = P(1), *c = P(2), *k = P(4), *v = P(6), *seqs = P(9), *start = P(10), *cu = P(11);
    int layer = I(3), dt = I(8), n_seqs = I(12);
    int64_t ld_k = L(5), ld_v = L(7), rows = L(13);
    CALL(tpb_kv_read(h, st, (const tpb_kv_cache *)c, layer, k, ld_k, v, ld_v, dt, (const int32_t *)seqs, (const int32_t *)start,
                     (const int32_t *)cu, n_seqs, rows));
}

static PyObject *kv_attention(PyObject *self, PyObject *const *a, Py_ssize_t n) {
    CHECK_ARGS("tpb_kv_attention", 18);
    tpb_handle_t h = (tpb_handle_t)P(0);
    void *st = P(1), *c = P(2), *out = P(4), *q = P(6), *seqs = P(9), *cu = P(10), *work = P(16);
    int layer = I(3), dt = I(8), n_seqs = I(11), heads = I(13);
    int64_t ld_out = L(5), ld_q = L(7), rows = L(12), max_len = L(15);
    size_t work_bytes = (size_t)L(17);
    float scale = F(14);
    CALL(tpb_kv_attention(h, st, (const tpb_kv_cache *)c, layer, out, ld_out, q, ld_q, dt, (const int32_t *)seqs, (const int32_t *)cu,
                          n_seqs, rows, heads, scale, max_len, work, work_bytes));
}

static PyMethodDef methods[] = {
    {"tpb_attention_packed", (PyCFunction)(void (*)(void))attention_packed, METH_FASTCALL, NULL},
    {"tpb_kv_append", (PyCFunction)(void (*)(void))kv_append, METH_FASTCALL, NULL},
    {"tpb_kv_read", (PyCFunction)(void (*)(void))kv_read, METH_FASTCALL, NULL},
    {"tpb_kv_attention", (PyCFunction)(void (*)(void))kv_attention, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL},
};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tpbattncall", NULL, -1, methods, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__tpbattncall(void) { return PyModule_Create(&module); }
