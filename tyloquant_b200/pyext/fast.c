/* Direct calls of the library's hot entry points from Python.
 *
 * A product of one row takes the GPU about 4 us; converting its six arguments through ctypes alone takes more than one.
 * These functions take plain integers (addresses, sizes, enum values) in METH_FASTCALL form and return the status.  The
 * entry points' addresses come from the ctypes binding (bind), so nothing is linked here. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

typedef int (*mul_mat_fn)(const void*, const void*, int, void*, int, void*);
typedef int (*topk_fn)(const void*, int, int, int, int, const void*, int, float, float, void*, void*, void*);
typedef int (*ffn_fn)(const void*, const void*, const void*, const void*, const void*, int, int, void*, int, void*);

typedef int (*extend_fn)(const void*, const void*, void*, void*);
typedef int (*fork_fn)(const void*, const void*, void*, void*, uint64_t, void*);
typedef int (*masks_fn)(const void*, int, int, void*, void*, void*);
typedef int (*write_fn)(const void*, int, const void*, int, int, const void*, const void*, void*, void*);
typedef int (*attend_fn)(const void*, int, const void*, int, int, const void*, float, void*, void*, uint64_t, void*);
typedef int (*accept_fn)(const void*, const void*, const void*, const void*, int, void*, void*, void*, void*, void*);
typedef int (*beam_fn)(const void*, int, int, int, const void*, const void*, int, int, void*, void*, void*, void*, uint64_t, void*);

static mul_mat_fn p_mul_mat;
static topk_fn p_topk;
static ffn_fn p_ffn;
static extend_fn p_extend;
static fork_fn p_fork;
static masks_fn p_masks;
static write_fn p_write;
static attend_fn p_attend;
static accept_fn p_accept;
static beam_fn p_beam;

static void* address(PyObject* o) { return o == Py_None ? NULL : (void*)(uintptr_t)PyLong_AsUnsignedLongLong(o); }
static int number(PyObject* o) {
    const long v = PyLong_AsLong(o);
    if (v != (int)v) PyErr_SetString(PyExc_OverflowError, "argument does not fit a C int");
    return (int)v;
}
static int arity(Py_ssize_t got, Py_ssize_t want) {
    if (got == want) return 1;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    return 0;
}

static PyObject* bind(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 10)) return NULL;
    p_mul_mat = (mul_mat_fn)address(a[0]);
    p_topk = (topk_fn)address(a[1]);
    p_ffn = (ffn_fn)address(a[2]);
    p_extend = (extend_fn)address(a[3]);
    p_fork = (fork_fn)address(a[4]);
    p_masks = (masks_fn)address(a[5]);
    p_write = (write_fn)address(a[6]);
    p_attend = (attend_fn)address(a[7]);
    p_accept = (accept_fn)address(a[8]);
    p_beam = (beam_fn)address(a[9]);
    if (PyErr_Occurred()) return NULL;
    Py_RETURN_NONE;
}
/* weight, x, m, y, y_dtype, stream */
static PyObject* mul_mat(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 6)) return NULL;
    const void *w = address(a[0]), *x = address(a[1]);
    const int m = number(a[2]);
    void* y = address(a[3]);
    const int dt = number(a[4]);
    void* s = address(a[5]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_mul_mat(w, x, m, y, dt, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* logits, tokens, experts, k, mode, bias, normalize, norm_floor, scale, ids, weights, stream */
static PyObject* moe_topk(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 12)) return NULL;
    const void* z = address(a[0]);
    const int t = number(a[1]), e = number(a[2]), k = number(a[3]), mode = number(a[4]);
    const void* bias = address(a[5]);
    const int norm = number(a[6]);
    const float norm_floor = (float)PyFloat_AsDouble(a[7]), scale = (float)PyFloat_AsDouble(a[8]);
    void *ids = address(a[9]), *w = address(a[10]), *s = address(a[11]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_topk(z, t, e, k, mode, bias, norm, norm_floor, scale, ids, w, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* gate_up, down, x, ids, weights, tokens, routes, y, y_dtype, stream */
static PyObject* moe_ffn(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 10)) return NULL;
    const void *g = address(a[0]), *d = address(a[1]), *x = address(a[2]), *ids = address(a[3]), *w = address(a[4]);
    const int t = number(a[5]), r = number(a[6]);
    void* y = address(a[7]);
    const int dt = number(a[8]);
    void* s = address(a[9]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_ffn(g, d, x, ids, w, t, r, y, dt, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

/* cache, tokens, status, stream */
static PyObject* cache_extend(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 4)) return NULL;
    void* c = address(a[0]);
    void* t = address(a[1]);
    void* st = address(a[2]);
    void* s = address(a[3]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_extend(c, t, st, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* cache, parents, status, work, work_bytes, stream */
static PyObject* cache_fork(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 6)) return NULL;
    void* c = address(a[0]);
    void* pa = address(a[1]);
    void* st = address(a[2]);
    void* w = address(a[3]);
    const uint64_t wb = PyLong_AsUnsignedLongLong(a[4]);
    void* s = address(a[5]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_fork(c, pa, st, w, wb, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* parents, rows, nodes, masks, depths, stream */
static PyObject* tree_masks(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 6)) return NULL;
    void* pa = address(a[0]);
    const int r = number(a[1]);
    const int nodes = number(a[2]);
    void* m = address(a[3]);
    void* d = address(a[4]);
    void* s = address(a[5]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_masks(pa, r, nodes, m, d, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* cache, layer, qkv, q_heads, nodes, depths, freqs, q_out, stream */
static PyObject* cache_write(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 9)) return NULL;
    void* c = address(a[0]);
    const int l = number(a[1]);
    void* x = address(a[2]);
    const int hq = number(a[3]);
    const int nodes = number(a[4]);
    void* d = address(a[5]);
    void* f = address(a[6]);
    void* q = address(a[7]);
    void* s = address(a[8]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_write(c, l, x, hq, nodes, d, f, q, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* cache, layer, q, q_heads, nodes, masks, scale, out, work, work_bytes, stream */
static PyObject* tree_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 11)) return NULL;
    void* c = address(a[0]);
    const int l = number(a[1]);
    void* q = address(a[2]);
    const int hq = number(a[3]);
    const int nodes = number(a[4]);
    void* m = address(a[5]);
    const float scale = (float)PyFloat_AsDouble(a[6]);
    void* o = address(a[7]);
    void* w = address(a[8]);
    const uint64_t wb = PyLong_AsUnsignedLongLong(a[9]);
    void* s = address(a[10]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_attend(c, l, q, hq, nodes, m, scale, o, w, wb, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* cache, ids, parents, targets, nodes, count, token, path, lens_out, stream */
static PyObject* tree_accept(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 10)) return NULL;
    void* c = address(a[0]);
    void* ids = address(a[1]);
    void* pa = address(a[2]);
    void* t = address(a[3]);
    const int nodes = number(a[4]);
    void* cnt = address(a[5]);
    void* tok = address(a[6]);
    void* path = address(a[7]);
    void* lens = address(a[8]);
    void* s = address(a[9]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_accept(c, ids, pa, t, nodes, cnt, tok, path, lens, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}
/* logits, groups, beams, vocab, scores, done, eos, k, out_scores, out_rows, out_tokens, work, work_bytes, stream */
static PyObject* beam_select(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    (void)self;
    if (!arity(n, 14)) return NULL;
    void* z = address(a[0]);
    const int g = number(a[1]);
    const int w = number(a[2]);
    const int v = number(a[3]);
    void* sc = address(a[4]);
    void* d = address(a[5]);
    const int eos = number(a[6]);
    const int k = number(a[7]);
    void* os = address(a[8]);
    void* orow = address(a[9]);
    void* ot = address(a[10]);
    void* wk = address(a[11]);
    const uint64_t wb = PyLong_AsUnsignedLongLong(a[12]);
    void* s = address(a[13]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = p_beam(z, g, w, v, sc, d, eos, k, os, orow, ot, wk, wb, s);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

static PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, "addresses of the entry points below, in their order"},
                                {"mul_mat", (PyCFunction)(void (*)(void))mul_mat, METH_FASTCALL, "mfqb_mul_mat"},
                                {"moe_topk", (PyCFunction)(void (*)(void))moe_topk, METH_FASTCALL, "mfqb_moe_topk"},
                                {"moe_ffn", (PyCFunction)(void (*)(void))moe_ffn, METH_FASTCALL, "mfqb_moe_ffn"},
                                {"cache_extend", (PyCFunction)(void (*)(void))cache_extend, METH_FASTCALL, "mfqb_cache_extend"},
                                {"cache_fork", (PyCFunction)(void (*)(void))cache_fork, METH_FASTCALL, "mfqb_cache_fork"},
                                {"tree_masks", (PyCFunction)(void (*)(void))tree_masks, METH_FASTCALL, "mfqb_tree_masks"},
                                {"cache_write", (PyCFunction)(void (*)(void))cache_write, METH_FASTCALL, "mfqb_cache_write"},
                                {"tree_attention", (PyCFunction)(void (*)(void))tree_attention, METH_FASTCALL, "mfqb_tree_attention"},
                                {"tree_accept", (PyCFunction)(void (*)(void))tree_accept, METH_FASTCALL, "mfqb_tree_accept"},
                                {"beam_select", (PyCFunction)(void (*)(void))beam_select, METH_FASTCALL, "mfqb_beam_select"},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", "Direct calls of the library's hot entry points.", -1, methods, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__fast(void) { return PyModule_Create(&module); }
