/* The operator calls as CPython functions.  lutamm_amm() on tensors of a few hundred rows takes the GPU less than the
 * host: through ctypes the binding alone (argument conversion, four attribute look-ups and two method calls in Python)
 * cost 3 us of a 10 us call.  Same arguments and checks as LutAmmContext.amm_host; anything but tensors - numpy
 * arrays, raw addresses - answers NotImplemented and takes the ctypes way. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "../../../include/lutamm.h"

typedef int (*amm_fn)(void*, int, const float*, float*, uint32_t, uint32_t);

static PyObject *s_is_contiguous, *s_data_ptr, *s_shape;

/* Address of a contiguous tensor; 1 on success, 0 if it is no tensor, -1 with an exception set. */
static int address_of(PyObject* t, void** out) {
    PyObject* ok = PyObject_CallMethodNoArgs(t, s_is_contiguous);
    if (!ok) {
        if (!PyErr_ExceptionMatches(PyExc_AttributeError)) return -1;
        PyErr_Clear();
        return 0;
    }
    const int contiguous = PyObject_IsTrue(ok);
    Py_DECREF(ok);
    if (contiguous < 0) return -1;
    if (!contiguous) {
        PyErr_SetString(PyExc_AssertionError, "tensors handed to the C ABI must be contiguous");
        return -1;
    }
    PyObject* a = PyObject_CallMethodNoArgs(t, s_data_ptr);
    if (!a) return -1;
    *out = PyLong_AsVoidPtr(a);
    Py_DECREF(a);
    return PyErr_Occurred() ? -1 : 1;
}

/* amm(function address, context address, layer id, input, output, tokens or None, flags) -> return code */
static PyObject* amm(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    (void)self;
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "amm takes 7 arguments");
        return NULL;
    }
    const amm_fn fn = (amm_fn)PyLong_AsVoidPtr(args[0]);
    void* ctx = PyLong_AsVoidPtr(args[1]);
    const long layer = PyLong_AsLong(args[2]);
    void *in = NULL, *out = NULL;
    if (PyErr_Occurred()) return NULL;
    int r = address_of(args[3], &in);
    if (r > 0) r = address_of(args[4], &out);
    if (r < 0) return NULL;
    if (r == 0) Py_RETURN_NOTIMPLEMENTED;
    PyObject* rows = NULL;
    if (args[5] == Py_None) {
        PyObject* shape = PyObject_GetAttr(args[3], s_shape);
        if (!shape) return NULL;
        rows = PySequence_GetItem(shape, 0);
        Py_DECREF(shape);
        if (!rows) return NULL;
    }
    PyObject* count = PyNumber_Long(rows ? rows : args[5]);   /* int() of it, as in amm_host */
    Py_XDECREF(rows);
    if (!count) return NULL;
    const unsigned long tokens = PyLong_AsUnsignedLongMask(count);
    Py_DECREF(count);
    const unsigned long flags = PyLong_AsUnsignedLongMask(args[6]);
    if (PyErr_Occurred()) return NULL;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(ctx, (int)layer, (const float*)in, (float*)out, (uint32_t)tokens, (uint32_t)flags);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

/* The dense operators: each fills its parameter block from tensors as the binding's Python does.  Whatever is not as it should be - another type, shape,
 * layout or object - answers NotImplemented and takes the Python way, which says what is wrong. */
static PyObject *s_dtype, *s_stride, *t_f32, *t_f16, *t_bf16, *t_i32;

typedef struct {
    void* data;
    PyObject* dtype;   /* borrowed: the types live as long as torch */
    int nd;
    int64_t shape[4], stride[4];
} tensor;

static int load_types(void) {
    if (t_i32) return 1;
    PyObject* torch = PyImport_ImportModule("torch");
    if (!torch) return 0;
    t_f32 = PyObject_GetAttrString(torch, "float32");
    t_f16 = PyObject_GetAttrString(torch, "float16");
    t_bf16 = PyObject_GetAttrString(torch, "bfloat16");
    t_i32 = PyObject_GetAttrString(torch, "int32");
    Py_DECREF(torch);
    return t_f32 && t_f16 && t_bf16 && t_i32;
}

static int numbers(PyObject* seq, int64_t* out, int most) {   /* how many; -1 if it is none */
    if (!seq) return -1;
    int n = -1;
    if (PyTuple_Check(seq) && PyTuple_GET_SIZE(seq) <= most) {
        n = (int)PyTuple_GET_SIZE(seq);
        for (int i = 0; i < n; ++i) out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(seq, i));
        if (PyErr_Occurred()) n = -1;
    }
    Py_DECREF(seq);
    return n;
}

static int read_tensor(PyObject* t, tensor* out) {   /* 1: read; an absent one (None) has null data */
    memset(out, 0, sizeof *out);
    if (t == Py_None) return 1;
    out->nd = numbers(PyObject_GetAttr(t, s_shape), out->shape, 4);
    if (out->nd < 1 || numbers(PyObject_CallMethodNoArgs(t, s_stride), out->stride, 4) != out->nd) return 0;
    out->dtype = PyObject_GetAttr(t, s_dtype);
    if (!out->dtype) return 0;
    Py_DECREF(out->dtype);
    PyObject* a = PyObject_CallMethodNoArgs(t, s_data_ptr);
    if (!a) return 0;
    out->data = PyLong_AsVoidPtr(a);
    Py_DECREF(a);
    return !PyErr_Occurred() && out->data;   /* (one without elements has no address: the Python way) */
}
static int dtype_code(const tensor* t) { return t->dtype == t_f32 ? LUTAMM_F32 : t->dtype == t_f16 ? LUTAMM_F16 : t->dtype == t_bf16 ? LUTAMM_BF16 : -1; }
static int is(const tensor* t, PyObject* dtype, int nd, int64_t a, int64_t b, int64_t c, int64_t d) {   /* absent, or of this type and shape, its last axis contiguous */
    if (!t->data) return 1;
    const int64_t want[4] = {a, b, c, d};
    if (t->dtype != dtype || t->nd != nd || (t->stride[nd - 1] != 1 && t->shape[nd - 1] > 1)) return 0;
    for (int i = 0; i < nd; ++i)
        if (t->shape[i] != want[i]) return 0;
    return 1;
}
static int packed(const tensor* t) { return !t->data || t->nd < 2 || t->shape[0] <= 1 || t->stride[0] == t->shape[1]; }
static int small(int64_t v) { return v >= 0 && v <= INT32_MAX; }

static PyObject* done(int rc) { return PyLong_FromLong(rc); }
static PyObject* not_here(void) {
    PyErr_Clear();
    Py_RETURN_NOTIMPLEMENTED;
}

/* layer_norm(function, context, x, weight, bias, out, eps, residual, stats, flags) */
static PyObject* layer_norm(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    (void)self;
    if (n != 10 || !load_types()) return not_here();
    int (*fn)(void*, const lutamm_norm_params*, uint32_t) = (int (*)(void*, const lutamm_norm_params*, uint32_t))PyLong_AsVoidPtr(args[0]);
    void* ctx = PyLong_AsVoidPtr(args[1]);
    tensor x, w, b, out, r, st;
    if (!read_tensor(args[2], &x) || !read_tensor(args[3], &w) || !read_tensor(args[4], &b) || !read_tensor(args[5], &out) || !read_tensor(args[7], &r) ||
        !read_tensor(args[8], &st) || !x.data || !out.data || x.nd != 2 || dtype_code(&x) < 0)
        return not_here();
    const int64_t rows = x.shape[0], width = x.shape[1];
    if (!small(rows) || !small(width) || !is(&x, x.dtype, 2, rows, width, 0, 0) || !is(&out, x.dtype, 2, rows, width, 0, 0) || !is(&r, x.dtype, 2, rows, width, 0, 0) ||
        !is(&w, t_f32, 1, width, 0, 0, 0) || !is(&b, t_f32, 1, width, 0, 0, 0) || !is(&st, t_f32, 2, rows, 2, 0, 0) || !packed(&st))
        return not_here();
    lutamm_norm_params p = {(uint32_t)dtype_code(&x), (uint32_t)rows, (uint32_t)width, (float)PyFloat_AsDouble(args[6]), x.data, x.stride[0], r.data, r.stride[0],
                            out.data, out.stride[0], w.data, b.data, st.data};
    const unsigned long flags = PyLong_AsUnsignedLongMask(args[9]);
    if (PyErr_Occurred()) return not_here();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(ctx, &p, (uint32_t)flags);
    Py_END_ALLOW_THREADS
    return done(rc);
}

/* layer_norm_backward(function, context, dout, x, weight, stats, dx, dweight, dbias, flags), without a workspace */
static PyObject* layer_norm_backward(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    (void)self;
    if (n != 10 || !load_types()) return not_here();
    int (*fn)(void*, const lutamm_norm_grad_params*, uint32_t) = (int (*)(void*, const lutamm_norm_grad_params*, uint32_t))PyLong_AsVoidPtr(args[0]);
    void* ctx = PyLong_AsVoidPtr(args[1]);
    tensor dy, x, w, st, dx, dw, db;
    if (!read_tensor(args[2], &dy) || !read_tensor(args[3], &x) || !read_tensor(args[4], &w) || !read_tensor(args[5], &st) || !read_tensor(args[6], &dx) ||
        !read_tensor(args[7], &dw) || !read_tensor(args[8], &db) || !x.data || !dy.data || !st.data || x.nd != 2 || dtype_code(&x) < 0)
        return not_here();
    const int64_t rows = x.shape[0], width = x.shape[1];
    if (!small(rows) || !small(width) || !is(&x, x.dtype, 2, rows, width, 0, 0) || !is(&dy, x.dtype, 2, rows, width, 0, 0) || !is(&dx, x.dtype, 2, rows, width, 0, 0) ||
        !is(&w, t_f32, 1, width, 0, 0, 0) || !is(&dw, t_f32, 1, width, 0, 0, 0) || !is(&db, t_f32, 1, width, 0, 0, 0) || !is(&st, t_f32, 2, rows, 2, 0, 0) || !packed(&st))
        return not_here();
    lutamm_norm_grad_params p = {(uint32_t)dtype_code(&x), (uint32_t)rows, (uint32_t)width, dy.data, dy.stride[0], x.data, x.stride[0], dx.data, dx.stride[0],
                                 w.data, st.data, dw.data, db.data, NULL};
    const unsigned long flags = PyLong_AsUnsignedLongMask(args[9]);
    if (PyErr_Occurred()) return not_here();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(ctx, &p, (uint32_t)flags);
    Py_END_ALLOW_THREADS
    return done(rc);
}

static lutamm_heads heads_of(const tensor* t) {   /* three axes are one sequence */
    lutamm_heads h = {t->data, t->nd == 4 ? t->stride[0] : 0, t->stride[t->nd - 3], t->stride[t->nd - 2]};
    return h;
}

/* rotary(function, context, x, positions, inv_freq, sections, out, interleaved, inverse, flags) */
static PyObject* rotary(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    (void)self;
    if (n != 10 || !load_types()) return not_here();
    int (*fn)(void*, const lutamm_rotary_params*, uint32_t) = (int (*)(void*, const lutamm_rotary_params*, uint32_t))PyLong_AsVoidPtr(args[0]);
    void* ctx = PyLong_AsVoidPtr(args[1]);
    tensor x, pos, freq, out;
    if (!read_tensor(args[2], &x) || !read_tensor(args[3], &pos) || !read_tensor(args[4], &freq) || !read_tensor(args[6], &out) || !x.data || !pos.data || !freq.data ||
        !out.data || x.nd < 3 || x.nd != out.nd || dtype_code(&x) < 0 || (!PyList_Check(args[5]) && !PyTuple_Check(args[5])))
        return not_here();
    const int64_t batch = x.nd == 4 ? x.shape[0] : 1, tokens = x.shape[x.nd - 3], heads = x.shape[x.nd - 2], dim = x.shape[x.nd - 1];
    const Py_ssize_t axes = PySequence_Fast_GET_SIZE(args[5]);
    if (axes < 1 || axes > LUTAMM_MAX_AXES || !small(batch) || !small(tokens) || !small(heads) || !small(dim) || !is(&x, x.dtype, x.nd, x.shape[0], x.shape[1], x.shape[2], x.shape[3]) ||
        !is(&out, x.dtype, x.nd, x.shape[0], x.shape[1], x.shape[2], x.shape[3]))
        return not_here();
    if (!(pos.nd == 2 ? is(&pos, t_i32, 2, tokens, axes, 0, 0) : is(&pos, t_i32, 3, batch, tokens, axes, 0))) return not_here();
    lutamm_rotary_params p;
    memset(&p, 0, sizeof p);
    int64_t pairs = 0;
    for (Py_ssize_t i = 0; i < axes; ++i) {
        const long long v = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(args[5], i));
        if (PyErr_Occurred() || !small(v)) return not_here();
        p.sections[i] = (uint32_t)v;
        pairs += v;
    }
    if (!is(&freq, t_f32, 1, pairs, 0, 0, 0)) return not_here();
    p.dtype = (uint32_t)dtype_code(&x);
    p.batch = (uint32_t)batch; p.tokens = (uint32_t)tokens; p.heads = (uint32_t)heads; p.head_dim = (uint32_t)dim; p.axes = (uint32_t)axes;
    const int interleaved = PyObject_IsTrue(args[7]), inverse = PyObject_IsTrue(args[8]);
    p.interleaved = interleaved > 0;
    p.inverse = inverse > 0;
    p.x = heads_of(&x);
    p.out = heads_of(&out);
    p.positions = pos.data;
    p.position_batch_stride = pos.nd == 3 ? pos.stride[0] : 0;
    p.position_token_stride = pos.stride[pos.nd - 2];
    p.inv_freq = freq.data;
    const unsigned long flags = PyLong_AsUnsignedLongMask(args[9]);
    if (PyErr_Occurred() || interleaved < 0 || inverse < 0) return not_here();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(ctx, &p, (uint32_t)flags);
    Py_END_ALLOW_THREADS
    return done(rc);
}

/* attention(function, context, q, k, v, out, scale, window, sinks, lengths, first, flags) */
static PyObject* attention(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    (void)self;
    if (n != 12 || !load_types()) return not_here();
    int (*fn)(void*, const lutamm_attention_params*, uint32_t) = (int (*)(void*, const lutamm_attention_params*, uint32_t))PyLong_AsVoidPtr(args[0]);
    void* ctx = PyLong_AsVoidPtr(args[1]);
    tensor q, k, v, out, len, first;
    if (!read_tensor(args[2], &q) || !read_tensor(args[3], &k) || !read_tensor(args[4], &v) || !read_tensor(args[5], &out) || !read_tensor(args[9], &len) ||
        !read_tensor(args[10], &first) || !q.data || !k.data || !v.data || !out.data || q.nd != 4 || k.nd != 4 || dtype_code(&q) < 0 || !PyTuple_Check(args[7]) ||
        PyTuple_GET_SIZE(args[7]) != 2)
        return not_here();
    const int64_t B = q.shape[0], Q = q.shape[1], H = q.shape[2], D = q.shape[3], K = k.shape[1], G = k.shape[2];
    if (!small(B) || !small(Q) || !small(H) || !small(D) || !small(K) || !small(G) || !is(&q, q.dtype, 4, B, Q, H, D) || !is(&out, q.dtype, 4, B, Q, H, D) ||
        !is(&k, q.dtype, 4, B, K, G, D) || !is(&v, q.dtype, 4, B, K, G, D) || !is(&len, t_i32, 1, B, 0, 0, 0) || !is(&first, t_i32, 1, B, 0, 0, 0))
        return not_here();
    const long long left = PyLong_AsLongLong(PyTuple_GET_ITEM(args[7], 0)), right = PyLong_AsLongLong(PyTuple_GET_ITEM(args[7], 1)), sinks = PyLong_AsLongLong(args[8]);
    const double scale = args[6] == Py_None ? 0.0 : PyFloat_AsDouble(args[6]);
    const unsigned long flags = PyLong_AsUnsignedLongMask(args[11]);
    if (PyErr_Occurred() || left > INT32_MAX || left < INT32_MIN || right > INT32_MAX || right < INT32_MIN || !small(sinks)) return not_here();
    lutamm_attention_params p = {(uint32_t)dtype_code(&q), (uint32_t)B, (uint32_t)Q, (uint32_t)K, (uint32_t)H, (uint32_t)G, (uint32_t)D, (uint32_t)sinks, (int32_t)left,
                                 (int32_t)right, (float)(args[6] == Py_None ? 1.0 / sqrt((double)D) : scale), heads_of(&q), heads_of(&k), heads_of(&v), heads_of(&out), len.data, first.data};
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fn(ctx, &p, (uint32_t)flags);
    Py_END_ALLOW_THREADS
    return done(rc);
}

#define ENTRY(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, "lutamm_" #name " on tensors"}
static PyMethodDef methods[] = {ENTRY(layer_norm), ENTRY(layer_norm_backward), ENTRY(rotary), ENTRY(attention), {"amm", (PyCFunction)(void (*)(void))amm, METH_FASTCALL, "lutamm_amm on two tensors"}, {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fastcall(void) {
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_shape = PyUnicode_InternFromString("shape");
    s_dtype = PyUnicode_InternFromString("dtype");
    s_stride = PyUnicode_InternFromString("stride");
    return PyModule_Create(&module);
}
