/*
 * binding.c -- CPython entry points of the decode operators on compressed data.
 *
 * A decode step calls them with a few microseconds of GPU work each, and ctypes
 * spends more than that on describing the tensors. Here a tensor's description
 * (dtype, device, pointer, extents, strides) is read straight into an ann_view,
 * about 0.3 us each. Every function takes the stream handle, then tensors (None
 * where optional), then scalars in the order of the C call, and returns its code;
 * MISMATCH (-1) says that a dtype or device is not what the call needs, or that
 * an argument is no tensor: nothing was called, and the caller words the error.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "ann_b200.h"

enum { MISMATCH = -1 };
enum { F32, F64, I8, I32, U32, NTYPES };
static PyObject* g_types[NTYPES];
static const Py_ssize_t g_size[NTYPES] = {4, 8, 1, 4, 4};
static PyObject *s_dtype, *s_get_device, *s_data_ptr, *s_shape, *s_stride;

/* A tensor of type `want` (I32: uint32 too, same bits) on *device (-2: the first
 * tensor decides; the CPU's -1 never fits) as a view. 0, MISMATCH or -2 with a
 * Python error set. */
static int take(PyObject* t, int want, long* device, ann_view* v) {
    PyObject* o = PyObject_GetAttr(t, s_dtype);
    if (o == NULL) goto no_tensor;
    int const same = o == g_types[want] || (want == I32 && o == g_types[U32]);
    Py_DECREF(o);
    if (!same) return MISMATCH;
    if ((o = PyObject_CallMethodNoArgs(t, s_get_device)) == NULL) goto no_tensor;
    long const dev = PyLong_AsLong(o);
    Py_DECREF(o);
    if (dev < 0 || (*device != -2 && dev != *device)) return MISMATCH;
    *device = dev;
    if ((o = PyObject_CallMethodNoArgs(t, s_data_ptr)) == NULL) return -2;
    v->data = PyLong_AsVoidPtr(o);
    Py_DECREF(o);
    PyObject* const shape = PyObject_GetAttr(t, s_shape);
    if (shape == NULL) return -2;
    PyObject* const stride = PyObject_CallMethodNoArgs(t, s_stride);
    if (stride == NULL) {
        Py_DECREF(shape);
        return -2;
    }
    int rc = MISMATCH;
    if (PyTuple_Check(shape) && PyTuple_Check(stride) && PyTuple_GET_SIZE(shape) == PyTuple_GET_SIZE(stride) &&
        PyTuple_GET_SIZE(shape) <= ANN_MAX_RANK) {
        v->rank = (int32_t)PyTuple_GET_SIZE(shape);
        v->reserved = 0;
        for (int i = 0; i < v->rank; ++i) {
            v->extents[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
            v->pitches[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, i)) * g_size[want];
        }
        rc = 0;
    }
    Py_DECREF(shape);
    Py_DECREF(stride);
    return PyErr_Occurred() ? -2 : rc;
no_tensor:
    PyErr_Clear();
    return MISMATCH;
}

/* n tensors of the given types; types[i] with OPT added may be None (p[i] NULL). */
enum { OPT = 16 };
static int take_all(PyObject* const* args, int n, const signed char* types, ann_view* v, const ann_view** p) {
    long device = -2;
    for (int i = 0; i < n; ++i) {
        p[i] = NULL;
        if ((types[i] & OPT) && args[i] == Py_None) continue;
        int const rc = take(args[i], types[i] & ~OPT, &device, &v[i]);
        if (rc != 0) return rc;
        p[i] = &v[i];
    }
    return 0;
}

/* An integer argument; OverflowError outside [low, high]. */
static long long in_range(PyObject* o, long long low, long long high) {
    long long const v = PyLong_AsLongLong(o);
    if (!PyErr_Occurred() && (v < low || v > high)) PyErr_SetString(PyExc_OverflowError, "integer argument out of range");
    return v;
}

#define BEGIN(count, ...)                                                              \
    static const signed char types[] = {__VA_ARGS__};                                  \
    enum { N = sizeof types };                                                         \
    ann_view v[N];                                                                     \
    const ann_view* p[N];                                                              \
    (void)self;                                                                        \
    if (nargs != 1 + N + (count)) {                                                    \
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");                 \
        return NULL;                                                                   \
    }                                                                                  \
    ann_stream const stream = PyLong_AsVoidPtr(args[0]);                               \
    if (PyErr_Occurred()) return NULL;                                                 \
    int rc = take_all(args + 1, N, types, v, p);                                       \
    if (rc == -2) return NULL;                                                         \
    if (rc == MISMATCH) return PyLong_FromLong(MISMATCH);                              \
    PyObject* const* const s = args + 1 + N
#define INT(i) ((int32_t)in_range(s[i], INT32_MIN, INT32_MAX))
#define UINT(i) ((uint32_t)in_range(s[i], 0, UINT32_MAX))
#define END(call)                                                                      \
    if (PyErr_Occurred()) return NULL;                                                 \
    Py_BEGIN_ALLOW_THREADS;                                                            \
    rc = call;                                                                         \
    Py_END_ALLOW_THREADS;                                                              \
    return PyLong_FromLong(rc)

static PyObject* rotary_f32(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    BEGIN(4, F32, F32 | OPT, I32, F64, F32, F32 | OPT);
    int32_t const pairs = INT(0), layout = INT(1), inverse = INT(3);
    float const magnitude = (float)PyFloat_AsDouble(s[2]);
    END(ann_rotary_f32(stream, p[0], p[1], p[2], p[3], p[4], p[5], pairs, layout, magnitude, inverse));
}
static PyObject* rotary_f64(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    BEGIN(4, F64, F64 | OPT, I32, F64, F64, F64 | OPT);
    int32_t const pairs = INT(0), layout = INT(1), inverse = INT(3);
    double const magnitude = PyFloat_AsDouble(s[2]);
    END(ann_rotary_f64(stream, p[0], p[1], p[2], p[3], p[4], p[5], pairs, layout, magnitude, inverse));
}
static PyObject* kv_cache_append_q8(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    BEGIN(2, F32, F32, I8, I8, F32, F32, I32, I32 | OPT);
    uint32_t const block = UINT(0);
    int32_t const layout = INT(1);
    END(ann_kv_cache_append_q8_f32(stream, p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], block, layout));
}
static PyObject* kv_cache_read_q8(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    BEGIN(2, I8, I8, F32, F32, F32, F32, I32 | OPT);
    uint32_t const block = UINT(0);
    int32_t const layout = INT(1);
    END(ann_kv_cache_read_q8_f32(stream, p[0], p[1], p[2], p[3], p[4], p[5], p[6], block, layout));
}
static PyObject* attention_decode_q8(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    BEGIN(5, F32, I8, I8, F32, F32, I32 | OPT, F32);
    float const scale = (float)PyFloat_AsDouble(s[0]);
    uint32_t const group = UINT(1), block = UINT(2);
    int32_t const layout = INT(3), causal = INT(4);
    END(ann_attention_decode_q8_f32(stream, p[0], p[1], p[2], p[3], p[4], p[5], p[6], scale, group, block, layout,
                                    causal));
}
static PyObject* linear_q4(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    BEGIN(2, F32, I32, F32, F32 | OPT, F32 | OPT, F32);
    uint32_t const group = UINT(0);
    int32_t const act = INT(1);
    END(ann_linear_q4_f32(stream, p[0], p[1], p[2], p[3], p[4], p[5], group, act));
}

/* types(float32, float64, int8, int32, uint32): torch's dtype objects, once. */
static PyObject* types_(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    (void)self;
    if (nargs != NTYPES) {
        PyErr_SetString(PyExc_TypeError, "types(float32, float64, int8, int32, uint32)");
        return NULL;
    }
    for (int i = 0; i < NTYPES; ++i) {
        Py_INCREF(args[i]);
        Py_XSETREF(g_types[i], args[i]);
    }
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {METHOD(rotary_f32),        METHOD(rotary_f64),          METHOD(kv_cache_append_q8),
                                METHOD(kv_cache_read_q8),  METHOD(attention_decode_q8), METHOD(linear_q4),
                                {"types", (PyCFunction)(void (*)(void))types_, METH_FASTCALL, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ann_binding", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__ann_binding(void) {
    if ((s_dtype = PyUnicode_InternFromString("dtype")) == NULL ||
        (s_get_device = PyUnicode_InternFromString("get_device")) == NULL ||
        (s_data_ptr = PyUnicode_InternFromString("data_ptr")) == NULL ||
        (s_shape = PyUnicode_InternFromString("shape")) == NULL ||
        (s_stride = PyUnicode_InternFromString("stride")) == NULL)
        return NULL;
    return PyModule_Create(&module);
}
