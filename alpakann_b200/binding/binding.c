/*
 * binding.c -- CPython entry points of the decode operators on compressed data.
 *
 * A decode step calls them with a few microseconds of GPU work each, and ctypes
 * spends more than that on describing the tensors. Here a tensor's description
 * is read through DLPack's C exchange interface, which torch offers, into an
 * ann_view. Every function takes the stream handle (None: the current
 * stream of the tensors' device), then tensors (None where optional), then scalars
 * in the order of the C call, and returns its code. Two more codes say that nothing
 * was called and that the caller is to word the error or to change the device:
 * MISMATCH (-1), a dtype or device is not what the call needs, or an argument is no
 * tensor; ELSEWHERE (-3), the tensors' device is not the current one.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/dlpack.h>

#include "ann_b200.h"

enum { MISMATCH = -1, FAILED = -2, ELSEWHERE = -3 };
enum { F32, F64, I8, I32, NTYPES };
static const unsigned char g_code[NTYPES] = {kDLFloat, kDLFloat, kDLInt, kDLInt}, g_bits[NTYPES] = {32, 64, 8, 32};
static PyTypeObject* g_tensor;
static PyObject* g_get_device;
static const DLPackExchangeAPI* g_api;

/* A tensor of type `want` (I32: uint32 too, same bits) on *device (-1: the first
 * tensor decides) as a view. 0, MISMATCH or FAILED with a Python error set. */
static int take(PyObject* t, int want, int* device, ann_view* v) {
    if (g_api == NULL || !PyObject_TypeCheck(t, g_tensor)) return MISMATCH;
    DLTensor d;
    if (g_api->dltensor_from_py_object_no_sync(t, &d) != 0) return FAILED;
    int const code = want == I32 && d.dtype.code == kDLUInt ? kDLInt : d.dtype.code;
    if (code != g_code[want] || d.dtype.bits != g_bits[want] || d.dtype.lanes != 1) return MISMATCH;
    if (d.device.device_type != kDLCUDA || (*device != -1 && d.device.device_id != *device)) return MISMATCH;
    if (d.ndim > ANN_MAX_RANK) return MISMATCH;
    *device = d.device.device_id;
    v->data = (char*)d.data + d.byte_offset;
    v->rank = d.ndim;
    v->reserved = 0;
    for (int i = 0; i < d.ndim; ++i) {
        v->extents[i] = d.shape[i];
        v->pitches[i] = d.strides[i] * (g_bits[want] / 8);
    }
    return 0;
}

/* n tensors of the given types; types[i] with OPT added may be None (p[i] NULL). */
enum { OPT = 16 };
static int take_all(PyObject* stream, PyObject* const* args, int n, const signed char* types, ann_view* v,
                    const ann_view** p, ann_stream* out) {
    int device = -1;
    for (int i = 0; i < n; ++i) {
        p[i] = NULL;
        if ((types[i] & OPT) && args[i] == Py_None) continue;
        int const rc = take(args[i], types[i] & ~OPT, &device, &v[i]);
        if (rc != 0) return rc;
        p[i] = &v[i];
    }
    PyObject* const o = PyObject_CallNoArgs(g_get_device);
    if (o == NULL) return FAILED;
    long const current = PyLong_AsLong(o);
    Py_DECREF(o);
    if (PyErr_Occurred()) return FAILED;
    if (current != device) return ELSEWHERE;
    if (stream != Py_None) {
        *out = PyLong_AsVoidPtr(stream);
        return PyErr_Occurred() ? FAILED : 0;
    }
    return g_api->current_work_stream(kDLCUDA, device, out) != 0 ? FAILED : 0;
}

/* An integer argument; OverflowError outside [low, high]. */
static long long in_range(PyObject* o, long long low, long long high) {
    long long v;
    if (PyLong_Check(o)) {
        v = PyLong_AsLongLong(o);
    } else {
        PyObject* const whole = PyNumber_Long(o);
        if (whole == NULL) return 0;
        v = PyLong_AsLongLong(whole);
        Py_DECREF(whole);
    }
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
    ann_stream stream = NULL;                                                          \
    int rc = take_all(args[0], args + 1, N, types, v, p, &stream);                     \
    if (rc == FAILED) return NULL;                                                     \
    if (rc != 0) return PyLong_FromLong(rc);                                           \
    PyObject* const* const s = args + 1 + N
#define INT(i) ((int32_t)in_range(s[i], INT32_MIN, INT32_MAX))
#define UINT(i) ((uint32_t)in_range(s[i], 0, UINT32_MAX))
#define TRUTH(i) (PyObject_IsTrue(s[i]) != 0)
#define END(call)                                                                      \
    if (PyErr_Occurred()) return NULL;                                                 \
    Py_BEGIN_ALLOW_THREADS;                                                            \
    rc = call;                                                                         \
    Py_END_ALLOW_THREADS;                                                              \
    return PyLong_FromLong(rc)

static PyObject* rotary_f32(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    BEGIN(4, F32, F32 | OPT, I32, F64, F32, F32 | OPT);
    int32_t const pairs = INT(0), layout = INT(1), inverse = TRUTH(3);
    float const magnitude = (float)PyFloat_AsDouble(s[2]);
    END(ann_rotary_f32(stream, p[0], p[1], p[2], p[3], p[4], p[5], pairs, layout, magnitude, inverse));
}
static PyObject* rotary_f64(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    BEGIN(4, F64, F64 | OPT, I32, F64, F64, F64 | OPT);
    int32_t const pairs = INT(0), layout = INT(1), inverse = TRUTH(3);
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
    int32_t const layout = INT(3), causal = TRUTH(4);
    END(ann_attention_decode_q8_f32(stream, p[0], p[1], p[2], p[3], p[4], p[5], p[6], scale, group, block, layout,
                                    causal));
}
static PyObject* linear_q4(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    BEGIN(2, F32, I32, F32, F32 | OPT, F32 | OPT, F32);
    uint32_t const group = UINT(0);
    int32_t const act = INT(1);
    END(ann_linear_q4_f32(stream, p[0], p[1], p[2], p[3], p[4], p[5], group, act));
}

/* setup(torch.Tensor, torch's function that returns the current device), once. */
static PyObject* setup(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
    (void)self;
    if (nargs != 2 || !PyType_Check(args[0])) {
        PyErr_SetString(PyExc_TypeError, "setup(Tensor, current_device)");
        return NULL;
    }
    PyObject* const capsule = PyObject_GetAttrString(args[0], "__dlpack_c_exchange_api__");
    if (capsule == NULL) return NULL;
    const DLPackExchangeAPI* const api = PyCapsule_GetPointer(capsule, "dlpack_exchange_api");
    Py_DECREF(capsule);
    if (api == NULL) return NULL;
    if (api->header.version.major != DLPACK_MAJOR_VERSION || api->dltensor_from_py_object_no_sync == NULL) {
        PyErr_SetString(PyExc_ImportError, "this torch has no DLPack exchange interface of the built version");
        return NULL;
    }
    Py_INCREF(args[0]);
    Py_XSETREF(g_tensor, (PyTypeObject*)args[0]);
    Py_INCREF(args[1]);
    Py_XSETREF(g_get_device, args[1]);
    g_api = api;
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {METHOD(rotary_f32),        METHOD(rotary_f64),          METHOD(kv_cache_append_q8),
                                METHOD(kv_cache_read_q8),  METHOD(attention_decode_q8), METHOD(linear_q4),
                                {"setup", (PyCFunction)(void (*)(void))setup, METH_FASTCALL, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ann_binding", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__ann_binding(void) { return PyModule_Create(&module); }
