// CPython binding of the two Q4_0 linear-layer entries and of the MXFP4 and sorted-row entries
// for device tensors.
//
// A decode step's kernel takes 3 to 6 us, less than Python needs to pass four tensors
// through ctypes (7.1 us a call at K=4096, N=4096, whose kernel takes 3.5 us).  Here the
// tensors' attributes are read and the C entry is called in one native function.  No torch
// header is needed: is_cuda, is_contiguous() and data_ptr() are looked up on the object, the
// current stream comes from the callable that the Python side hands over once.
//
// linear(split, current_stream, x, w, y, in_features, out_features, num_tokens, ws, stream)
//   -> status code of linear_q4_0_forward_device / linear_q4_0s_forward_device, or None if a
//      size or an address is no int (the caller then leaves the conversion to ctypes)
// entry(which, stream_of_device, current_device, stream, arguments...) -> status code of the
//      which-th entry of kEntries, its arguments in the C order without the stream.  Tensors must be
//      contiguous and on the current device; an address (int) is taken as it is.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <string.h>

#include "jjjetson_ops_amd.h"

namespace {

PyObject *s_is_cuda, *s_is_contiguous, *s_data_ptr, *s_cuda_stream, *s_get_device;

// An address as an int; -1 where it is none (no exception set).
int address(PyObject *r, void **out) {
    *out = PyLong_AsVoidPtr(r);
    if (*out != nullptr || !PyErr_Occurred()) return 1;
    PyErr_Clear();
    return -1;
}

// A C int as ctypes converts one (an int or an object with __index__, truncated); -1 for
// anything else: ctypes also takes its own c_int and _as_parameter_, and names the argument
// that it refuses.
int c_int(PyObject *o, int *out) {
    const unsigned long v = PyLong_AsUnsignedLongMask(o);
    *out = (int)v;
    if (v != (unsigned long)-1 || !PyErr_Occurred()) return 1;
    PyErr_Clear();
    return -1;
}

// The tensor's device address: 1, -1 (no int), or 0 with an exception set.
int device_ptr(PyObject *t, const char *name, void **out) {
    PyObject *r = PyObject_GetAttr(t, s_is_cuda);
    if (r == nullptr) return 0;
    int yes = PyObject_IsTrue(r);
    Py_DECREF(r);
    if (yes < 0) return 0;
    if (yes == 0) {
        PyErr_Format(PyExc_ValueError, "%s must be a device tensor", name);
        return 0;
    }
    if ((r = PyObject_CallMethodNoArgs(t, s_is_contiguous)) == nullptr) return 0;
    yes = PyObject_IsTrue(r);
    Py_DECREF(r);
    if (yes < 0) return 0;
    if (yes == 0) {
        PyErr_Format(PyExc_ValueError, "%s must be contiguous", name);
        return 0;
    }
    if ((r = PyObject_CallMethodNoArgs(t, s_data_ptr)) == nullptr) return 0;
    const int rc = address(r, out);
    Py_DECREF(r);
    return rc;
}

// None: the current stream (of `device`, where the callable takes one); an int: a hipStream_t; anything
// else: its cuda_stream.
int stream_ptr(PyObject *stream, PyObject *current_stream, PyObject *device, void **out) {
    PyObject *r;
    if (stream == Py_None)
        r = device == nullptr ? PyObject_CallNoArgs(current_stream) : PyObject_CallOneArg(current_stream, device);
    else if (PyLong_Check(stream))
        r = Py_NewRef(stream);
    else
        r = PyObject_GetAttr(stream, s_cuda_stream);
    if (r == nullptr) return 0;
    const int rc = address(r, out);
    Py_DECREF(r);
    return rc;
}

PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 10) {
        PyErr_SetString(PyExc_TypeError, "linear takes 10 arguments");
        return nullptr;
    }
    const int split = PyObject_IsTrue(a[0]);
    if (split < 0) return nullptr;
    void *stream, *ws = nullptr, *x, *w, *y;
    int in, out, tokens;
    int rc = stream_ptr(a[9], a[1], nullptr, &stream);
    if (rc > 0 && a[8] != Py_None) rc = device_ptr(a[8], "ws", &ws);
    if (rc > 0) rc = device_ptr(a[2], "x", &x);
    if (rc > 0) rc = device_ptr(a[3], "w", &w);
    if (rc > 0) rc = device_ptr(a[4], "y", &y);
    if (rc > 0) rc = c_int(a[5], &in);
    if (rc > 0) rc = c_int(a[6], &out);
    if (rc > 0) rc = c_int(a[7], &tokens);
    if (rc == 0) return nullptr;
    if (rc < 0) Py_RETURN_NONE;
    Py_BEGIN_ALLOW_THREADS
    rc = split ? linear_q4_0s_forward_device(stream, ws, (const float *)x, w, (float *)y, in, out, tokens)
               : linear_q4_0_forward_device(stream, ws, (const float *)x, w, (float *)y, in, out, tokens);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// One argument of an entry: a tensor or an address, or a number.
union Arg {
    void *p;
    int64_t i;
};

#define P(k) a[k].p
#define I(k) ((int)a[k].i)
int run_quantize(void *s, const Arg *a) { return quantize_mxfp4_device(s, P(0), I(1), a[2].i, P(3), a[4].i, a[5].i); }
int run_dequantize(void *s, const Arg *a) {
    return dequantize_mxfp4_device(s, P(0), P(1), I(2), a[3].i, a[4].i, a[5].i);
}
int run_mat_mul(void *s, const Arg *a) {
    return mat_mul_mxfp4_device(P(0), P(1), P(2), I(3), I(4), I(5), I(6), s);
}
int run_linear(void *s, const Arg *a) {
    return linear_mxfp4_forward_device(s, P(0), P(1), I(2), P(3), P(4), I(5), I(6), I(7), I(8));
}
int run_grouped(void *s, const Arg *a) {
    return mat_mul_mxfp4_grouped_device(P(0), P(1), (const int32_t *)P(2), I(3), (const int32_t *)P(4), P(5), I(6), I(7),
                                        I(8), I(9), s);
}
int run_gate_up(void *s, const Arg *a) {
    return moe_mxfp4_gate_up_swiglu_device(s, P(0), P(1), P(2), (const int32_t *)P(3), I(4), P(5), I(6), I(7), I(8));
}
int run_ffn(void *s, const Arg *a) {
    return moe_mxfp4_ffn_forward_device(s, P(0), (const float *)P(1), P(2), P(3), P(4), P(5), I(6), I(7), I(8), I(9),
                                        I(10), I(11), P(12), a[13].i);
}
int run_dispatch(void *s, const Arg *a) {
    return moe_dispatch_rows_device(s, (const int32_t *)P(0), P(1), I(2), I(3), I(4), I(5), I(6), (int32_t *)P(7),
                                    (int32_t *)P(8), (int32_t *)P(9), P(10));
}
int run_dispatch_backward(void *s, const Arg *a) {
    return moe_dispatch_rows_backward_device(s, P(0), I(1), (const int32_t *)P(2), P(3), I(4), I(5), I(6));
}
int run_combine(void *s, const Arg *a) {
    return moe_combine_rows_device(s, P(0), I(1), (const int32_t *)P(2), (const float *)P(3), P(4), I(5), I(6), I(7));
}
int run_combine_backward(void *s, const Arg *a) {
    return moe_combine_rows_backward_device(s, P(0), P(1), I(2), (const int32_t *)P(3), (const float *)P(4), P(5),
                                            (float *)P(6), I(7), I(8), I(9));
}
#undef P
#undef I

constexpr int kMaxArgs = 14;
// The argument kinds: t a tensor or an address, o one that may be None, i a C int, l an int64_t.  The names
// stand in the messages of the arguments that are refused.
struct Entry {
    int (*run)(void *stream, const Arg *a);
    const char *kinds;
    const char *names[kMaxArgs];
};
const Entry kEntries[] = {
    {run_quantize, "tiltll", {"x", "dtype", "row_stride", "out", "rows", "cols"}},
    {run_dequantize, "ttilll", {"q", "y", "dtype", "row_stride", "rows", "cols"}},
    {run_mat_mul, "tttiiii", {"w", "xq", "y", "dtype", "K", "N", "M"}},
    {run_linear, "otittiiii", {"ws", "x", "dtype", "w", "y", "dtype", "in_features", "out_features", "num_tokens"}},
    {run_grouped, "tttiotiiii",
     {"w", "xq", "expert_offsets", "num_experts", "route_dst", "y", "dtype", "K", "N", "n_routes"}},
    {run_gate_up, "ttttitiii",
     {"w_gate", "w_up", "xq_perm", "offsets", "num_experts", "mid_q", "hidden", "inter", "n_routes"}},
    {run_ffn, "ttttttiiiiiitl",
     {"x", "logits", "w_gate", "w_up", "w_down", "y", "dtype", "num_tokens", "hidden", "inter", "num_experts", "top_k",
      "ws", "ws_bytes"}},
    {run_dispatch, "ttiiiiitttt",
     {"ids", "x", "dtype", "num_tokens", "top_k", "hidden", "num_experts", "offsets", "src_route", "dst_of_route",
      "x_sorted"}},
    {run_dispatch_backward, "tittiii",
     {"grad_sorted", "dtype", "dst_of_route", "grad_x", "num_tokens", "hidden", "top_k"}},
    {run_combine, "titttiii",
     {"expert_out", "dtype", "dst_of_route", "weights", "y", "num_tokens", "hidden", "top_k"}},
    {run_combine_backward, "ttittttiii",
     {"grad_y", "expert_out", "dtype", "dst_of_route", "weights", "grad_expert_out", "grad_weights", "num_tokens",
      "hidden", "top_k"}},
};

// A tensor's or an int's address; false with an exception set.
bool entry_ptr(PyObject *t, const char *name, long device, void **out) {
    if (PyLong_Check(t)) {
        *out = PyLong_AsVoidPtr(t);
        return *out != nullptr || !PyErr_Occurred();
    }
    PyObject *r = PyObject_CallMethodNoArgs(t, s_get_device);
    if (r == nullptr) return false;
    const long on = PyLong_AsLong(r);
    Py_DECREF(r);
    if (on == -1 && PyErr_Occurred()) return false;
    if (on < 0) {
        PyErr_Format(PyExc_ValueError, "%s must be a device tensor", name);
        return false;
    }
    if (on != device) {
        PyErr_Format(PyExc_ValueError, "%s is on device %ld, the current device is %ld", name, on, device);
        return false;
    }
    if ((r = PyObject_CallMethodNoArgs(t, s_is_contiguous)) == nullptr) return false;
    const int yes = PyObject_IsTrue(r);
    Py_DECREF(r);
    if (yes < 0) return false;
    if (yes == 0) {
        PyErr_Format(PyExc_ValueError, "%s must be contiguous", name);
        return false;
    }
    if ((r = PyObject_CallMethodNoArgs(t, s_data_ptr)) == nullptr) return false;
    *out = PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    return *out != nullptr || !PyErr_Occurred();
}

// An int (or an object with __index__) in the range of its C type; false with an exception set.
bool entry_int(PyObject *o, const char *name, bool wide, int64_t *out) {
    PyObject *n = PyNumber_Index(o);
    if (n == nullptr) {
        PyErr_Format(PyExc_TypeError, "%s must be an int", name);
        return false;
    }
    int over = 0;
    *out = PyLong_AsLongLongAndOverflow(n, &over);
    Py_DECREF(n);
    if (over != 0 || (!wide && *out != (int)*out)) {
        PyErr_Format(PyExc_ValueError, "%s is out of range", name);
        return false;
    }
    return true;
}

PyObject *entry(PyObject *, PyObject *const *a, Py_ssize_t n) {
    const long which = n >= 4 ? PyLong_AsLong(a[0]) : -1;
    if (which < 0 || which >= (long)(sizeof kEntries / sizeof kEntries[0])) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "entry: unknown entry");
        return nullptr;
    }
    const Entry &e = kEntries[which];
    const char *kinds = e.kinds;
    if (n - 4 != (Py_ssize_t)strlen(kinds)) {
        PyErr_SetString(PyExc_TypeError, "entry: wrong number of arguments");
        return nullptr;
    }
    PyObject *r = PyObject_CallNoArgs(a[2]);
    if (r == nullptr) return nullptr;
    const long device = PyLong_AsLong(r);
    void *stream;
    int rc = device == -1 && PyErr_Occurred() ? 0 : stream_ptr(a[3], a[1], r, &stream);
    Py_DECREF(r);
    if (rc == 0) return nullptr;
    if (rc < 0) {
        PyErr_SetString(PyExc_TypeError, "stream must be a stream, its address or None");
        return nullptr;
    }
    Arg args[kMaxArgs];
    for (int k = 0; kinds[k] != 0; ++k) {
        PyObject *o = a[4 + k];
        if (kinds[k] == 'i' || kinds[k] == 'l') {
            if (!entry_int(o, e.names[k], kinds[k] == 'l', &args[k].i)) return nullptr;
        } else if (kinds[k] == 'o' && o == Py_None) {
            args[k].p = nullptr;
        } else if (!entry_ptr(o, e.names[k], device, &args[k].p)) {
            return nullptr;
        }
    }
    Py_BEGIN_ALLOW_THREADS
    rc = e.run(stream, args);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

PyMethodDef methods[] = {
    {"entry", (PyCFunction)(void (*)(void))entry, METH_FASTCALL, "One MXFP4 or sorted-row entry on device tensors."},
    {"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, "One linear layer on device tensors."},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_linear", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__linear(void) {
    s_is_cuda = PyUnicode_InternFromString("is_cuda");
    s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_cuda_stream = PyUnicode_InternFromString("cuda_stream");
    s_get_device = PyUnicode_InternFromString("get_device");
    if (s_get_device == nullptr || s_is_cuda == nullptr || s_is_contiguous == nullptr || s_data_ptr == nullptr ||
        s_cuda_stream == nullptr)
        return nullptr;
    return PyModule_Create(&module);
}
