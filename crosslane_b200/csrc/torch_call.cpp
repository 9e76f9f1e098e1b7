// The Python face of the operators around the routed experts (block_ops.py): checks torch
// tensors and calls the C entry points (include/crosslane_b200.h). A decode step makes these
// calls once a layer with a few microseconds of GPU work each; the same checks in Python take
// 3 to 5 us a call on top of the launch's 3, here a few tenths of one.
//
// The module links no CUDA code of this project: the entry points' addresses come from the
// library that the ctypes binding loaded (bind), so both always call the same build.
#include <Python.h>

#include <cstdarg>
#include <cstdio>
#include <cstring>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/crosslane_b200.h"

namespace {

decltype(&clb_route_experts_device) g_route;
decltype(&clb_block_norm_device) g_norm;
decltype(&clb_int8_quantize_device) g_quantize;
decltype(&clb_int8_linear_device) g_linear;
PyObject* g_error;  // ClbError(code, message)

enum Kind : int { kF32 = CLB_F32, kBF16 = CLB_BF16, kF16 = CLB_F16, kI8 = CLB_I8, kI32, kU8, kOther };
constexpr unsigned bit(int k) { return 1u << k; }
constexpr unsigned kFloats = bit(kF32) | bit(kBF16) | bit(kF16);
const char* const kNames[] = {"float32", "bfloat16", "float16", "int8", "int32", "uint8"};

struct Refused {};  // a Python error is set

[[noreturn]] void refuse(int code, const char* fmt, ...) {
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    if (PyObject* e = PyObject_CallFunction(g_error, "is", code, text)) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw Refused{};
}

const char* kind_names(unsigned kinds, char (&text)[96]) {
    text[0] = 0;
    for (int k = 0; k < kOther; ++k)
        if (kinds & bit(k)) {
            if (text[0]) std::strcat(text, " / ");
            std::strcat(text, kNames[k]);
        }
    return text;
}

struct Rows {
    int kind;
    int device;
    int64_t n, w, ld;  // rows, their length and pitch (a single row: its length)
    void* p;
};

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "%s: a torch tensor is needed, not %s", name, Py_TYPE(o)->tp_name);
        throw Refused{};
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    // torch negates such a view's values when it reads them (the imaginary part of a conjugated tensor is one)
    if (t.is_neg()) refuse(CLB_E_INVALID, "%s: a lazily negated view (resolve_neg gives its values)", name);
    return t;
}
int kind_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return kF32;
        case at::kBFloat16: return kBF16;
        case at::kHalf: return kF16;
        case at::kChar: return kI8;
        case at::kInt: return kI32;
        case at::kByte: return kU8;
        default: return kOther;
    }
}
int device_of(const at::Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }

// A [tokens][width] tensor of one of `kinds` with its last stride 1, on `device` (-2: any; tokens or
// width -1: any).
Rows rows(PyObject* o, const char* name, unsigned kinds, int device, int64_t tokens, int64_t width) {
    const at::Tensor& t = tensor(o, name);
    Rows r;
    char text[96];
    r.kind = kind_of(t);
    if (!(kinds & bit(r.kind)) || t.layout() != at::kStrided || t.dim() != 2 || (device != -2 && device_of(t) != device))
        refuse(CLB_E_INVALID, "%s: a 2-D tensor of %s on the operator's device is needed", name, kind_names(kinds, text));
    r.device = device_of(t);
    r.n = t.size(0), r.w = t.size(1);
    if ((tokens >= 0 && r.n != tokens) || (width >= 0 && r.w != width))
        refuse(CLB_E_INVALID, "%s is (%lld, %lld), not (%lld, %lld)", name, (long long)r.n, (long long)r.w, (long long)tokens,
               (long long)width);
    if (r.w > 1 && t.stride(1) != 1) refuse(CLB_E_INVALID, "%s: the last stride is %lld, not 1", name, (long long)t.stride(1));
    r.ld = r.n > 1 ? t.stride(0) : r.w;
    if (r.ld < r.w) refuse(CLB_E_INVALID, "%s: rows overlap (stride %lld, width %lld)", name, (long long)r.ld, (long long)r.w);
    if (r.n > INT32_MAX || r.w > INT32_MAX) refuse(CLB_E_INVALID, "%s: more than 2^31 - 1 rows or columns", name);
    r.p = t.numel() ? t.data_ptr() : nullptr;
    return r;
}
// The same, the rows one behind the other.
void* dense(PyObject* o, const char* name, int kind, int device, int64_t tokens, int64_t width) {
    const Rows r = rows(o, name, bit(kind), device, tokens, width);
    if (r.ld != width) refuse(CLB_E_INVALID, "%s: a contiguous tensor is needed", name);
    return r.p;
}
// A contiguous vector of n (-1: any); null for None.
void* vector(PyObject* o, const char* name, unsigned kinds, int device, int64_t n, int* kind = nullptr, uint64_t* count = nullptr) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor(o, name);
    char text[96];
    const int k = kind_of(t);
    if (!(kinds & bit(k)) || t.layout() != at::kStrided || t.dim() != 1 || (n >= 0 && t.size(0) != n) || device_of(t) != device ||
        (t.size(0) > 1 && t.stride(0) != 1))
        refuse(CLB_E_INVALID, "%s: a contiguous vector of %lld %s on the operator's device is needed", name,
               (long long)(n >= 0 ? n : t.size(0)), kind_names(kinds, text));
    if (kind) *kind = k;
    if (count) *count = (uint64_t)t.size(0);
    return t.numel() ? t.data_ptr() : nullptr;
}

void on_cuda(int device, const char* what) {
    if (device < 0) refuse(CLB_E_INVALID, "%s: not on a CUDA device", what);
}

// The stream of a call: the given address, or the device's current one.
void* stream_of(PyObject* o, int device) {
    if (o == Py_None) return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    void* s = PyLong_AsVoidPtr(o);
    if (PyErr_Occurred()) throw Refused{};
    return s;
}

template <class T>
T config(PyObject* o) {
    T c;
    if (!PyBytes_Check(o) || PyBytes_GET_SIZE(o) != (Py_ssize_t)sizeof c) {
        PyErr_SetString(PyExc_TypeError, "not this operator's configuration");
        throw Refused{};
    }
    std::memcpy(&c, PyBytes_AS_STRING(o), sizeof c);
    return c;
}

void arguments(Py_ssize_t got, Py_ssize_t want) {
    if (got != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", got, want);
        throw Refused{};
    }
}

// `body(err)` with the device current; a status of the entry point becomes a ClbError.
template <class F>
void call(int device, F&& body) {
    const c10::cuda::OptionalCUDAGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)device));
    clb_error_v1 err;
    const int rc = body(&err);
    if (rc != CLB_OK) refuse(rc, "%s", err.message);
}

template <class F>
PyObject* python(F&& body) {
    try {
        body();
        Py_RETURN_NONE;
    } catch (const Refused&) {
    } catch (const std::exception& e) {  // torch: a tensor without storage, no CUDA
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// route(config, logits, ids, w, bias, status, stream)
PyObject* py_route(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return python([&] {
        arguments(n, 7);
        clb_route_config_v1 c = config<clb_route_config_v1>(a[0]);
        const Rows l = rows(a[1], "logits", kFloats, -2, -1, c.n_experts);
        void* ids = dense(a[2], "ids", kI32, l.device, l.n, c.k);
        void* w = dense(a[3], "weights", kF32, l.device, l.n, c.k);
        void* bias = vector(a[4], "bias", bit(kF32), l.device, c.n_experts);
        void* status = vector(a[5], "status", bit(kI32), l.device, 1);
        on_cuda(l.device, "logits");
        c.logits_type = l.kind;
        call(l.device, [&](clb_error_v1* err) {
            return g_route(&c, l.p, l.ld, static_cast<float*>(bias), (int32_t)l.n, static_cast<int32_t*>(ids),
                           static_cast<float*>(w), static_cast<int32_t*>(status), stream_of(a[6], l.device), err);
        });
    });
}

// norm(config, pre, h, y, gate, w_post, w_pre, h_out, x, stream)
PyObject* py_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return python([&] {
        arguments(n, 10);
        clb_block_norm_config_v1 c = config<clb_block_norm_config_v1>(a[0]);
        const Rows h = rows(a[2], "h", kFloats, -2, -1, c.dim);
        const int d = h.device;
        c.h_type = h.kind, c.ld_h = h.ld;
        void *y = nullptr, *gate = nullptr, *out = nullptr, *x = nullptr;
        if ((a[8] != Py_None) != (a[1] == Py_True)) refuse(CLB_E_INVALID, "x goes with the norm before the next block");
        if ((a[3] != Py_None) != (a[7] != Py_None)) refuse(CLB_E_INVALID, "h_out goes with y");
        if (a[3] != Py_None) {
            const Rows r = rows(a[3], "y", kFloats, d, h.n, c.dim), o = rows(a[7], "h_out", bit(h.kind), d, h.n, c.dim);
            c.y_type = r.kind, c.ld_y = r.ld, y = r.p;
            c.ld_h_out = o.ld, out = o.p;
        }
        if (a[4] != Py_None) {
            if (c.gate == CLB_GATE_FULL) {
                const Rows r = rows(a[4], "gate", kFloats, d, h.n, c.dim);
                c.gate_type = r.kind, c.ld_gate = r.ld, gate = r.p;
            } else {
                int kind = 0;
                gate = vector(a[4], "gate", kFloats, d, c.gate == CLB_GATE_CHANNEL ? c.dim : h.n, &kind);
                c.gate_type = kind;
            }
        }
        void* w_post = vector(a[5], "w_post", bit(kF32), d, c.dim);
        void* w_pre = vector(a[6], "w_pre", bit(kF32), d, c.dim);
        if (a[8] != Py_None) {
            const Rows r = rows(a[8], "x", kFloats, d, h.n, c.dim);
            c.x_type = r.kind, c.ld_x = r.ld, x = r.p;
        }
        on_cuda(d, "h");
        call(d, [&](clb_error_v1* err) {
            return g_norm(&c, (int32_t)h.n, h.p, y, gate, static_cast<float*>(w_post), static_cast<float*>(w_pre), out, x,
                          stream_of(a[9], d), err);
        });
    });
}

// The pitch of int8 rows; that of a single row is never used.
int64_t pitch16(const Rows& r) { return r.n <= 1 ? (r.w + 15) / 16 * 16 : r.ld; }

// quantize(x, q, scale, stream)
PyObject* py_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return python([&] {
        arguments(n, 4);
        const Rows x = rows(a[0], "x", kFloats, -2, -1, -1);
        const Rows q = rows(a[1], "q", bit(kI8), x.device, x.n, x.w);
        if (a[2] == Py_None) refuse(CLB_E_INVALID, "scale: a vector is needed");
        void* scale = vector(a[2], "scale", bit(kF32), x.device, x.n);
        on_cuda(x.device, "x");
        call(x.device, [&](clb_error_v1* err) {
            return g_quantize(x.kind, x.p, x.ld, (int32_t)x.n, (int32_t)x.w, static_cast<int8_t*>(q.p), pitch16(q),
                              static_cast<float*>(scale), stream_of(a[3], x.device), err);
        });
    });
}

// weights(w, w_scale, bias) -> (n, k, row pitch): the checks of a linear's own tensors
PyObject* py_weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
    Rows w{};
    PyObject* none = python([&] {
        arguments(n, 3);
        w = rows(a[0], "w", bit(kI8), -2, -1, -1);
        if (a[1] == Py_None) refuse(CLB_E_INVALID, "w_scale: a vector is needed");
        vector(a[1], "w_scale", bit(kF32), w.device, w.n);
        vector(a[2], "bias", bit(kF32), w.device, w.n);
    });
    if (!none) return nullptr;
    Py_DECREF(none);
    return Py_BuildValue("LLL", (long long)w.n, (long long)w.w, (long long)pitch16(w));
}

// linear(config, w, w_scale, bias, x, out, ws, x_scale, status, stream). The linear's own tensors are checked again: they
// may have been replaced or changed in place (moved, resized) since weights.
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return python([&] {
        arguments(n, 10);
        clb_int8_linear_config_v1 c = config<clb_int8_linear_config_v1>(a[0]);
        const Rows w = rows(a[1], "w", bit(kI8), -2, c.n, c.k);
        const int d = w.device;
        if (a[2] == Py_None) refuse(CLB_E_INVALID, "w_scale: a vector is needed");
        void* w_scale = vector(a[2], "w_scale", bit(kF32), d, c.n);
        void* bias = vector(a[3], "bias", bit(kF32), d, c.n);
        on_cuda(d, "the weights");
        c.ld_w = pitch16(w);
        const Rows x = rows(a[4], "x", kFloats | bit(kI8), d, -1, c.k), o = rows(a[5], "out", kFloats, d, x.n, c.n);
        c.x_type = x.kind, c.ld_x = x.kind == kI8 ? pitch16(x) : x.ld;
        c.out_type = o.kind, c.ld_out = o.ld;
        uint64_t ws_bytes = 0;
        void* ws = vector(a[6], "workspace", bit(kU8), d, -1, nullptr, &ws_bytes);
        void* scale = vector(a[7], "x_scale", bit(kF32), d, x.n);
        void* status = vector(a[8], "status", bit(kI32), d, 1);
        call(d, [&](clb_error_v1* err) {
            return g_linear(&c, static_cast<int8_t*>(w.p), static_cast<float*>(w_scale), static_cast<float*>(bias),
                            (int32_t)x.n, x.p, static_cast<float*>(scale), o.p, ws, ws_bytes, static_cast<int32_t*>(status),
                            stream_of(a[9], d), err);
        });
    });
}

// bind(route, norm, quantize, linear, ClbError): addresses of the entry points
PyObject* py_bind(PyObject*, PyObject* args) {
    PyObject *f[4], *error;
    if (!PyArg_ParseTuple(args, "OOOOO", &f[0], &f[1], &f[2], &f[3], &error)) return nullptr;
    void* p[4];
    for (int i = 0; i < 4; ++i)
        if (!(p[i] = PyLong_AsVoidPtr(f[i]))) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
            return nullptr;
        }
    g_route = reinterpret_cast<decltype(g_route)>(p[0]);
    g_norm = reinterpret_cast<decltype(g_norm)>(p[1]);
    g_quantize = reinterpret_cast<decltype(g_quantize)>(p[2]);
    g_linear = reinterpret_cast<decltype(g_linear)>(p[3]);
    Py_INCREF(error);
    Py_XSETREF(g_error, error);
    Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef kMethods[] = {{"bind", py_bind, METH_VARARGS, nullptr},
                          {"route", FAST(py_route), METH_FASTCALL, nullptr},
                          {"norm", FAST(py_norm), METH_FASTCALL, nullptr},
                          {"quantize", FAST(py_quantize), METH_FASTCALL, nullptr},
                          {"weights", FAST(py_weights), METH_FASTCALL, nullptr},
                          {"linear", FAST(py_linear), METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_call", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyMODINIT_FUNC PyInit__torch_call(void) { return PyModule_Create(&kModule); }
