// The regular calls of the small-launch operators without Python in between: a tensor's
// pointer, sizes and strides go straight into the C-ABI's descriptors and the result is
// allocated here.  A launch takes about 3 us of host time; describing five tensors through
// ctypes and allocating the result from Python takes 6 to 8 more, which is what a projection
// of one token would then wait for.
//
// Only what is in order is handled: exact torch tensors on the current device, matching
// widths, a status of H3_OK.  Anything else returns None before or without effect, and the
// Python wrapper takes the ctypes path, whose checks raise the errors; there is no second
// implementation of any check or op here.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/h3_b200.h"

namespace {

using QuantizeFn = decltype(&h3_quantize_fp4);
using DequantizeFn = decltype(&h3_dequantize_fp4);
using LinearFn = decltype(&h3_linear_fp4);
using CrossFn = decltype(&h3_cross_attention);

QuantizeFn g_quantize;
DequantizeFn g_dequantize;
LinearFn g_linear;
CrossFn g_cross;

// The exact tensor behind `o`, on the device `dev` (or, with dev < 0, on the current one,
// which is then returned in dev); null if it is anything else.
const at::Tensor *tensor_on(PyObject *o, int *dev) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || t.dim() > H3_MAX_DIMS) return nullptr;
    if (*dev < 0) {
        *dev = (int)c10::cuda::current_device();
    }
    return t.get_device() == *dev ? &t : nullptr;
}

bool describe(const at::Tensor &t, h3_tensor *d) {
    std::memset(d, 0, sizeof *d);
    switch (t.scalar_type()) {
        case at::kBFloat16: d->dtype = H3_BF16; break;
        case at::kLong: d->dtype = H3_I64; break;
        case at::kByte: d->dtype = H3_U8; break;
        default: return false;
    }
    d->data = t.data_ptr();
    d->ndim = (int32_t)t.dim();
    for (int i = 0; i < d->ndim; ++i) {
        d->shape[i] = t.size(i);
        d->strides[i] = t.stride(i);
    }
    return true;
}

// [..., C] as its rows where that needs no copy
bool describe_rows(const at::Tensor &t, h3_tensor *d) {
    if (t.dim() < 2 || !describe(t, d)) return false;
    if (t.dim() == 2) return true;
    if (!t.is_contiguous()) return false;
    const int64_t cols = t.size(-1);
    int64_t rows = 1;
    for (int i = 0; i < t.dim() - 1; ++i) rows *= t.size(i);
    d->ndim = 2;
    d->shape[0] = rows, d->shape[1] = cols;
    d->strides[0] = cols, d->strides[1] = 1;
    return true;
}

h3_tensor bytes(void *data, std::initializer_list<int64_t> shape) {
    h3_tensor d;
    std::memset(&d, 0, sizeof d);
    d.data = data;
    d.dtype = H3_U8;
    d.ndim = (int32_t)shape.size();
    int i = 0;
    for (int64_t s : shape) d.shape[i++] = s;
    int64_t stride = 1;
    for (i = d.ndim - 1; i >= 0; --i) {
        d.strides[i] = stride;
        stride *= d.shape[i];
    }
    return d;
}

// a descriptor's bytes, as the Python side keeps those of a 4-bit matrix
const h3_tensor *held(PyObject *o) {
    if (!PyBytes_CheckExact(o) || PyBytes_GET_SIZE(o) != (Py_ssize_t)sizeof(h3_tensor)) return nullptr;
    return reinterpret_cast<const h3_tensor *>(PyBytes_AS_STRING(o));
}
PyObject *as_bytes(const h3_tensor &d) { return PyBytes_FromStringAndSize(reinterpret_cast<const char *>(&d), sizeof d); }

void *stream(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

template <typename F>
int unlocked(F f) {
    int status;
    Py_BEGIN_ALLOW_THREADS;
    status = f();
    Py_END_ALLOW_THREADS;
    return status;
}

// C++ exceptions (out of memory, say) stay here: the Python path meets the same one
template <typename F>
PyObject *guarded(F f) {
    PyObject *r = nullptr;
    try {
        r = f();
    } catch (...) {
        r = nullptr;
    }
    if (r) return r;
    if (PyErr_Occurred()) PyErr_Clear();
    Py_RETURN_NONE;
}

// bind(address of h3_quantize_fp4, h3_dequantize_fp4, h3_linear_fp4, h3_cross_attention)
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    if (n != 4) {
        PyErr_SetString(PyExc_TypeError, "bind takes four addresses");
        return nullptr;
    }
    g_quantize = reinterpret_cast<QuantizeFn>(PyLong_AsVoidPtr(a[0]));
    g_dequantize = reinterpret_cast<DequantizeFn>(PyLong_AsVoidPtr(a[1]));
    g_linear = reinterpret_cast<LinearFn>(PyLong_AsVoidPtr(a[2]));
    g_cross = reinterpret_cast<CrossFn>(PyLong_AsVoidPtr(a[3]));
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
}

// quantize_fp4(x, format, tensor scale) -> (buffer, descriptor of codes, of scales, rows, cols)
PyObject *quantize(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        int dev = -1;
        h3_tensor x;
        if (n != 3 || !g_quantize) return nullptr;
        const at::Tensor *t = tensor_on(a[0], &dev);
        if (!t || !describe_rows(*t, &x) || x.shape[1] < 1) return nullptr;
        const int fmt = (int)PyLong_AsLong(a[1]);
        const float scale = (float)PyFloat_AsDouble(a[2]);
        if (PyErr_Occurred()) return nullptr;
        const int64_t rows = x.shape[0], cols = x.shape[1], per = fmt == H3_MXFP4 ? 128 : 64;
        const int64_t pitch = (cols + 31) / 32 * 16, groups = (rows + 127) / 128, chunks = (cols + per - 1) / per;
        at::Tensor buf = at::empty({rows * pitch + groups * chunks * 512}, t->options().dtype(at::kByte));
        uint8_t *at = static_cast<uint8_t *>(buf.data_ptr());
        const h3_tensor codes = bytes(at, {rows, pitch}), scales = bytes(at + rows * pitch, {groups, chunks, 512});
        void *s = stream(dev);
        if (unlocked([&] { return g_quantize(&codes, &scales, &x, fmt, scale, s); }) != H3_OK) return nullptr;
        PyObject *b = THPVariable_Wrap(std::move(buf)), *c = as_bytes(codes), *d = as_bytes(scales);
        return Py_BuildValue("(NNNLL)", b, c, d, (long long)rows, (long long)cols);
    });
}

// dequantize_fp4(buffer, descriptor of codes, of scales, rows, cols, format, tensor scale) -> values
PyObject *dequantize(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        int dev = -1;
        if (n != 7 || !g_dequantize) return nullptr;
        const at::Tensor *buf = tensor_on(a[0], &dev);
        const h3_tensor *codes = held(a[1]), *scales = held(a[2]);
        if (!buf || !codes || !scales) return nullptr;
        const int64_t rows = PyLong_AsLongLong(a[3]), cols = PyLong_AsLongLong(a[4]);
        const int fmt = (int)PyLong_AsLong(a[5]);
        const float scale = (float)PyFloat_AsDouble(a[6]);
        if (PyErr_Occurred()) return nullptr;
        at::Tensor out = at::empty({rows, cols}, buf->options().dtype(at::kBFloat16));
        h3_tensor y;
        if (!describe(out, &y)) return nullptr;
        void *s = stream(dev);
        if (unlocked([&] { return g_dequantize(&y, codes, scales, fmt, scale, s); }) != H3_OK) return nullptr;
        return THPVariable_Wrap(std::move(out));
    });
}

// linear_fp4(x, weight's buffer, descriptor of codes, of scales, rows, cols, bias or None, format,
//            x's tensor scale, weight's, rows up to which the product quantises x itself) -> y
PyObject *linear(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        int dev = -1;
        h3_tensor x, y, bias, work;
        if (n != 11 || !g_linear) return nullptr;
        const at::Tensor *t = tensor_on(a[0], &dev), *w = t ? tensor_on(a[1], &dev) : nullptr;
        const h3_tensor *codes = held(a[2]), *scales = held(a[3]);
        if (!w || !codes || !scales || !describe_rows(*t, &x)) return nullptr;
        const int64_t outs = PyLong_AsLongLong(a[4]), cols = PyLong_AsLongLong(a[5]);
        const bool has_bias = a[6] != Py_None;
        if (has_bias) {
            const at::Tensor *b = tensor_on(a[6], &dev);
            if (!b || !describe(*b, &bias)) return nullptr;
        }
        const int fmt = (int)PyLong_AsLong(a[7]);
        const float tx = (float)PyFloat_AsDouble(a[8]), tw = (float)PyFloat_AsDouble(a[9]);
        const int64_t fused = PyLong_AsLongLong(a[10]);
        if (PyErr_Occurred() || x.shape[1] != cols) return nullptr;
        const int64_t rows = x.shape[0], per = fmt == H3_MXFP4 ? 128 : 64;
        at::DimVector sizes(t->sizes().begin(), t->sizes().end());
        sizes.back() = outs;
        at::Tensor out = at::empty(sizes, w->options().dtype(at::kBFloat16)), held_x;
        if (!describe_rows(out, &y)) return nullptr;
        const bool inside = rows <= fused;
        if (!inside) {
            held_x = at::empty({rows * ((cols + 31) / 32 * 16) + (rows + 127) / 128 * ((cols + per - 1) / per) * 512},
                               w->options().dtype(at::kByte));
            if (!describe(held_x, &work)) return nullptr;
        }
        void *s = stream(dev);
        if (unlocked([&] {
                return g_linear(&y, &x, inside ? nullptr : &work, codes, scales, has_bias ? &bias : nullptr, fmt, tx,
                                tw, s);
            }) != H3_OK)
            return nullptr;
        return THPVariable_Wrap(std::move(out));
    });
}

// cross_attention(q, k, v, lengths or None, scale) -> out
PyObject *cross(PyObject *, PyObject *const *a, Py_ssize_t n) {
    return guarded([&]() -> PyObject * {
        int dev = -1;
        h3_tensor d[5];
        if (n != 5 || !g_cross) return nullptr;
        const at::Tensor *q = tensor_on(a[0], &dev);
        if (!q || !describe(*q, &d[1])) return nullptr;
        const bool ragged = a[3] != Py_None;
        for (int i = 1; i < (ragged ? 4 : 3); ++i) {
            const at::Tensor *t = tensor_on(a[i], &dev);
            if (!t || !describe(*t, &d[i + 1])) return nullptr;
        }
        const float scale = (float)PyFloat_AsDouble(a[4]);
        if (PyErr_Occurred()) return nullptr;
        at::Tensor out = at::empty(q->sizes(), q->options());
        if (!describe(out, &d[0])) return nullptr;
        void *s = stream(dev);
        if (unlocked([&] { return g_cross(&d[0], &d[1], &d[2], &d[3], ragged ? &d[4] : nullptr, scale, s); }) != H3_OK)
            return nullptr;
        return THPVariable_Wrap(std::move(out));
    });
}

#define H3_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(fn)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {H3_METHOD("bind", bind),       H3_METHOD("quantize_fp4", quantize),
                           H3_METHOD("dequantize_fp4", dequantize), H3_METHOD("linear_fp4", linear),
                           H3_METHOD("cross_attention", cross), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_h3host", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__h3host(void) { return PyModule_Create(&g_module); }
