// The ordinary calls of ops.quantize_rows, inner_prod_quantized and group_norm_nhwc, from Python straight to the C ABI: tensors on the
// current device and stream, rows and images that lie one after the other, outputs that are allocated.  A kernel of these can be done in
// 2 us, where the checks, the allocations and the call take some 8 us in Python and half of that here.
//
// Each function returns its result, or None for any call that is not an ordinary one, wrong ones among them: ops.py then makes the same call
// by its general way, which takes every layout that there is and says what is wrong with the others.  (A status other than TSB_OK means that
// nothing was launched, so that way may be gone again.)
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/tennis_b200.h"

namespace {

using at::Tensor;

bool type_of(at::ScalarType t, int *type) {
    switch (t) {
        case at::kFloat: *type = TSB_TYPE_F32; return true;
        case at::kHalf: *type = TSB_TYPE_F16; return true;
        case at::kBFloat16: *type = TSB_TYPE_BF16; return true;
        default: return false;
    }
}

Tensor room(at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType type, c10::Device device) {
    return at::Tensor(at::detail::empty_strided_cuda(sizes, strides, type, device));
}
Tensor bytes(int64_t n, c10::Device device) { return room({n}, {1}, at::kByte, device); }

// A tensor argument on `device` (-1: any CUDA device that is the current one); NULL for anything else
const Tensor *tensor(PyObject *o, int device) {
    if (!THPVariable_Check(o)) return nullptr;
    const Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || (device >= 0 && t.get_device() != device) || (device < 0 && t.get_device() != c10::cuda::current_device())) return nullptr;
    return &t;
}

// A vector of `size` floats or None; false for anything else
bool vector(PyObject *o, int64_t size, int device, const float **at) {
    *at = nullptr;
    if (o == Py_None) return true;
    const Tensor *t = tensor(o, device);
    if (!t || t->scalar_type() != at::kFloat || t->numel() != size || !t->is_contiguous()) return false;
    *at = static_cast<const float *>(t->const_data_ptr());
    return true;
}

// The rows of t [..., k]: how many, and the elements between them
bool rows_of(const Tensor &t, int64_t *rows, int64_t *pitch) {
    const int64_t dims = t.dim();
    if (dims < 1) return false;
    const int64_t k = t.size(dims - 1);
    if (k < 1) return false;
    if (dims == 2 && (t.stride(1) == 1 || k == 1)) {
        *rows = t.size(0);
        *pitch = t.stride(0);
        return true;
    }
    if (!t.is_contiguous()) return false;
    *rows = t.numel() / k;
    *pitch = k;
    return true;
}

// An int argument; -1, which is none of the values that the C ABI takes, for numbers that an int does not hold
int int_of(PyObject *o) {
    const long v = PyLong_AsLong(o);
    return v == (int)v ? (int)v : -1;
}

void *stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// The sizes of x with another last one
c10::SmallVector<int64_t, 6> sizes_with(const Tensor &x, int64_t last) {
    c10::SmallVector<int64_t, 6> s(x.sizes().begin(), x.sizes().end());
    s.back() = last;
    return s;
}
Tensor dense(const Tensor &x, int64_t last, at::ScalarType type) {
    const auto sizes = sizes_with(x, last);
    c10::SmallVector<int64_t, 6> strides(sizes.size());
    int64_t step = 1;
    for (size_t i = sizes.size(); i-- > 0;) {
        strides[i] = step;
        step *= sizes[i] > 0 ? sizes[i] : 1;
    }
    return room(sizes, strides, type, x.device());
}

// quantize_rows(x) -> (q, scales)
PyObject *quantize_rows(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    const Tensor *x = count == 1 ? tensor(args[0], -1) : nullptr;
    int type;
    int64_t rows, pitch;
    if (!x || !type_of(x->scalar_type(), &type) || !rows_of(*x, &rows, &pitch)) Py_RETURN_NONE;
    const int64_t k = x->size(-1), room_k = (k + 15) / 16 * 16;
    if (x->dim() != 2 && (x->dim() == 1 || room_k != k)) Py_RETURN_NONE;
    const Tensor q = x->dim() == 2 ? room({rows, k}, {room_k, 1}, at::kChar, x->device()) : dense(*x, k, at::kChar);
    c10::SmallVector<int64_t, 6> lead(x->sizes().begin(), x->sizes().end() - 1);
    Tensor s = room({rows}, {1}, at::kFloat, x->device());
    if (x->dim() != 2) s = s.view(lead);
    const int device = x->get_device();
    if (tsb_quantize_rows_i8(x->const_data_ptr(), type, pitch, static_cast<int8_t *>(q.mutable_data_ptr()), room_k, static_cast<float *>(s.mutable_data_ptr()), rows, k, stream_of(device)) != TSB_OK)
        Py_RETURN_NONE;
    PyObject *pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(q));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(s));
    return pair;
    END_HANDLE_TH_ERRORS
}

// inner_prod(x, x_scales, w, w_scales, bias, residual, activation, leaky, out_dtype, residual_after) -> y
PyObject *inner_prod(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    const Tensor *x = count == 10 ? tensor(args[0], -1) : nullptr;
    if (!x) Py_RETURN_NONE;
    const int device = x->get_device();
    const Tensor *w = tensor(args[2], device);
    tsb_inner_prod_args a = {};
    if (!w || w->scalar_type() != at::kChar || w->dim() != 2 || !rows_of(*x, &a.m, &a.x_pitch)) Py_RETURN_NONE;
    a.n = w->size(0);
    a.k = w->size(1);
    if (a.m < 1 || a.n < 1 || x->size(-1) != a.k || (w->stride(1) != 1 && a.k > 1)) Py_RETURN_NONE;
    a.w_pitch = w->stride(0);
    at::ScalarType out = at::kFloat;
    if (args[1] == Py_None) {
        if (!type_of(x->scalar_type(), &a.x_type)) Py_RETURN_NONE;
        out = x->scalar_type();
    } else {
        const Tensor *xs = tensor(args[1], device);
        if (x->scalar_type() != at::kChar || !xs || !vector(args[1], xs->numel() == 1 ? 1 : a.m, device, &a.x_scales)) Py_RETURN_NONE;
        a.x_type = TSB_TYPE_I8;
        a.x_scales_stride = xs->numel() == 1 ? 0 : 1;
    }
    if (args[8] != Py_None) {
        if (!THPDtype_Check(args[8])) Py_RETURN_NONE;
        out = reinterpret_cast<THPDtype *>(args[8])->scalar_type;
    }
    if (!type_of(out, &a.y_type) || args[3] == Py_None || !vector(args[3], a.n, device, &a.w_scales) || !vector(args[4], a.n, device, &a.bias)) Py_RETURN_NONE;
    if (args[5] != Py_None) {
        const Tensor *r = tensor(args[5], device);
        int64_t rows;
        if (!r || r->scalar_type() != out || r->dim() != x->dim() || r->size(-1) != a.n || !rows_of(*r, &rows, &a.residual_pitch) || rows != a.m ||
            r->sizes().slice(0, r->dim() - 1) != x->sizes().slice(0, x->dim() - 1))
            Py_RETURN_NONE;
        a.residual = r->const_data_ptr();
    }
    a.activation = int_of(args[6]);
    a.leaky_scale = (float)PyFloat_AsDouble(args[7]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    a.residual_after_activation = args[9] == Py_True;
    a.x = x->const_data_ptr();
    a.w = static_cast<const int8_t *>(w->const_data_ptr());
    const Tensor y = dense(*x, a.n, out);
    a.y = y.mutable_data_ptr();
    a.y_pitch = a.n;
    const size_t size = a.x_type == TSB_TYPE_I8 ? 0 : tsb_inner_prod_i8_workspace_bytes(&a);
    Tensor workspace;
    if (size) workspace = bytes((int64_t)size, x->device());
    if (tsb_inner_prod_i8(&a, size ? workspace.mutable_data_ptr() : nullptr, size, stream_of(device)) != TSB_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// group_norm(x, groups, gamma, beta, eps, activation, leaky, out_dtype, requant_scales) -> y
PyObject *group_norm(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    const Tensor *x = count == 9 ? tensor(args[0], -1) : nullptr;
    tsb_group_norm_desc d = {};
    if (!x || x->dim() < 3 || x->numel() < 1 || !x->is_contiguous() || !type_of(x->scalar_type(), &d.x_type)) Py_RETURN_NONE;
    const int device = x->get_device();
    d.n = x->size(0);
    d.channels = x->size(-1);
    d.pixels = x->numel() / (d.n * d.channels);
    d.x_pixel_stride = d.y_pixel_stride = d.channels;
    d.x_image_stride = d.y_image_stride = d.pixels * d.channels;
    if (!vector(args[2], d.channels, device, &d.gamma) || !vector(args[3], d.channels, device, &d.beta)) Py_RETURN_NONE;
    at::ScalarType out = x->scalar_type();
    if (args[7] != Py_None) {
        if (!THPDtype_Check(args[7])) Py_RETURN_NONE;
        out = reinterpret_cast<THPDtype *>(args[7])->scalar_type;
    }
    float scales[TSB_MAX_REQUANT_SCALES];
    int64_t channels = d.channels;
    if (out == at::kChar) {
        if (!PyList_Check(args[8]) || PyList_GET_SIZE(args[8]) < 1 || PyList_GET_SIZE(args[8]) > TSB_MAX_REQUANT_SCALES) Py_RETURN_NONE;
        d.n_requant_scales = (int)PyList_GET_SIZE(args[8]);
        for (int i = 0; i < d.n_requant_scales; ++i) scales[i] = (float)PyFloat_AsDouble(PyList_GET_ITEM(args[8], i));
        d.requant_scales_host = scales;
        d.y_type = TSB_TYPE_I8;
        channels = tsb_padded_channels((int)d.channels);
    } else {
        if (out != x->scalar_type() || args[8] != Py_None) Py_RETURN_NONE;
        d.y_type = d.x_type;
    }
    d.groups = PyLong_AsLongLong(args[1]);
    d.eps = PyFloat_AsDouble(args[4]);
    d.activation = int_of(args[5]);
    d.leaky_scale = (float)PyFloat_AsDouble(args[6]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const Tensor y = dense(*x, channels, out);
    d.x = x->const_data_ptr();
    d.y = y.mutable_data_ptr();
    const size_t size = tsb_group_norm_workspace_bytes(&d);
    Tensor workspace;
    if (size) workspace = bytes((int64_t)size, x->device());
    if (tsb_group_norm_nhwc(&d, size ? workspace.mutable_data_ptr() : nullptr, size, stream_of(device)) != TSB_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"quantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(quantize_rows)), METH_FASTCALL, nullptr},
    {"inner_prod", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(inner_prod)), METH_FASTCALL, nullptr},
    {"group_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(group_norm)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", "The ordinary calls of the int8 layers.", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&kModule); }
