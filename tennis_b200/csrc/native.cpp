// The ordinary calls of ops.quantize_rows, inner_prod_quantized, group_norm_nhwc, (de)quantize_rows_mxfp4, inner_prod_mxfp4 and rms_norm, from Python
// straight to the C ABI: tensors on the current device and stream, rows and images that lie one after the other, outputs that are allocated.  A kernel of these can be done in
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

#include <array>
#include <utility>

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

// ---- 4 bits
// (a PyTorch without these types: bytes, as in ops.py)
#if TSB_TORCH_FP4
constexpr at::ScalarType kFp4 = at::ScalarType::Float4_e2m1fn_x2;
#else
constexpr at::ScalarType kFp4 = at::kByte;
#endif
#if TSB_TORCH_E8M0
constexpr at::ScalarType kE8m0 = at::ScalarType::Float8_e8m0fnu;
#else
constexpr at::ScalarType kE8m0 = at::kByte;
#endif
int64_t row_bytes(int64_t k) { return (k + 31) / 32 * 16; }

// Values and their scales, which are of use together alone, in one allocation (a second one takes 0.7 us of a call of 5): a tensor of `type` of `sizes`, `step` elements between rows of
// its last dimension's, and one of `scale_type` behind it.
struct Pair {
    Tensor values, scales;
};
Tensor view_of(const Tensor &room, at::ScalarType type, at::IntArrayRef sizes, at::IntArrayRef strides, int64_t offset) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(room.storage()), room.key_set(), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(offset);
    t.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides);
    return t;
}
Pair pair_of(at::ScalarType type, at::IntArrayRef sizes, int64_t step, at::ScalarType scale_type, at::IntArrayRef scale_sizes, c10::Device device) {
    c10::SmallVector<int64_t, 6> strides(sizes.size()), scale_strides(scale_sizes.size());
    int64_t rows = 1, count = 1;
    for (size_t i = sizes.size(); i-- > 0;) {
        strides[i] = i + 1 == sizes.size() ? 1 : step * rows;
        if (i + 1 < sizes.size()) rows *= sizes[i] > 0 ? sizes[i] : 1;
    }
    for (size_t i = scale_sizes.size(); i-- > 0;) {
        scale_strides[i] = count;
        count *= scale_sizes[i] > 0 ? scale_sizes[i] : 1;
    }
    const int64_t element = (int64_t)c10::elementSize(scale_type), at = (rows * step + 511) / 512 * 512;      // (values are bytes)
    const Tensor all = bytes(at + count * element, device);
    return {view_of(all, type, sizes, strides, 0), view_of(all, scale_type, scale_sizes, scale_strides, at / element)};
}
// The sizes of the scales of m rows of k values
std::array<int64_t, 5> scale_sizes(int64_t m, int64_t k) { return {(m + 127) / 128, (k + 127) / 128, 32, 4, 4}; }

// A 4-bit matrix's scales; false for anything else
bool scales_of(PyObject *o, int64_t m, int64_t k, int device, const void **at) {
    const Tensor *t = tensor(o, device);
    if (!t || (t->scalar_type() != kE8m0 && t->scalar_type() != at::kByte) || t->dim() != 5 || t->size(0) != (m + 127) / 128 || t->size(1) != (k + 127) / 128 || t->size(2) != 32 ||
        t->size(3) != 4 || t->size(4) != 4 || !t->is_contiguous())
        return false;
    *at = t->const_data_ptr();
    return true;
}
bool is_fp4(const Tensor &t) { return (t.scalar_type() == kFp4 || t.scalar_type() == at::kByte) && t.dim() >= 1 && t.size(-1) > 0 && t.size(-1) % 16 == 0; }

PyObject *tuple_of(std::initializer_list<Tensor> all) {
    PyObject *t = PyTuple_New((Py_ssize_t)all.size());
    if (!t) return nullptr;
    Py_ssize_t i = 0;
    for (const Tensor &v : all) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(v));
    return t;
}

// quantize_rows_mxfp4(x) -> (q, scales)
PyObject *quantize_rows_mxfp4(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    const Tensor *x = count == 1 ? tensor(args[0], -1) : nullptr;
    int type;
    int64_t rows, pitch;
    if (!x || !type_of(x->scalar_type(), &type) || !rows_of(*x, &rows, &pitch)) Py_RETURN_NONE;
    const int64_t k = x->size(-1);
    const Pair y = pair_of(kFp4, sizes_with(*x, row_bytes(k)), row_bytes(k), kE8m0, scale_sizes(rows, k), x->device());
    if (tsb_quantize_rows_mxfp4(x->const_data_ptr(), type, pitch, y.values.mutable_data_ptr(), row_bytes(k), y.scales.mutable_data_ptr(), rows, k, stream_of(x->get_device())) != TSB_OK)
        Py_RETURN_NONE;
    return tuple_of({y.values, y.scales});
    END_HANDLE_TH_ERRORS
}

// dequantize_rows_mxfp4(q, scales, k, dtype) -> y
PyObject *dequantize_rows_mxfp4(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    const Tensor *q = count == 4 ? tensor(args[0], -1) : nullptr;
    int type;
    int64_t rows, pitch;
    const void *scales;
    if (!q || !is_fp4(*q) || !rows_of(*q, &rows, &pitch) || !THPDtype_Check(args[3])) Py_RETURN_NONE;
    const at::ScalarType out = reinterpret_cast<THPDtype *>(args[3])->scalar_type;
    const int64_t k = args[2] == Py_None ? 2 * q->size(-1) : PyLong_AsLongLong(args[2]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (k < 1 || row_bytes(k) != q->size(-1) || !type_of(out, &type) || !scales_of(args[1], rows, k, q->get_device(), &scales)) Py_RETURN_NONE;
    const Tensor y = dense(*q, k, out);
    if (tsb_dequantize_rows_mxfp4(q->const_data_ptr(), pitch, scales, y.mutable_data_ptr(), type, k, rows, k, stream_of(q->get_device())) != TSB_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// inner_prod_mxfp4(x, x_scales, w, w_scales, bias, residual, activation, leaky, out_dtype, residual_after) -> y
PyObject *inner_prod_mxfp4(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    const Tensor *x = count == 10 ? tensor(args[0], -1) : nullptr;
    if (!x) Py_RETURN_NONE;
    const int device = x->get_device();
    const Tensor *w = tensor(args[2], device);
    tsb_inner_prod_mxfp4_args a = {};
    if (!w || !is_fp4(*w) || w->dim() != 2 || w->stride(1) != 1 || !rows_of(*x, &a.m, &a.x_pitch)) Py_RETURN_NONE;
    a.n = w->size(0);
    a.k = 2 * w->size(1);
    if (a.m < 1 || a.n < 1) Py_RETURN_NONE;
    a.w_pitch = w->stride(0);
    at::ScalarType out = at::kFloat;
    if (args[1] == Py_None) {
        if (!type_of(x->scalar_type(), &a.x_type) || row_bytes(x->size(-1)) != w->size(1)) Py_RETURN_NONE;
        a.k = x->size(-1);
        out = x->scalar_type();
    } else {
        if (!is_fp4(*x) || x->size(-1) != w->size(1) || !scales_of(args[1], a.m, a.k, device, &a.x_scales)) Py_RETURN_NONE;
        a.x_type = TSB_TYPE_MXFP4;
    }
    if (args[8] != Py_None) {
        if (!THPDtype_Check(args[8])) Py_RETURN_NONE;
        out = reinterpret_cast<THPDtype *>(args[8])->scalar_type;
    }
    if (!type_of(out, &a.y_type) || !scales_of(args[3], a.n, a.k, device, &a.w_scales) || !vector(args[4], a.n, device, &a.bias)) Py_RETURN_NONE;
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
    a.w = w->const_data_ptr();
    const Tensor y = dense(*x, a.n, out);
    a.y = y.mutable_data_ptr();
    a.y_pitch = a.n;
    const size_t size = a.x_type == TSB_TYPE_MXFP4 ? 0 : tsb_inner_prod_mxfp4_workspace_bytes(&a);
    Tensor workspace;
    if (size) workspace = bytes((int64_t)size, x->device());
    if (tsb_inner_prod_mxfp4(&a, size ? workspace.mutable_data_ptr() : nullptr, size, stream_of(device)) != TSB_OK) Py_RETURN_NONE;
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// rms_norm(x, gamma, residual, eps, out_dtype) -> y, or (q, scales); with a residual the sum as one result more
PyObject *rms_norm(PyObject *, PyObject *const *args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    const Tensor *x = count == 5 ? tensor(args[0], -1) : nullptr;
    tsb_rms_norm_desc d = {};
    if (!x || !type_of(x->scalar_type(), &d.x_type) || !rows_of(*x, &d.rows, &d.x_pitch) || d.rows < 1) Py_RETURN_NONE;
    const int device = x->get_device();
    d.cols = x->size(-1);
    if (!vector(args[1], d.cols, device, &d.gamma)) Py_RETURN_NONE;
    Tensor sum;
    if (args[2] != Py_None) {
        const Tensor *r = tensor(args[2], device);
        int64_t rows;
        if (!r || r->scalar_type() != x->scalar_type() || r->sizes() != x->sizes() || !rows_of(*r, &rows, &d.residual_pitch) || rows != d.rows) Py_RETURN_NONE;
        d.residual = r->const_data_ptr();
    }
    d.eps = PyFloat_AsDouble(args[3]);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    at::ScalarType out = x->scalar_type();
    if (args[4] != Py_None) {
        if (!THPDtype_Check(args[4])) Py_RETURN_NONE;
        out = reinterpret_cast<THPDtype *>(args[4])->scalar_type;
    }
    Tensor y, scales;
    if (out == x->scalar_type()) {
        d.y_type = d.x_type;
        d.y_pitch = d.cols;
        y = dense(*x, d.cols, out);
    } else if (out == at::kChar || out == kFp4) {
        const bool int8 = out == at::kChar;
        d.y_type = int8 ? TSB_TYPE_I8 : TSB_TYPE_MXFP4;
        d.y_pitch = int8 ? (d.cols + 15) / 16 * 16 : row_bytes(d.cols);
        const std::array<int64_t, 5> tiles = scale_sizes(d.rows, d.cols);
        Pair made = pair_of(out, sizes_with(*x, int8 ? d.cols : d.y_pitch), d.y_pitch, int8 ? at::kFloat : kE8m0, int8 ? x->sizes().slice(0, x->dim() - 1) : at::IntArrayRef(tiles), x->device());
        y = std::move(made.values);
        scales = std::move(made.scales);
    } else {
        Py_RETURN_NONE;
    }
    if (d.residual) {
        sum = dense(*x, d.cols, x->scalar_type());
        d.sum = sum.mutable_data_ptr();
        d.sum_pitch = d.cols;
    }
    d.x = x->const_data_ptr();
    d.y = y.mutable_data_ptr();
    d.scales = scales.defined() ? scales.mutable_data_ptr() : nullptr;
    if (tsb_rms_norm(&d, stream_of(device)) != TSB_OK) Py_RETURN_NONE;
    if (scales.defined()) return d.residual ? tuple_of({y, scales, sum}) : tuple_of({y, scales});
    return d.residual ? tuple_of({y, sum}) : THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"quantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(quantize_rows)), METH_FASTCALL, nullptr},
    {"inner_prod", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(inner_prod)), METH_FASTCALL, nullptr},
    {"group_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(group_norm)), METH_FASTCALL, nullptr},
    {"quantize_rows_mxfp4", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(quantize_rows_mxfp4)), METH_FASTCALL, nullptr},
    {"dequantize_rows_mxfp4", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(dequantize_rows_mxfp4)), METH_FASTCALL, nullptr},
    {"inner_prod_mxfp4", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(inner_prod_mxfp4)), METH_FASTCALL, nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(rms_norm)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", "The ordinary calls of the int8 and 4-bit layers.", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&kModule); }
