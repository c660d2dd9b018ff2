"""Python mirror of the two TenniS operators on the path, over the C ABI.

The shipping host side is the C++ plugin in tennis_b200/plugin/ (TS_REGISTER_OPERATOR on device "gpu"); this
module states the same interface for Python callers and for the parity tests: same operator names, same
attribute names and meaning, the same checks in ``init`` / ``infer`` and the same error texts as

* ts::base::Quantize          src/backend/base/base_quantize.cpp:12-49
* ts::base::Conv2DQuantized   src/backend/base/base_conv2d_quantized.cpp:13-219
* ts::Operator                src/runtime/operator.cpp:22-128 (fields, set, check_params)

Tensors are torch CUDA tensors used as device buffers; all arithmetic happens in libtennis_b200.so.
"""
import ctypes
import operator

import numpy as np
import torch

from . import _lib
from ._lib import (ACT_GELU, ACT_LEAKY_RELU, ACT_NONE, ACT_RELU, ACT_SILU, KERNEL_AUTO, KERNEL_DIRECT, KERNEL_TCGEN05, LAYOUT_NCHW,
                   LAYOUT_NHWC_PAD, LAYOUT_STAGED, ConvDesc, ConvEpilogue, TsbError, check, float_array)

REQUIRED, OPTIONAL = "required", "optional"


class EjectionException(RuntimeError):
    """What TS_LOG_ERROR << ... << eject raises in the reference (include/utils/log.h:162-166)."""


# The raw handle of the current stream.  A small convolution takes the GPU 4 us and the driver 3 us to launch;
# torch.cuda.current_stream() builds a Stream object for 3 us more, these two calls take 0.2 us.
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_current_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr(stream=None):
    if stream is None:
        return _current_raw_stream(_current_device())
    return stream.cuda_stream


def _ptr(t):
    return t.data_ptr() if t is not None else None


def padded_channels(c):
    return _lib.load().tsb_padded_channels(int(c))


def conv_out_dim(x, pad_lo, pad_hi, k, stride, dilation):
    """include/backend/common_function.h:30-40: integer division truncating toward zero."""
    num = x + pad_lo + pad_hi - (dilation * (k - 1) + 1)
    q = abs(num) // stride
    return (q if num >= 0 else -q) + 1


class Operator:
    """Field handling of ts::Operator (src/runtime/operator.cpp:22-128)."""

    op = "operator"

    def __init__(self):
        self._fields = {}
        self._params = {}

    def field(self, name, attr, default=None):
        self._fields[name] = attr
        if default is not None:
            self._params[name] = default

    def has(self, name):
        return name in self._params

    def get(self, name):
        if name not in self._params:
            raise EjectionException('Unidentified param "%s"' % name)
        return self._params[name]

    def set(self, name, value):
        if name not in self._fields:
            raise EjectionException('Unidentified param "%s", did you mean "%s"' % (name, self._closest(name)))
        self._params[name] = value

    def _closest(self, name):
        import difflib
        m = difflib.get_close_matches(name, list(self._fields), n=1, cutoff=0.0)
        return m[0] if m else ""

    def init(self):
        missing = [f for f, a in self._fields.items() if a == REQUIRED and f not in self._params]
        if missing:
            raise EjectionException("Operator %s has unsatisfied fields: %s" % (self.op, ", ".join(missing)))


def _auto_check(cond, text):
    if not cond:
        raise EjectionException("Check failed: (%s)." % text)


class Quantize(Operator):
    """Operator "quantize" on the GPU: fp32 -> int8, attribute ``quantize_scale`` (one scale per sample)."""

    op = "quantize"

    def __init__(self):
        super().__init__()
        self.field("quantize_scale", REQUIRED)
        self.scales = None
        self._array = self._array_of = None

    def init(self):
        super().init()
        self.scales = [float(v) for v in np.asarray(self.get("quantize_scale"), dtype=np.float32).reshape(-1)]
        self._scale_array()

    def infer(self, inputs):
        _auto_check(len(inputs) == 1, "stack.size() == 1")
        x = inputs[0]
        _auto_check(len(self.scales) == x.shape[0], "m_quantize_scales.size() == x_tensor.sizes()[0]")
        return [("int8", tuple(x.shape))]

    def _scale_array(self):
        """The scales as the library takes them, laid out again when they are others than last time."""
        if self.scales != self._array_of:
            self._array, self._array_of = float_array(self.scales), list(self.scales)
        return self._array

    def run(self, inputs, stream=None):
        self.infer(inputs)
        x = inputs[0]
        if x.dtype not in (torch.float32, torch.float64):   # the reference's dispatch: src/kernels/cpu/quantize.cpp:130-141
            raise EjectionException("%s not support this data type: %s" % (self.op, str(x.dtype).replace("torch.", "")))
        x = x.contiguous()
        y = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        lib = _lib.load()
        fn = lib.tsb_quantize_f32_i8 if x.dtype == torch.float32 else lib.tsb_quantize_f64_i8
        scales = self._scale_array()
        status = fn(x.data_ptr(), y.data_ptr(), x.numel(), scales, len(scales), _stream_ptr(stream))
        if status:
            check(status)
        return y


class Call:
    """A library call with every argument but the stream bound, and what those arguments point to kept alive: ``tensors``, and
    ``keep`` for the rest.

    ``sources``: (container, key, object) of the objects among them that a program could replace, for those who call again and again
    (BoundCalls)."""

    __slots__ = ("fn", "args", "keep", "tensors", "sources")

    def __init__(self, fn, args, keep, tensors, sources=()):
        self.fn, self.args, self.keep, self.tensors, self.sources = fn, args, keep, tensors, sources

    def __call__(self, stream_ptr):
        status = self.fn(*self.args, stream_ptr)
        if status:
            check(status)


class BoundCalls:
    """Calls that are made one after the other as long as they would be bound the same today: the containers that their objects came
    from still hold them, and every tensor still lies where it did.

    The check (some 0.7 us a call) goes ahead of the calls in groups, so that the GPU, which is busy with a call for longer than
    the host, does not wait for it."""

    GROUP = 6

    def __init__(self, calls):
        self.groups = []
        for i in range(0, len(calls), self.GROUP):
            group = calls[i:i + self.GROUP]
            containers, keys, held = zip(*[s for c in group for s in c.sources])
            where = [t.data_ptr for c in group for t in c.tensors if t is not None]
            self.groups.append((group, containers, keys, held, where, [f() for f in where]))

    def run(self, stream_ptr):
        """Makes the calls; False, with some of them made, once one would be bound differently."""
        for group, containers, keys, held, where, at in self.groups:
            try:
                if not all(map(operator.is_, map(operator.getitem, containers, keys), held)) or [f() for f in where] != at:
                    return False
            except (KeyError, IndexError):
                return False
            for call in group:
                status = call.fn(*call.args, stream_ptr)
                if status:
                    check(status)
        return True


def _scales_of(values):
    return values if isinstance(values, ctypes.Array) else float_array(values)


def _epilogue(dq, bias, residual, activation, leaky, out_f32, out_f32_layout, out_i8, out_i8_layout, requant_scales, out_acc,
              residual_after_activation):
    """The ConvEpilogue of these tensors (it refers to requant_scales, a ctypes array, which the caller keeps)."""
    e = ConvEpilogue()
    e.dequantize_scales = dq.data_ptr()
    e.activation = int(activation)
    e.leaky_scale = leaky
    if residual_after_activation:
        e.residual_after_activation = 1
    if bias is not None:
        e.bias = bias.data_ptr()
    if residual is not None:
        e.residual = residual.data_ptr()
    if out_f32 is not None:
        e.out_f32 = out_f32.data_ptr()
    e.out_f32_layout = out_f32_layout
    if out_i8 is not None:
        e.out_i8 = out_i8.data_ptr()
    e.out_i8_layout = out_i8_layout
    if requant_scales is not None:
        e.requant_scales_host = requant_scales
        e.n_requant_scales = len(requant_scales)
    if out_acc is not None:
        e.out_acc = out_acc.data_ptr()
    return e


class ConvPlan:
    """Owner of a tsb_conv_plan, its workspace and the device copies of the per-channel vectors."""

    def __init__(self, xshape, wshape, pad, stride, dilation, padding_value=0.0, kernel=KERNEL_AUTO, device="cuda",
                 mma_orientation=0, raw_row_mode=0, patch_mode=0):
        lib = self._lib = _lib.load()
        d = ConvDesc()
        d.mma_orientation, d.raw_row_mode, d.patch_mode = int(mma_orientation), int(raw_row_mode), int(patch_mode)
        d.n, d.c, d.h, d.w = [int(v) for v in xshape]
        d.o, _, d.kh, d.kw = [int(v) for v in wshape]
        d.pad_top, d.pad_bottom, d.pad_left, d.pad_right = [int(v) for v in pad]
        d.stride_h, d.stride_w = [int(v) for v in stride]
        d.dilation_h, d.dilation_w = [int(v) for v in dilation]
        d.padding_value = float(padding_value)
        d.kernel = int(kernel)
        self.desc = d
        handle = ctypes.c_void_p()
        check(lib.tsb_conv2d_i8_plan_create(ctypes.byref(d), ctypes.byref(handle)))
        self.handle = handle
        shape = (ctypes.c_int * 4)()
        check(lib.tsb_conv2d_i8_output_shape(handle, shape))
        self.out_shape = tuple(shape)
        self.kernel = lib.tsb_conv2d_i8_kernel(handle)
        self.ws_bytes = lib.tsb_conv2d_i8_workspace_bytes(handle)
        self.workspace = torch.empty(self.ws_bytes, dtype=torch.uint8, device=device)
        self.weights = None
        self.device = device

    def __del__(self):
        try:
            if self.handle:
                _lib.load().tsb_conv2d_i8_plan_destroy(self.handle)
                self.handle = None
        except Exception:
            pass

    def set_weights(self, w, stream=None):
        assert w.dtype == torch.int8 and w.is_cuda
        self.weights = w.contiguous()  # the direct kernel reads this tensor at run time
        check(_lib.load().tsb_conv2d_i8_set_weights(self.handle, _ptr(self.weights), _ptr(self.workspace), self.ws_bytes,
                                                    _stream_ptr(stream)))

    def quantize_input(self, x_f32, scales, stream=None):
        """fp32 NCHW -> the plan's staged int8 input; run() is then called with x=None, x_layout=LAYOUT_STAGED."""
        arr = scales if not isinstance(scales, (list, tuple)) else float_array(scales)
        status = self._lib.tsb_conv2d_i8_quantize_input(self.handle, x_f32.data_ptr(), arr, len(arr), self.workspace.data_ptr(),
                                                        self.ws_bytes, _stream_ptr(stream))
        if status:
            check(status)

    def run(self, x, x_layout, dq, bias=None, residual=None, activation=ACT_NONE, leaky=0.0, out_f32=None,
            out_f32_layout=LAYOUT_NCHW, out_i8=None, out_i8_layout=LAYOUT_NCHW, requant_scales=None, out_acc=None,
            stream=None, residual_after_activation=False):
        rq = None if requant_scales is None else _scales_of(requant_scales)
        e = _epilogue(dq, bias, residual, activation, leaky, out_f32, out_f32_layout, out_i8, out_i8_layout, rq, out_acc,
                      residual_after_activation)
        status = self._lib.tsb_conv2d_i8_run(self.handle, None if x is None else x.data_ptr(), x_layout, e, self.workspace.data_ptr(),
                                             self.ws_bytes, _stream_ptr(stream))
        if status:
            check(status)

    def bind_run(self, x, x_layout, dq, bias=None, residual=None, activation=ACT_NONE, leaky=0.0, out_f32=None,
                 out_f32_layout=LAYOUT_NCHW, out_i8=None, out_i8_layout=LAYOUT_NCHW, requant_scales=None,
                 residual_after_activation=False):
        """run() with these tensors as a Call, for programs that launch the same layer on the same buffers again and again."""
        rq = None if requant_scales is None else _scales_of(requant_scales)
        e = _epilogue(dq, bias, residual, activation, leaky, out_f32, out_f32_layout, out_i8, out_i8_layout, rq, None,
                      residual_after_activation)
        args = (self.handle, _ptr(x), int(x_layout), ctypes.byref(e), self.workspace.data_ptr(), self.ws_bytes)
        return Call(self._lib.tsb_conv2d_i8_run, args, (self, e, rq), (self.workspace, x, dq, bias, residual, out_f32, out_i8))

    def bind_projected(self, x, shortcut, x_shortcut, dq, shortcut_dq, bias=None, shortcut_bias=None, activation=ACT_NONE,
                       leaky=0.0, out_f32=None, out_i8=None, requant_scales=None, residual_after_activation=False,
                       tile_channels=0):
        """run_projected() with these tensors as a Call."""
        rq = None if requant_scales is None else _scales_of(requant_scales)
        e = _epilogue(dq, bias, None, activation, leaky, out_f32, LAYOUT_NHWC_PAD, out_i8, LAYOUT_NHWC_PAD, rq, None,
                      residual_after_activation)
        args = (self.handle, _ptr(x), shortcut.handle, _ptr(x_shortcut), _ptr(shortcut_dq), _ptr(shortcut_bias), ctypes.byref(e),
                int(tile_channels), self.workspace.data_ptr(), self.ws_bytes)
        return Call(self._lib.tsb_conv2d_i8_run_projected, args, (self, shortcut, e, rq),
                    (self.workspace, shortcut.workspace, x, x_shortcut, dq, shortcut_dq, bias, shortcut_bias, out_f32, out_i8))

    def run_projected(self, x, shortcut, x_shortcut, dq, shortcut_dq, bias=None, shortcut_bias=None, activation=ACT_NONE,
                      leaky=0.0, out_f32=None, out_i8=None, requant_scales=None, stream=None,
                      residual_after_activation=False, tile_channels=0):
        """This convolution with the 1x1 projection `shortcut` (another ConvPlan, its weights set) as its residual, in
        one launch (tsb_conv2d_i8_run_projected): NHWC_PAD int8 inputs, pixel-major fp32 / NHWC_PAD int8 outputs."""
        self.bind_projected(x, shortcut, x_shortcut, dq, shortcut_dq, bias, shortcut_bias, activation, leaky, out_f32, out_i8,
                            requant_scales, residual_after_activation, tile_channels)(_stream_ptr(stream))

    def bind_concat(self, x, first, x_first, dq, bias=None, activation=ACT_NONE, leaky=0.0, out_f32=None, out_i8=None,
                    requant_scales=None, tile_channels=0):
        """run_concat() with these tensors as a Call."""
        rq = None if requant_scales is None else _scales_of(requant_scales)
        e = _epilogue(dq, bias, None, activation, leaky, out_f32, LAYOUT_NHWC_PAD, out_i8, LAYOUT_NHWC_PAD, rq, None, False)
        args = (self.handle, _ptr(x), first.handle, _ptr(x_first), ctypes.byref(e), int(tile_channels), self.workspace.data_ptr(),
                self.ws_bytes)
        return Call(self._lib.tsb_conv2d_i8_run_concat, args, (self, first, e, rq),
                    (self.workspace, first.workspace, x, x_first, dq, bias, out_f32, out_i8))

    def run_concat(self, x, first, x_first, dq, bias=None, activation=ACT_NONE, leaky=0.0, out_f32=None, out_i8=None,
                   requant_scales=None, stream=None, tile_channels=0):
        """The convolution over concat(x_first, x) along channels in one launch (tsb_conv2d_i8_run_concat): `first` holds the
        weight columns of the leading channels (a 1x1 plan), this plan the rest; NHWC_PAD int8 inputs quantized with the
        same scales, pixel-major fp32 / NHWC_PAD int8 outputs."""
        self.bind_concat(x, first, x_first, dq, bias, activation, leaky, out_f32, out_i8, requant_scales,
                         tile_channels)(_stream_ptr(stream))

    def status(self, stream=None):
        check(_lib.load().tsb_conv2d_i8_status(self.handle, _ptr(self.workspace), _stream_ptr(stream)))

    def describe(self):
        buf = ctypes.create_string_buffer(512)
        n = _lib.load().tsb_conv2d_i8_plan_describe(self.handle, buf, len(buf))
        if n < 0:
            check(n)
        return buf.value.decode()


def _to_string(arr):
    return "[" + ", ".join(str(int(v)) for v in arr) + "]"


def _writes(t):
    """How often a tensor's memory was written so far; None where PyTorch does not count (inference tensors)."""
    return None if t.is_inference() else t._version


class Conv2DQuantized(Operator):
    """Operator "conv2d_quantized" on the GPU: int8 NCHW x int8 OIHW -> fp32 NCHW."""

    op = "conv2d_quantized"

    def __init__(self, kernel=KERNEL_AUTO):
        super().__init__()
        self.field("format", REQUIRED)
        self.field("padding", REQUIRED)
        self.field("padding_value", OPTIONAL, 0.0)
        self.field("stride", REQUIRED)
        self.field("dilation", OPTIONAL)
        self.field("dialations", OPTIONAL)
        self.field("dequantize_scales", REQUIRED)
        self._kernel = kernel
        # plans by what they were made from, this operator's own configuration included: attributes that are set again do not
        # meet a plan of the ones before them, and a plan that a captured graph refers to stays where it is
        self._plans = {}
        self._dq_dev = {}
        self._config = None

    def init(self):
        self._config = object()           # no plan is of a configuration that fails a check below
        super().init()
        fmt = self.get("format")
        padding = np.asarray(self.get("padding")).astype(np.int32)
        self.padding_value = float(np.asarray(self.get("padding_value")).reshape(-1)[0])
        stride = np.asarray(self.get("stride")).astype(np.int32)
        dilation = None
        if self.has("dilation"):
            dilation = np.asarray(self.get("dilation")).astype(np.int32)
        elif self.has("dialations"):
            dilation = np.asarray(self.get("dialations")).astype(np.int32)
        if dilation is None or dilation.size == 0:
            raise EjectionException("%s must set dilation or dialations" % self.op)
        _auto_check(padding.shape == (4, 2), "padding_tensor.has_shape({ 4, 2 })")
        _auto_check(stride.shape == (4,), "stride_tensor.has_shape({ 4, })")
        _auto_check(dilation.shape == (4,), "dilation_tensor.has_shape({ 4, })")
        if fmt not in ("NCHW", "NHWC"):
            raise EjectionException("%s do not support format: %s" % (self.op, fmt))
        self.format = fmt
        p = padding.reshape(-1)
        if fmt == "NCHW":
            bad_p, bad_s, bad_d = p[:4].any(), (stride[:2] != 1).any(), (dilation[:2] != 1).any()
        else:
            bad_p = p[[0, 1, 6, 7]].any()
            bad_s, bad_d = (stride[[0, 3]] != 1).any(), (dilation[[0, 3]] != 1).any()
        if bad_p:
            raise EjectionException("%s do not support padding: %s" % (self.op, _to_string(p)))
        if bad_s:
            raise EjectionException("%s do not support stride: %s" % (self.op, _to_string(stride)))
        if bad_d:
            raise EjectionException("%s do not support dialations: %s" % (self.op, _to_string(dilation)))
        self.padding4x2, self.stride4, self.dilation4 = p, stride, dilation
        self.dequantize_scales = np.asarray(self.get("dequantize_scales"), dtype=np.float32).reshape(-1)
        self._config = (fmt, p.tobytes(), stride.tobytes(), dilation.tobytes(), self.padding_value, self.dequantize_scales.tobytes())

    def _geometry(self):
        p, s, d = self.padding4x2, self.stride4, self.dilation4
        if self.format == "NCHW":
            return (p[4], p[5], p[6], p[7]), (s[2], s[3]), (d[2], d[3])
        return (p[2], p[3], p[4], p[5]), (s[1], s[2]), (d[1], d[2])

    def infer(self, inputs):
        _auto_check(len(inputs) == 2, "stack.size() == 2")
        x, w = inputs
        _auto_check(x.dim() == 4, "x_tensor.dims() == 4")
        _auto_check(w.dim() == 4, "w_tensor.dims() == 4")
        _auto_check(x.dtype == w.dtype, "x_tensor.dtype() == w_tensor.dtype()")
        _auto_check(w.shape[1] == x.shape[1], "w_tensor.size(1) == x_tensor.size(1)")
        _auto_check(x.dtype == torch.int8, "x_tensor.dtype() == INT8")
        _auto_check(len(self.dequantize_scales) == w.shape[0], "m_dequantize_scales.size() == w_tensor.size(0)")
        pad, stride, dil = self._geometry()
        if self.format == "NCHW":
            H, W, KH, KW = x.shape[2], x.shape[3], w.shape[2], w.shape[3]
        else:
            H, W, KH, KW = x.shape[1], x.shape[2], w.shape[1], w.shape[2]
        OH = conv_out_dim(H, pad[0], pad[1], KH, stride[0], dil[0])
        OW = conv_out_dim(W, pad[2], pad[3], KW, stride[1], dil[1])
        if self.format == "NCHW":
            return [("float32", (x.shape[0], w.shape[0], OH, OW))]
        return [("float32", (x.shape[0], OH, OW, w.shape[0]))]

    def run(self, inputs, stream=None, out_acc=None):
        """The weights are packed when they are new and when they were written since, as far as PyTorch counts writes (a write
        through ``.data`` or a raw pointer is not counted)."""
        kept = None
        if len(inputs) == 2:
            x, w = inputs
            # a plan was made for this configuration, these shapes and types only after they had passed every check
            key = (self._config, x.shape, w.shape, w.stride(), w.data_ptr(), x.dtype, w.dtype, x.device)
            kept = self._plans.get(key)
        if kept is None:
            self.infer(inputs)
            if self.format != "NCHW":
                raise EjectionException("Conv2D_quantized only support NCHW")  # conv2d_quantized_core.cpp:131-133
            pad, strides, dil = self._geometry()
            try:
                plan = ConvPlan(x.shape, w.shape, pad, strides, dil, self.padding_value, self._kernel, x.device)
            except TsbError as e:
                raise EjectionException(e.message)
            plan.set_weights(w, stream)
            # (the tensor is kept, so that its address stays its own)
            self._plans[key] = [plan, w, _writes(w)]
        else:
            plan = kept[0]
            writes = _writes(w)
            if writes is None or writes != kept[2]:
                plan.set_weights(w, stream)
                kept[2] = writes
        dq = self._dq_dev.get((self._config, x.device))
        if dq is None:
            dq = self._dq_dev[self._config, x.device] = torch.from_numpy(self.dequantize_scales.copy()).to(x.device)
        x = x.contiguous()
        out = torch.empty(plan.out_shape, dtype=torch.float32, device=x.device)
        plan.run(x, LAYOUT_NCHW, dq, out_f32=out, out_acc=out_acc, stream=stream)
        return out


def add_bias(x, bias, stream=None):
    """Operator "add_bias", format NCHW (src/kernels/gpu/add_bias.cu:19-26)."""
    x = x.contiguous()
    y = torch.empty_like(x)
    n, c = x.shape[0], x.shape[1]
    check(_lib.load().tsb_add_bias_f32_nchw(_ptr(x), _ptr(y), n, c, x.numel() // (n * c), _ptr(bias), _stream_ptr(stream)))
    return y


def relu(x, stream=None):
    x = x.contiguous()
    y = torch.empty_like(x)
    check(_lib.load().tsb_relu_f32(_ptr(x), _ptr(y), x.numel(), _stream_ptr(stream)))
    return y


def leaky_relu(x, scale, stream=None):
    x = x.contiguous()
    y = torch.empty_like(x)
    check(_lib.load().tsb_leaky_relu_f32(_ptr(x), _ptr(y), x.numel(), float(scale), _stream_ptr(stream)))
    return y


def quantize_nchw_to_nhwc(x, scales, stream=None):
    """fp32 NCHW -> int8 NHWC_PAD with the arithmetic of "quantize"."""
    x = x.contiguous()
    n, c, h, w = x.shape
    y = torch.empty((n, h, w, padded_channels(c)), dtype=torch.int8, device=x.device)
    check(_lib.load().tsb_quantize_f32_nchw_to_nhwc(_ptr(x), _ptr(y), n, c, h, w, float_array(scales), len(scales),
                                                    _stream_ptr(stream)))
    return y


def repack_nchw_to_nhwc(x, stream=None):
    x = x.contiguous()
    n, c, h, w = x.shape
    y = torch.empty((n, h, w, padded_channels(c)), dtype=torch.int8, device=x.device)
    check(_lib.load().tsb_repack_i8_nchw_to_nhwc(_ptr(x), _ptr(y), n, c, h, w, _stream_ptr(stream)))
    return y


def repack_nhwc_to_nchw(x, channels, stream=None):
    x = x.contiguous()
    n, h, w, _ = x.shape
    y = torch.empty((n, channels, h, w), dtype=torch.int8, device=x.device)
    check(_lib.load().tsb_repack_i8_nhwc_to_nchw(_ptr(x), _ptr(y), n, channels, h, w, _stream_ptr(stream)))
    return y


# ---- int8 layers with scales per token: quantize_rows, inner_prod_quantized, group_norm_nhwc --------------------------------
# These three work on the device that their tensors are on, on its current stream or on `stream`; what they allocate (outputs,
# workspace) belongs to that stream.  Memory of an input that another stream allocated is the caller's to keep until the work is done.
# Ordinary calls go through native.cpp (4 us a call), those on another stream or device too once it is made the current one; the Python below them is the
# general way: every layout, outputs of the caller's, and the texts of refusals.
_TYPE = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16, torch.int8: _lib.TYPE_I8}
_FLOATS = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}
_FLOAT_NAMES = "float32, float16 or bfloat16, not %s"
_int8, _float32 = torch.int8, torch.float32
_uint8 = torch.uint8
# (a PyTorch without the types of 4-bit values or their scales: their bytes, which are taken everywhere, in their place)
_mxfp4, _e8m0 = getattr(torch, "float4_e2m1fn_x2", _uint8), getattr(torch, "float8_e8m0fnu", _uint8)


_native = None


def _ordinary():
    """The calls of native.cpp: an operator's result where tensors, layouts and arguments are the ordinary ones, else None."""
    global _native
    _lib.load()
    try:
        from . import _native as module
    except ImportError as e:
        raise RuntimeError("tennis_b200: the module _native has not been built for this Python and PyTorch (python -c 'import __graft_entry__ as g; "
                           "g.build()' or make -C tennis_b200/csrc python): %s" % e)
    _native = module
    return module


def _refuse(text, *values):
    raise EjectionException("Check failed: (%s)." % (text % values if values else text))


def _elsewhere(call, x, stream, *args):
    """call(x, *args) with x's device and `stream` as the current ones."""
    if not x.is_cuda:
        _refuse("x.is_cuda")
    if stream is None:
        with torch.cuda.device(x.device):
            return call(x, *args)
    if stream.device != x.device:
        _refuse("stream.device == x.device")
    with torch.cuda.stream(stream):
        return call(x, *args)


def _rows_of(t):
    """t [..., k] as rows: a tensor [m, k] whose values of a row are neighbours (a copy only where no view is)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _rows_to(out):
    """The rows of an output as a view."""
    if out.dim() == 2:
        return out
    try:
        return out.view(-1, out.shape[-1])
    except RuntimeError:
        _refuse("out: its rows lie a fixed step apart")


def _check_vector(t, size, device, name):
    if t.dtype is not _float32 or t.numel() != size or t.get_device() != device or not t.is_contiguous():
        _refuse("%s: %d contiguous float32 values on x's device", name, size)


def quantize_rows(x, out=None, scales=None, stream=None):
    """int8 values of x [..., k] (fp32, fp16 or bf16) with a scale for each row, taken from the row: (q, scales) with
    ``scales[..., None] * q`` standing for x (tsb_quantize_rows_i8 says how it rounds, and what rows of zeros, NaN and infinities give).

    q is [..., k]; its rows start a multiple of 16 bytes apart, the way inner_prod_quantized reads them fastest.  The rows of x are
    tokens of an activation, or output channels of a weight tensor.  ``out`` (int8, x's shape, values of a row next to each other)
    and ``scales`` take the results where they are given."""
    if out is None and scales is None and stream is None:
        done = (_native or _ordinary()).quantize_rows(x)
        if done is not None:
            return done
    device = x.get_device()
    if device < 0 or stream is not None or device != _current_device():
        return _elsewhere(quantize_rows, x, stream, out, scales)
    kind = _FLOATS.get(x.dtype)
    if kind is None:
        _refuse("x.dtype: " + _FLOAT_NAMES, x.dtype)
    shape = x.shape
    if not shape or shape[-1] < 1:
        _refuse("x_tensor.size(-1) > 0")
    rows = _rows_of(x)
    m, k = rows.shape
    if out is None:
        pitch = (k + 15) // 16 * 16
        q = torch.empty_strided((m, k), (pitch, 1), dtype=_int8, device=x.device)
        out = q if len(shape) == 2 else q.view(shape) if k == pitch else torch.empty(shape[:-1] + (pitch,), dtype=_int8, device=x.device)[..., :k]
    elif out.dtype is not _int8 or out.shape != shape or out.get_device() != device or (out.stride(-1) != 1 and k > 1):
        _refuse("out: int8 of x's shape on x's device, values of a row next to each other")
    if m:
        q = _rows_to(out)
    if scales is None:
        scales = torch.empty((m,), dtype=_float32, device=x.device)
        if len(shape) != 2:
            scales = scales.view(shape[:-1])
    else:
        _check_vector(scales, m, device, "scales")
    if not m:
        return out, scales
    status = _lib.load().tsb_quantize_rows_i8(rows.data_ptr(), kind, rows.stride(0), q.data_ptr(), q.stride(0), scales.data_ptr(), m, k,
                                              _current_raw_stream(device))
    if status:
        check(status)
    return out, scales


def inner_prod_quantized(x, x_scales, w, w_scales, bias=None, residual=None, activation=ACT_NONE, leaky=0.0, out_dtype=None, out=None,
                         residual_after_activation=False, kernel=KERNEL_AUTO, stream=None):
    """x [..., k] times w [n, k] transposed, in int8 with int32 sums, a scale per token and per output channel:
    ``activation(sum * w_scales * x_scales + bias + residual)`` (or ``activation(...) + residual``), [..., n].

    x is int8 with ``x_scales`` (one per row, or one value for all), as quantize_rows gives them, or floating with ``x_scales=None``: then
    its rows are quantized in the call.  w int8 and w_scales [n] are what quantize_rows makes of a float weight tensor.  ``residual``
    has the output's type and shape.  ``out_dtype`` is x's type (of int8 rows: float32) unless given; ``out`` takes the result where
    it is given (it may be ``residual``, and no other operand)."""
    if out is None and stream is None and kernel == KERNEL_AUTO:
        done = (_native or _ordinary()).inner_prod(x, x_scales, w, w_scales, bias, residual, activation, leaky, out_dtype, bool(residual_after_activation))
        if done is not None:
            return done
    device = x.get_device()
    if device < 0 or stream is not None or device != _current_device():
        return _elsewhere(inner_prod_quantized, x, stream, x_scales, w, w_scales, bias, residual, activation, leaky, out_dtype, out,
                          residual_after_activation, kernel)
    x_dtype, shape = x.dtype, x.shape
    if x_scales is None:
        if x_dtype not in _FLOATS:
            _refuse("x.dtype: int8 with x_scales, without " + _FLOAT_NAMES, x_dtype)
    elif x_dtype is not _int8:
        _refuse("x.dtype: int8 with x_scales, not %s", x_dtype)
    if w.dtype is not _int8 or w.dim() != 2 or w.get_device() != device:
        _refuse("w: an int8 matrix on x's device")
    n, k = w.shape
    if not shape or shape[-1] != k:
        _refuse("w_tensor.size(1) == x_tensor.size(-1)")
    if k < 1:
        _refuse("x_tensor.size(-1) > 0")
    rows, w = _rows_of(x), _rows_of(w)
    m = rows.shape[0]
    _check_vector(w_scales, n, device, "w_scales")
    scales_at = scales_step = 0
    if x_scales is not None:
        one = x_scales.numel() == 1
        _check_vector(x_scales, 1 if one else m, device, "x_scales")
        scales_at, scales_step = x_scales.data_ptr(), 0 if one else 1
    bias_at = 0
    if bias is not None:
        _check_vector(bias, n, device, "bias")
        bias_at = bias.data_ptr()
    dtype = out_dtype if out_dtype is not None else out.dtype if out is not None else x_dtype if x_scales is None else _float32
    kind = _FLOATS.get(dtype)
    if kind is None:
        _refuse("out_dtype: " + _FLOAT_NAMES, dtype)
    want = (m, n) if len(shape) == 2 else shape[:-1] + (n,)
    if out is None:
        y = torch.empty((m, n), dtype=dtype, device=x.device)
        out = y if len(shape) == 2 else y.view(want)
    else:
        if out.dtype is not dtype or out.shape != want or out.get_device() != device or (out.stride(-1) != 1 and n > 1):
            _refuse("out: of out_dtype, [..., n] on x's device, values of a row next to each other")
        y = _rows_to(out) if out.numel() else out
    residual_at = residual_step = 0
    if residual is not None:
        if residual.dtype is not dtype or residual.shape != want or residual.get_device() != device:
            _refuse("residual: of the output's type and shape on x's device")
    if not (m and n):
        return out
    if residual is not None:
        residual = _rows_of(residual)
        residual_at, residual_step = residual.data_ptr(), residual.stride(0)
    lib = _lib.load()
    args = _lib.INNER_PROD_ARGS.pack(m, n, k, rows.data_ptr(), rows.stride(0), scales_at, scales_step, w.data_ptr(), w.stride(0), w_scales.data_ptr(),
                                     bias_at, residual_at, residual_step, y.data_ptr(), y.stride(0), _TYPE[x_dtype], kind, activation, leaky,
                                     1 if residual_after_activation else 0, kernel)
    workspace = size = 0
    if x_scales is None:
        size = lib.tsb_inner_prod_i8_workspace_bytes(args)
        if size:
            room = torch.empty((size,), dtype=torch.uint8, device=x.device)
            workspace = room.data_ptr()
    status = lib.tsb_inner_prod_i8(args, workspace, size, _current_raw_stream(device))
    if status:
        check(status)
    return out


def inner_prod_status(device=None, stream=None):
    """Waits for ``stream`` (the device's current one) and raises TsbError where a wait inside a tensor-core inner product on that
    device ran out since the last check: its results are not to be used."""
    with torch.cuda.device(device):
        check(_lib.load().tsb_inner_prod_i8_status(_stream_ptr(stream)))


def group_norm_nhwc(x, groups, gamma=None, beta=None, eps=1e-5, activation=ACT_NONE, leaky=0.0, out_dtype=None, requant_scales=None,
                    out=None, stream=None):
    """Group norm and activation of a channels-last x [n, ..., channels] (fp32, fp16 or bf16): mean and variance of each image's
    ``groups`` equal runs of channels over all its pixels, ``activation((x - mean) / sqrt(variance + eps) * gamma + beta)``.

    The result has x's type and shape (``out`` takes it where it is given; it may be x).  ``out_dtype=torch.int8`` with
    ``requant_scales`` (one, or one per image) gives ``quantize`` of it as NHWC_PAD [n, ..., padded_channels(channels)] instead, what
    a convolution plan reads."""
    if out is None and stream is None:
        done = (_native or _ordinary()).group_norm(x, groups, gamma, beta, eps, activation, leaky, out_dtype, requant_scales)
        if done is not None:
            return done
    device = x.get_device()
    if device < 0 or stream is not None or device != _current_device():
        return _elsewhere(group_norm_nhwc, x, stream, groups, gamma, beta, eps, activation, leaky, out_dtype, requant_scales, out)
    kind, shape = _FLOATS.get(x.dtype), x.shape
    if kind is None:
        _refuse("x.dtype: " + _FLOAT_NAMES, x.dtype)
    if len(shape) < 3:
        _refuse("x_tensor.dims() >= 3")
    n, c = shape[0], shape[-1]
    if c < 1:
        _refuse("x_tensor.size(-1) > 0")
    dtype = out_dtype if out_dtype is not None else x.dtype if out is None else out.dtype
    if dtype is not x.dtype and dtype is not _int8:
        _refuse("out_dtype: x's type or int8, not %s", dtype)
    pixels = x.numel() // (n * c) if n else 0
    gamma_at = beta_at = 0
    if gamma is not None:
        _check_vector(gamma, c, device, "gamma")
        gamma_at = gamma.data_ptr()
    if beta is not None:
        _check_vector(beta, c, device, "beta")
        beta_at = beta.data_ptr()
    lib = _lib.load()
    scales_at = n_scales = 0
    if dtype is _int8:
        if requant_scales is None:
            _refuse("out_dtype int8 comes with requant_scales")
        scales = _scales_of(requant_scales)
        scales_at, n_scales = ctypes.addressof(scales), len(scales)
        want = shape[:-1] + (lib.tsb_padded_channels(c),)
    else:
        if requant_scales is not None:
            _refuse("requant_scales come with out_dtype int8")
        want = shape
    x_step = _pixel_step(x)
    if x_step is None:
        x, x_step = x.contiguous(), c
    y_image = y_step = 0
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format) if want is shape else torch.empty(want, dtype=dtype, device=x.device)
        y_image, y_step = pixels * c, c
    else:
        if out.dtype is not dtype or out.shape != want or out.get_device() != device:
            _refuse("out: x's shape (int8: NHWC_PAD) and the output's type on x's device")
        y_image, y_step = out.stride(0), _pixel_step(out)
        if y_step is None or (dtype is _int8 and not out.is_contiguous()):
            _refuse("out: pixels of an image a fixed step apart, channels next to each other (int8: contiguous)")
    desc = _lib.GROUP_NORM_DESC.pack(n, pixels, c, groups, x.data_ptr(), x_step, x.stride(0), out.data_ptr(), y_step, y_image, gamma_at, beta_at, eps,
                                     scales_at, n_scales, kind, _TYPE[dtype], activation, leaky)
    size = lib.tsb_group_norm_workspace_bytes(desc)
    workspace = 0
    if size:
        room = torch.empty((size,), dtype=torch.uint8, device=x.device)
        workspace = room.data_ptr()
    status = lib.tsb_group_norm_nhwc(desc, workspace, size, _current_raw_stream(device))
    if status:
        check(status)
    return out


def _pixel_step(x):
    """Elements between neighbouring pixels of an image of x [n, ..., c]; None where they lie no fixed step apart, or a pixel's
    channels not next to each other."""
    c = x.shape[-1]
    if x.is_contiguous():
        return c
    if x.stride(-1) != 1 and c > 1:
        return None
    first = step = None
    for size, stride in zip(x.shape[-2:0:-1], x.stride()[-2:0:-1]):
        if size != 1:
            if first is None:
                first = stride
            elif stride != step:
                return None
            step = stride * size
    return c if first is None else first


# ---- layers in 4 bits: quantize_rows_mxfp4, dequantize_rows_mxfp4, inner_prod_mxfp4; rms_norm, in front of products in 8 or 4 bits ----------
# Devices, streams, and which calls go through native.cpp: as above.  A 4-bit matrix [m, k] is a tensor of torch.float4_e2m1fn_x2 (two
# values an element), [m, 16 * ceil(k / 32)], and its scales are one of torch.float8_e8m0fnu, [ceil(m / 128), ceil(k / 128), 32, 4, 4] in the order that the
# tensor cores read (mxfp4_scale_tiles makes it of scales row by row); uint8 tensors of the same bytes are taken too, and are what comes out where PyTorch has
# no such types.
def _row_bytes(k):
    return (k + 31) // 32 * 16


def _scale_shape(m, k):
    return ((m + 127) // 128, (k + 127) // 128, 32, 4, 4)


def _check_mxfp4(t, device, name):
    if (t.dtype is not _mxfp4 and t.dtype is not _uint8) or t.get_device() != device:
        _refuse("%s: float4_e2m1fn_x2 (or its bytes as uint8) on x's device, not %s", name, t.dtype)
    if not t.dim() or t.shape[-1] % 16 or not t.shape[-1]:
        _refuse("%s.size(-1): 16 bytes for every 32 values", name)


def _check_scales(t, m, k, device, name):
    if (t.dtype is not _e8m0 and t.dtype is not _uint8) or t.shape != _scale_shape(m, k) or t.get_device() != device or not t.is_contiguous():
        _refuse("%s: contiguous float8_e8m0fnu (or its bytes as uint8) of %s on x's device", name, list(_scale_shape(m, k)))


def mxfp4_scale_tiles(scales, out=None):
    """Scales of a 4-bit matrix as other programs hold them, [m, ceil(k / 32)] row by row (float8_e8m0fnu or uint8), in the order of
    quantize_rows_mxfp4's: [ceil(m / 128), ceil(groups / 4), 32, 4, 4], zero where there is no row or group.  For weights, once."""
    if scales.dim() != 2 or (scales.dtype is not _e8m0 and scales.dtype is not _uint8):
        _refuse("scales: float8_e8m0fnu or uint8 [m, groups], not %s", scales.dtype)
    m, groups = scales.shape
    room = torch.zeros(((m + 127) // 128 * 128, (groups + 3) // 4 * 4), dtype=_uint8, device=scales.device)
    room[:m, :groups] = scales.view(_uint8)
    tiles = room.view(-1, 4, 32, room.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    if out is None:
        return tiles.contiguous().view(_e8m0)
    _check_scales(out, m, 32 * groups, scales.get_device(), "out")
    out.view(_uint8).copy_(tiles)
    return out


def quantize_rows_mxfp4(x, out=None, scales=None, stream=None):
    """4-bit values of x [..., k] (fp32, fp16 or bf16) with a power of two for every 32 of a row: (q, scales), as tsb_quantize_rows_mxfp4 says.

    q is [..., 16 * ceil(k / 32)] float4_e2m1fn_x2, scales [ceil(m / 128), ceil(k / 128), 32, 4, 4] float8_e8m0fnu over the m rows of x.  The
    rows are tokens of an activation, or output channels of a weight tensor.  ``out`` and ``scales`` take the results where they are given; else both may
    lie in one storage (clone() one that is kept, or written to a file, without the other)."""
    if out is None and scales is None and stream is None:
        done = (_native or _ordinary()).quantize_rows_mxfp4(x)
        if done is not None:
            return done
    device = x.get_device()
    if device < 0 or stream is not None or device != _current_device():
        return _elsewhere(quantize_rows_mxfp4, x, stream, out, scales)
    kind, shape = _FLOATS.get(x.dtype), x.shape
    if kind is None:
        _refuse("x.dtype: " + _FLOAT_NAMES, x.dtype)
    if not shape or shape[-1] < 1:
        _refuse("x_tensor.size(-1) > 0")
    rows = _rows_of(x)
    m, k = rows.shape
    want = shape[:-1] + (_row_bytes(k),)
    if out is None:
        out = torch.empty(want, dtype=_mxfp4, device=x.device)
    elif (out.dtype is not _mxfp4 and out.dtype is not _uint8) or out.shape != want or out.get_device() != device or out.stride(-1) != 1:
        _refuse("out: float4_e2m1fn_x2 %s on x's device, bytes of a row next to each other", list(want))
    if scales is None:
        scales = torch.empty(_scale_shape(m, k), dtype=_e8m0, device=x.device)
    else:
        _check_scales(scales, m, k, device, "scales")
    if m:
        q = _rows_to(out)
        status = _lib.load().tsb_quantize_rows_mxfp4(rows.data_ptr(), kind, rows.stride(0), q.data_ptr(), q.stride(0), scales.data_ptr(), m, k, _current_raw_stream(device))
        if status:
            check(status)
    return out, scales


def dequantize_rows_mxfp4(q, scales, k=None, dtype=torch.float32, out=None, stream=None):
    """The values [..., k] that 4-bit rows q [..., 16 * ceil(k / 32)] with these scales stand for, rounded once to ``dtype`` (``out`` takes
    them where it is given, and says their type).  k: twice q's last size unless given."""
    if out is None and stream is None:
        done = (_native or _ordinary()).dequantize_rows_mxfp4(q, scales, k, dtype)
        if done is not None:
            return done
    device = q.get_device()
    if device < 0 or stream is not None or device != _current_device():
        return _elsewhere(dequantize_rows_mxfp4, q, stream, scales, k, dtype, out)
    _check_mxfp4(q, device, "q")
    shape = q.shape
    k = 2 * shape[-1] if k is None else operator.index(k)
    if k < 1 or _row_bytes(k) != shape[-1]:
        _refuse("k: a row of %d bytes holds %d to %d values", shape[-1], 2 * shape[-1] - 31, 2 * shape[-1])
    rows = _rows_of(q)
    m = rows.shape[0]
    _check_scales(scales, m, k, device, "scales")
    dtype = dtype if out is None else out.dtype
    kind, want = _FLOATS.get(dtype), shape[:-1] + (k,)
    if kind is None:
        _refuse("dtype: " + _FLOAT_NAMES, dtype)
    if out is None:
        out = torch.empty(want, dtype=dtype, device=q.device)
    elif out.shape != want or out.get_device() != device or (out.stride(-1) != 1 and k > 1):
        _refuse("out: %s on q's device, values of a row next to each other", list(want))
    if m:
        y = _rows_to(out)
        status = _lib.load().tsb_dequantize_rows_mxfp4(rows.data_ptr(), rows.stride(0), scales.data_ptr(), y.data_ptr(), kind, y.stride(0), m, k, _current_raw_stream(device))
        if status:
            check(status)
    return out


def inner_prod_mxfp4(x, x_scales, w, w_scales, bias=None, residual=None, activation=ACT_NONE, leaky=0.0, out_dtype=None, out=None,
                     residual_after_activation=False, kernel=KERNEL_AUTO, stream=None):
    """x [..., k] times w [n, k] transposed, both in 4 bits with a power of two for every 32 values of a row, sums in fp32:
    ``activation(sum + bias + residual)`` (or ``activation(...) + residual``), [..., n].

    w and w_scales are what quantize_rows_mxfp4 makes of a float weight tensor; x and x_scales what it (or rms_norm) makes of activations, or x is
    floating with ``x_scales=None``: then its rows are quantized in the call.  ``residual`` has the output's type and shape.  ``out_dtype`` is
    x's type (of 4-bit rows: float32) unless given; ``out`` takes the result where it is given (it may be ``residual``, and no other operand)."""
    if out is None and stream is None and kernel == KERNEL_AUTO:
        done = (_native or _ordinary()).inner_prod_mxfp4(x, x_scales, w, w_scales, bias, residual, activation, leaky, out_dtype, bool(residual_after_activation))
        if done is not None:
            return done
    device = x.get_device()
    if device < 0 or stream is not None or device != _current_device():
        return _elsewhere(inner_prod_mxfp4, x, stream, x_scales, w, w_scales, bias, residual, activation, leaky, out_dtype, out, residual_after_activation, kernel)
    x_dtype, shape = x.dtype, x.shape
    _check_mxfp4(w, device, "w")
    if w.dim() != 2:
        _refuse("w: a matrix")
    n, k = w.shape[0], 2 * w.shape[1]
    if x_scales is None:
        if x_dtype not in _FLOATS:
            _refuse("x.dtype: 4 bits with x_scales, without " + _FLOAT_NAMES, x_dtype)
        if not shape or shape[-1] < 1 or _row_bytes(shape[-1]) != w.shape[1]:
            _refuse("w_tensor.size(1) == 16 * ceil(x_tensor.size(-1) / 32)")
        k = shape[-1]
    else:
        _check_mxfp4(x, device, "x")
        if shape[-1] != w.shape[1]:
            _refuse("w_tensor.size(1) == x_tensor.size(-1)")
    rows, w = _rows_of(x), _rows_of(w)
    m = rows.shape[0]
    _check_scales(w_scales, n, k, device, "w_scales")
    scales_at = bias_at = 0
    if x_scales is not None:
        _check_scales(x_scales, m, k, device, "x_scales")
        scales_at = x_scales.data_ptr()
    if bias is not None:
        _check_vector(bias, n, device, "bias")
        bias_at = bias.data_ptr()
    dtype = out_dtype if out_dtype is not None else out.dtype if out is not None else x_dtype if x_scales is None else _float32
    kind = _FLOATS.get(dtype)
    if kind is None:
        _refuse("out_dtype: " + _FLOAT_NAMES, dtype)
    want = shape[:-1] + (n,)
    if out is None:
        out = torch.empty(want, dtype=dtype, device=x.device)
    elif out.dtype is not dtype or out.shape != want or out.get_device() != device or (out.stride(-1) != 1 and n > 1):
        _refuse("out: of out_dtype, [..., n] on x's device, values of a row next to each other")
    residual_at = residual_step = 0
    if residual is not None:
        if residual.dtype is not dtype or residual.shape != want or residual.get_device() != device:
            _refuse("residual: of the output's type and shape on x's device")
    if not (m and n):
        return out
    y = _rows_to(out)
    if residual is not None:
        residual = _rows_of(residual)
        residual_at, residual_step = residual.data_ptr(), residual.stride(0)
    lib = _lib.load()
    args = _lib.INNER_PROD_MXFP4_ARGS.pack(m, n, k, rows.data_ptr(), rows.stride(0), scales_at, w.data_ptr(), w.stride(0), w_scales.data_ptr(), bias_at, residual_at,
                                           residual_step, y.data_ptr(), y.stride(0), _TYPE.get(x_dtype, _lib.TYPE_MXFP4), kind, activation, leaky,
                                           1 if residual_after_activation else 0, kernel)
    workspace = size = 0
    if x_scales is None:
        size = lib.tsb_inner_prod_mxfp4_workspace_bytes(args)
        if size:
            room = torch.empty((size,), dtype=_uint8, device=x.device)
            workspace = room.data_ptr()
    status = lib.tsb_inner_prod_mxfp4(args, workspace, size, _current_raw_stream(device))
    if status:
        check(status)
    return out


def inner_prod_mxfp4_status(device=None, stream=None):
    """inner_prod_status for inner_prod_mxfp4."""
    with torch.cuda.device(device):
        check(_lib.load().tsb_inner_prod_mxfp4_status(_stream_ptr(stream)))


def rms_norm(x, gamma=None, residual=None, eps=1e-6, out_dtype=None, out=None, scales=None, sum_out=None, stream=None):
    """Root-mean-square norm of the rows of x [..., k] (fp32, fp16 or bf16): ``h / sqrt(mean(h * h) + eps) * gamma`` with h = x + residual (x's
    type) where a residual of x's type and shape is given, else x.

    The result has x's type and shape; with ``out_dtype=torch.int8`` it is (q, scales) as quantize_rows gives them, what inner_prod_quantized reads,
    with ``out_dtype=torch.float4_e2m1fn_x2`` (q, scales) as quantize_rows_mxfp4 gives them, what inner_prod_mxfp4 reads.  With a residual h comes
    as one result more: y, h or q, scales, h.  ``out``, ``scales`` and ``sum_out`` (h; it may be ``residual`` or x) take the results where they are given; q and
    scales that are not may lie in one storage, as quantize_rows_mxfp4's."""
    if out is None and scales is None and sum_out is None and stream is None:
        done = (_native or _ordinary()).rms_norm(x, gamma, residual, eps, out_dtype)
        if done is not None:
            return done
    device = x.get_device()
    if device < 0 or stream is not None or device != _current_device():
        return _elsewhere(rms_norm, x, stream, gamma, residual, eps, out_dtype, out, scales, sum_out)
    kind, shape = _FLOATS.get(x.dtype), x.shape
    if kind is None:
        _refuse("x.dtype: " + _FLOAT_NAMES, x.dtype)
    if not shape or shape[-1] < 1:
        _refuse("x_tensor.size(-1) > 0")
    dtype = out_dtype if out_dtype is not None else x.dtype if out is None else out.dtype
    packed = dtype is _mxfp4 or (dtype is _uint8 and out is not None and out_dtype is None)
    if dtype is not x.dtype and dtype is not _int8 and not packed:
        _refuse("out_dtype: x's type, int8 or float4_e2m1fn_x2, not %s", dtype)
    if residual is not None and (residual.dtype is not x.dtype or residual.shape != shape or residual.get_device() != device):
        _refuse("residual: of x's type and shape on x's device")
    rows = _rows_of(x)
    m, k = rows.shape
    gamma_at = residual_at = residual_step = sum_at = sum_step = scales_at = 0
    if gamma is not None:
        _check_vector(gamma, k, device, "gamma")
        gamma_at = gamma.data_ptr()
    want = shape[:-1] + (_row_bytes(k),) if packed else shape
    if out is not None:
        if (out.dtype is not dtype and not (packed and out.dtype is _uint8)) or out.shape != want or out.get_device() != device or (out.stride(-1) != 1 and want[-1] > 1):
            _refuse("out: %s of out_dtype on x's device, values of a row next to each other", list(want))
    elif dtype is _int8:
        # rows start a multiple of 16 bytes apart, as quantize_rows has them
        out = torch.empty(shape[:-1] + ((k + 15) // 16 * 16,), dtype=_int8, device=x.device)[..., :k]
    else:
        out = torch.empty(want, dtype=dtype, device=x.device)
    if dtype is x.dtype:
        if scales is not None:
            _refuse("scales come with out_dtype int8 or float4_e2m1fn_x2")
    elif scales is not None:
        if packed:
            _check_scales(scales, m, k, device, "scales")
        else:
            _check_vector(scales, m, device, "scales")
    else:
        scales = torch.empty(_scale_shape(m, k), dtype=_e8m0, device=x.device) if packed else torch.empty(shape[:-1], dtype=_float32, device=x.device)
    if residual is None:
        if sum_out is not None:
            _refuse("sum_out comes with a residual")
    elif sum_out is None:
        sum_out = torch.empty(shape, dtype=x.dtype, device=x.device)
    elif sum_out.dtype is not x.dtype or sum_out.shape != shape or sum_out.get_device() != device or (sum_out.stride(-1) != 1 and k > 1):
        _refuse("sum_out: of x's type and shape on x's device, values of a row next to each other")
    if m:
        y = _rows_to(out)
        if residual is not None:
            residual = _rows_of(residual)
            residual_at, residual_step = residual.data_ptr(), residual.stride(0)
            h = _rows_to(sum_out)
            sum_at, sum_step = h.data_ptr(), h.stride(0)
        if scales is not None:
            scales_at = scales.data_ptr()
        desc = _lib.RMS_NORM_DESC.pack(m, k, rows.data_ptr(), rows.stride(0), residual_at, residual_step, sum_at, sum_step, gamma_at, y.data_ptr(), y.stride(0), scales_at, eps,
                                       kind, _lib.TYPE_MXFP4 if packed else _TYPE[dtype])
        status = _lib.load().tsb_rms_norm(desc, _current_raw_stream(device))
        if status:
            check(status)
    done = (out,) + ((scales,) if scales is not None else ()) + ((sum_out,) if residual is not None else ())
    return done if len(done) > 1 else out
