"""Refusals of quantize_rows, inner_prod_quantized and group_norm_nhwc that need no GPU, the layout of their argument blocks, and the
plain forms that their GPU tests compare with."""
import ctypes
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

import int8_layers as plain
from conftest import ROOT


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    from tennis_b200 import _lib
    return _lib.load()


P = 4096      # an address that is never followed: every call here is refused, or has nothing to do


def rows(lib, x=P, x_type=0, x_pitch=64, y=P, y_pitch=64, scales=P, m=2, k=64):
    return lib.tsb_quantize_rows_i8(x, x_type, x_pitch, y, y_pitch, scales, m, k, None)


@pytest.mark.parametrize("bad,text", [(dict(x_type=3), "no floating type"), (dict(x_type=-1), "no floating type"), (dict(m=-1), "bad shape"), (dict(k=0), "bad shape"),
                                      (dict(x=0), "null"), (dict(y=None), "null"), (dict(scales=0), "null"), (dict(x=P + 2), "aligned"), (dict(scales=P + 2), "aligned"),
                                      (dict(y_pitch=63), "overlap"), (dict(x_pitch=-64), "pitch"), (dict(x_pitch=1 << 61), "address range"), (dict(m=1 << 61), "address range")])
def test_quantize_rows_refuses(lib, bad, text):
    launched = lib.tsb_kernel_launch_count()
    assert rows(lib, **bad) == -1 and text in lib.tsb_last_error().decode() and lib.tsb_kernel_launch_count() == launched


def test_nothing_to_do(lib):
    assert rows(lib, m=0, x=None, y=None, scales=None) == 0
    assert product(lib, m=0) == 0 and product(lib, n=0) == 0
    assert norm(lib, n=0, n_scales=0) == 0 and norm(lib, pixels=0) == 0


def product(lib, m=2, n=8, k=64, x=P, x_pitch=64, xs=P, xs_stride=1, w=P, w_pitch=64, ws=P, bias=0, res=0, res_pitch=8, y=P, y_pitch=8, x_type=3, y_type=0, act=0, leaky=0.0,
            after=0, kernel=0, workspace=None, size=0):
    from tennis_b200 import _lib
    args = _lib.INNER_PROD_ARGS.pack(m, n, k, x, x_pitch, xs, xs_stride, w, w_pitch, ws, bias, res, res_pitch, y, y_pitch, x_type, y_type, act, leaky, after, kernel)
    return lib.tsb_inner_prod_i8(args, workspace, size, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(m=-1), -1, "bad shape"), (dict(n=-1), -1, "bad shape"), (dict(n=1 << 31), -1, "bad shape"), (dict(k=0), -1, "k = 0"), (dict(k=131072, x_pitch=131072, w_pitch=131072), -1, "k = 131072"),
    (dict(x_type=4), -1, "x_type 4"), (dict(y_type=3), -1, "y_type 3"), (dict(act=5), -1, "activation 5"), (dict(act=-1), -1, "activation -1"), (dict(kernel=7), -1, "kernel 7"),
    (dict(x=0), -1, "null"), (dict(w=0), -1, "null"), (dict(ws=0), -1, "null"), (dict(y=0), -1, "null"), (dict(xs=0), -1, "x_scales"), (dict(x_type=0), -1, "x_scales"),
    (dict(xs_stride=2), -1, "x_scales_stride"), (dict(y=P + 2), -1, "aligned"), (dict(xs=P + 1), -1, "aligned"), (dict(ws=P + 2), -1, "aligned"), (dict(bias=P + 3), -1, "aligned"),
    (dict(res=P + 1), -1, "aligned"), (dict(x_type=0, xs=0, x=P + 1), -1, "aligned"), (dict(y_pitch=7), -1, "pitch"), (dict(x_pitch=-1), -1, "pitch"), (dict(w_pitch=-64), -1, "pitch"),
    (dict(res=P, res_pitch=-8), -1, "pitch"), (dict(x_pitch=1 << 62), -1, "address range"), (dict(y_pitch=1 << 61), -1, "address range"),
    (dict(x_type=1, xs=0), -3, "workspace"), (dict(x_type=1, xs=0, workspace=P, size=100), -3, "workspace"), (dict(x_type=1, xs=0, workspace=P + 16, size=1 << 20), -1, "256-byte")])
def test_inner_prod_refuses(lib, bad, status, text):
    launched = lib.tsb_kernel_launch_count()
    assert product(lib, **bad) == status and text in lib.tsb_last_error().decode() and lib.tsb_kernel_launch_count() == launched


def norm(lib, n=2, pixels=9, channels=32, groups=4, x=P, x_pixel=32, x_image=288, y=P, y_pixel=32, y_image=288, gamma=0, beta=0, eps=1e-5, scales=None, n_scales=None, x_type=0, y_type=0,
         act=0, leaky=0.0, workspace=P, size=1 << 30):
    from tennis_b200 import _lib
    arr = None if scales is None else _lib.float_array(scales)
    desc = _lib.GROUP_NORM_DESC.pack(n, pixels, channels, groups, x, x_pixel, x_image, y, y_pixel, y_image, gamma, beta, eps, 0 if arr is None else ctypes.addressof(arr),
                                     (0 if arr is None else len(arr)) if n_scales is None else n_scales, x_type, y_type, act, leaky)
    return lib.tsb_group_norm_nhwc(desc, workspace, size, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(n=-1), -1, "bad shape"), (dict(pixels=-1), -1, "bad shape"), (dict(channels=0), -1, "bad shape"), (dict(groups=0), -1, "bad shape"), (dict(groups=5), -1, "do not make"),
    (dict(x_type=3, y_type=3), -1, "x_type 3"), (dict(y_type=1), -1, "y_type"), (dict(act=9), -1, "activation 9"), (dict(eps=-1.0), -1, "eps"), (dict(eps=float("nan")), -1, "eps"),
    (dict(eps=float("inf")), -1, "eps"), (dict(y_type=3), -1, "requant_scales"), (dict(y_type=3, scales=[1.0] * 3), -1, "one per image"),
    (dict(y_type=3, n=129, scales=[1.0] * 129), -2, "128"), (dict(x=0), -1, "null"), (dict(y=0), -1, "null"), (dict(x=P + 2), -1, "aligned"), (dict(gamma=P + 1), -1, "aligned"),
    (dict(y_type=3, y=P + 8, scales=[1.0]), -1, "aligned"), (dict(x_pixel=-32), -1, "stride"), (dict(y_pixel=31), -1, "overlap"), (dict(y_image=287), -1, "overlap"),
    (dict(x_image=1 << 61), -1, "address range"), (dict(large=True, workspace=None), -3, "workspace"), (dict(large=True, size=16), -3, "workspace"),
    (dict(large=True, workspace=P + 64), -1, "256-byte")])
def test_group_norm_refuses(lib, bad, status, text):
    bad = dict(bad)
    if bad.pop("large", False):      # an image that no cluster holds: its sums go through a workspace
        bad = dict(pixels=1 << 20, channels=512, x_pixel=512, x_image=1 << 29, y_pixel=512, y_image=1 << 29, **bad)
    launched = lib.tsb_kernel_launch_count()
    assert norm(lib, **bad) == status and text in lib.tsb_last_error().decode() and lib.tsb_kernel_launch_count() == launched


def test_convolutions_refuse_the_new_activations(lib):
    """silu and gelu belong to the operators behind products and norms: a convolution's epilogue has neither."""
    from tennis_b200 import _lib
    d = _lib.ConvDesc()
    d.n, d.c, d.h, d.w, d.o, d.kh, d.kw = 1, 64, 4, 4, 64, 1, 1
    d.stride_h = d.stride_w = d.dilation_h = d.dilation_w = 1
    d.kernel = _lib.KERNEL_DIRECT
    plan = ctypes.c_void_p()
    assert lib.tsb_conv2d_i8_plan_create(ctypes.byref(d), ctypes.byref(plan)) == 0
    e = _lib.ConvEpilogue()
    e.dequantize_scales = e.out_f32 = P
    for act in (_lib.ACT_SILU, _lib.ACT_GELU):
        e.activation = act
        assert lib.tsb_conv2d_i8_run(plan, P, 0, ctypes.byref(e), P, 1 << 20, None) < 0
    lib.tsb_conv2d_i8_plan_destroy(plan)


def test_argument_blocks_match_the_header():
    """Names, order and types of the header's two structures are those of the packed blocks."""
    from tennis_b200 import _lib
    text = re.sub(r"/\*.*?\*/", "", open(ROOT + "/include/tennis_b200.h").read(), flags=re.S)
    for name, packed in (("tsb_inner_prod_args", _lib.INNER_PROD_ARGS), ("tsb_group_norm_desc", _lib.GROUP_NORM_DESC)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        codes = []
        for line in body.split(";"):
            if line.strip():
                kind = "P" if "*" in line else {"int64_t": "q", "double": "d", "int": "i", "float": "f"}[line.split()[0]]
                codes += [kind] * len(line.split(","))
        want = "".join(c * int(k or 1) for k, c in re.findall(r"(\d*)([qPdif])", packed.format.replace("0q", "")))
        assert "".join(codes) == want, name
        assert packed.size % 8 == 0


def cpu(shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_operators_refuse_host_tensors():
    from tennis_b200 import ops
    for call in (lambda: ops.quantize_rows(cpu((2, 8))), lambda: ops.inner_prod_quantized(cpu((2, 8)), None, cpu((4, 8), torch.int8), cpu(4)),
                 lambda: ops.group_norm_nhwc(cpu((1, 2, 2, 8)), 2)):
        with pytest.raises(ops.EjectionException, match="is_cuda"):
            call()


def test_the_module_of_ordinary_calls(monkeypatch):
    """It takes nothing that is not ordinary, and its absence is told."""
    from tennis_b200 import ops
    native = ops._ordinary()
    assert native.quantize_rows(cpu((2, 8))) is None and native.quantize_rows("x") is None and native.quantize_rows() is None
    assert native.inner_prod(*[None] * 10) is None and native.inner_prod(cpu((2, 8)), None, cpu((4, 8), torch.int8), cpu(4), None, None, 0, 0.0, None, False) is None
    assert native.group_norm(*[None] * 9) is None and native.group_norm(cpu((1, 2, 2, 8)), 2, None, None, 1e-5, 0, 0.0, None, None) is None
    import sys
    monkeypatch.setattr(ops, "_native", None)
    monkeypatch.delattr(__import__("tennis_b200"), "_native", raising=False)
    monkeypatch.setitem(sys.modules, "tennis_b200._native", None)
    with pytest.raises(RuntimeError, match="_native has not been built"):
        ops.quantize_rows(cpu((2, 8)))


def make(*goals):
    """What make would run, and its status."""
    done = subprocess.run(["make", "-n", "-C", ROOT + "/tennis_b200/csrc"] + list(goals), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    return done.returncode, done.stdout


def test_the_c_library_is_built_without_python(tmp_path):
    status, text = make("-B", "PYTHON=" + str(tmp_path / "none"))
    assert status == 0 and "libtennis_b200.so" in text and "native" not in text
    status, text = make("python", "PYTHON=" + str(tmp_path / "none"))
    assert status != 0 and "no PyTorch" in text


def test_the_module_is_built_again_for_another_pytorch(lib, tmp_path):
    """(lib: built just now for this one.)"""
    status, text = make("python", "PYTHON=" + sys.executable)
    assert status == 0 and "native.cpp" not in text
    other = tmp_path / "python"
    other.write_text("#!/bin/sh\necho another\n")
    other.chmod(0o755)
    status, text = make("python", "PYTHON=" + str(other))
    assert status == 0 and "native.cpp" in text


def test_pixel_step():
    from tennis_b200.ops import _pixel_step
    x = cpu((2, 5, 6, 16))
    assert _pixel_step(x) == 16 and _pixel_step(x[..., 2:10]) == 16 and _pixel_step(x[:, :, :1]) == 96 and _pixel_step(x[:, :1, :, :4]) == 16
    assert _pixel_step(x[:, :, :3]) is None and _pixel_step(x.permute(0, 2, 1, 3)) is None and _pixel_step(x.permute(0, 3, 1, 2)) is None
    assert _pixel_step(x[:, ::5]) == 16 and _pixel_step(x[:, :1, :1, :3]) == 3 and _pixel_step(x[..., ::16]) == 16 and _pixel_step(x[:, :, ::2]) == 32
    assert _pixel_step(cpu((2, 7, 16))[:, ::2]) == 32


def test_plain_rows():
    """The plain form itself, on values worked out by hand."""
    x = torch.tensor([[127.0, -63.5, 0.5, 1.5, -2.5], [0.0, 0.0, 0.0, -0.0, 0.0], [1.0, float("nan"), 2.0, 3.0, 4.0], [1.0, float("inf"), 2.0, -float("inf"), 4.0], [1e-31, 0, 0, 0, 0]])
    q, s = plain.quantize_rows(x)
    assert q.tolist() == [[127, -64, 0, 2, -2], [0] * 5, [-128] * 5, [0, -128, 0, -128, 0], [0] * 5]
    assert s[0] == 1.0 and s[1] == 0.0 and np.isnan(s[2]) and np.isinf(s[3]) and s[4] == 0.0


def test_plain_norm_and_product():
    x = np.arange(16, dtype=np.float64).reshape(1, 2, 2, 4)
    y, _ = plain.group_norm(x, 2, eps=0.0)
    assert abs(y[..., :2].mean()) < 1e-12 and abs((y[..., 2:] ** 2).mean() - 1) < 1e-12
    v, _ = plain.inner_prod(np.array([[1, 2]], dtype=np.int8), np.array([0.5]), np.array([[3, -4], [1, 1]], dtype=np.int8), np.array([1.0, 2.0]), bias=np.array([0.0, 1.0]), act=1)
    assert v.tolist() == [[0.0, 4.0]]
