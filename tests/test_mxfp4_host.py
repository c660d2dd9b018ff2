"""Refusals of the 4-bit rows and products and of rms_norm that need no GPU, the layout of their argument blocks, and the plain forms that their
GPU tests compare with."""
import re

import numpy as np
import pytest
import torch

import mxfp4_layers as plain
from conftest import ROOT


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    from tennis_b200 import _lib
    return _lib.load()


P = 4096      # an address that is never followed: every call here is refused, or has nothing to do


def refused(lib, call, status, text):
    launched = lib.tsb_kernel_launch_count()
    assert call() == status and text in lib.tsb_last_error().decode() and lib.tsb_kernel_launch_count() == launched


def test_bytes(lib):
    assert [lib.tsb_mxfp4_row_bytes(k) for k in (0, -5, 1, 32, 33, 4096, 8191)] == [0, 0, 16, 16, 32, 2048, 4096]
    assert [lib.tsb_mxfp4_scale_bytes(*s) for s in ((0, 5), (5, 0), (-1, 5), (1, 1), (128, 128), (129, 128), (128, 129), (300, 1000))] == [0, 0, 0, 512, 512, 1024, 1024, 3 * 8 * 512]


def quantize(lib, x=P, x_type=0, x_pitch=64, q=P, q_pitch=32, scales=P, m=2, k=64):
    return lib.tsb_quantize_rows_mxfp4(x, x_type, x_pitch, q, q_pitch, scales, m, k, None)


def dequantize(lib, q=P, q_pitch=32, scales=P, y=P, y_type=0, y_pitch=64, m=2, k=64):
    return lib.tsb_dequantize_rows_mxfp4(q, q_pitch, scales, y, y_type, y_pitch, m, k, None)


@pytest.mark.parametrize("bad,text", [(dict(x_type=3), "no floating type"), (dict(x_type=4), "no floating type"), (dict(m=-1), "bad shape"), (dict(k=0), "bad shape"), (dict(k=1 << 31), "bad shape"),
                                      (dict(x=0), "null"), (dict(q=0), "null"), (dict(scales=0), "null"), (dict(x=P + 2), "aligned"), (dict(x_pitch=-64), "pitch"), (dict(q_pitch=31), "pitch"),
                                      (dict(x_pitch=1 << 61), "address range"), (dict(m=1 << 61, x_pitch=0), "address range"), (dict(m=1 << 39, x_pitch=0), "address range")])
def test_quantize_refuses(lib, bad, text):
    refused(lib, lambda: quantize(lib, **bad), -1, text)


@pytest.mark.parametrize("bad,text", [(dict(y_type=4), "no floating type"), (dict(m=-1), "bad shape"), (dict(k=-3), "bad shape"), (dict(q=0), "null"), (dict(y=0), "null"), (dict(scales=0), "null"),
                                      (dict(y=P + 1), "aligned"), (dict(y_pitch=63), "pitch"), (dict(q_pitch=-1), "pitch"), (dict(y_pitch=1 << 61), "address range")])
def test_dequantize_refuses(lib, bad, text):
    refused(lib, lambda: dequantize(lib, **bad), -1, text)


def product(lib, m=2, n=8, k=64, x=P, x_pitch=32, xs=P, w=P, w_pitch=32, ws=P, bias=0, res=0, res_pitch=8, y=P, y_pitch=8, x_type=4, y_type=0, act=0, leaky=0.0, after=0, kernel=0,
            workspace=None, size=0):
    from tennis_b200 import _lib
    args = _lib.INNER_PROD_MXFP4_ARGS.pack(m, n, k, x, x_pitch, xs, w, w_pitch, ws, bias, res, res_pitch, y, y_pitch, x_type, y_type, act, leaky, after, kernel)
    return lib.tsb_inner_prod_mxfp4(args, workspace, size, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(m=-1), -1, "bad shape"), (dict(n=-1), -1, "bad shape"), (dict(n=1 << 31), -1, "bad shape"), (dict(k=0), -1, "k = 0"), (dict(k=1 << 31), -1, "bad k"),
    (dict(x_type=3), -1, "x_type 3"), (dict(x_type=5), -1, "x_type 5"), (dict(y_type=4), -1, "y_type 4"), (dict(act=5), -1, "activation 5"), (dict(act=-1), -1, "activation -1"),
    (dict(kernel=7), -1, "kernel 7"), (dict(x=0), -1, "null"), (dict(w=0), -1, "null"), (dict(ws=0), -1, "null"), (dict(y=0), -1, "null"), (dict(xs=0), -1, "x_scales"), (dict(x_type=0), -1, "x_scales"),
    (dict(y=P + 2), -1, "aligned"), (dict(bias=P + 3), -1, "aligned"), (dict(res=P + 1), -1, "aligned"), (dict(x_type=0, xs=0, x=P + 1), -1, "aligned"), (dict(y_pitch=7), -1, "pitch"),
    (dict(x_pitch=-1), -1, "pitch"), (dict(w_pitch=-64), -1, "pitch"), (dict(res=P, res_pitch=-8), -1, "pitch"), (dict(x_pitch=1 << 62), -1, "address range"), (dict(y_pitch=1 << 61), -1, "address range"),
    (dict(x_type=1, xs=0, x_pitch=0, m=1 << 37, y_pitch=8, k=1 << 30), -1, "address range"), (dict(m=1 << 39, y_pitch=8), -1, "address range"),
    (dict(m=64, x_type=1, xs=0, x_pitch=64), -3, "workspace"), (dict(m=64, x_type=1, xs=0, x_pitch=64, workspace=P, size=100), -3, "workspace"),
    (dict(m=64, x_type=1, xs=0, x_pitch=64, workspace=P + 16, size=1 << 20), -1, "256-byte")])
def test_inner_prod_refuses(lib, bad, status, text):
    refused(lib, lambda: product(lib, **bad), status, text)


def norm(lib, m=2, k=64, x=P, x_pitch=64, res=0, res_pitch=64, total=0, sum_pitch=64, gamma=0, y=P, y_pitch=64, scales=0, eps=1e-6, x_type=0, y_type=0):
    from tennis_b200 import _lib
    return lib.tsb_rms_norm(_lib.RMS_NORM_DESC.pack(m, k, x, x_pitch, res, res_pitch, total, sum_pitch, gamma, y, y_pitch, scales, eps, x_type, y_type), None)


@pytest.mark.parametrize("bad,text", [
    (dict(m=-1), "bad shape"), (dict(k=0), "bad shape"), (dict(k=1 << 31), "bad shape"), (dict(x_type=3, y_type=3), "x_type 3"), (dict(y_type=1), "y_type 1"), (dict(y_type=7), "y_type 7"),
    (dict(eps=-1e-9), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(total=P), "residual"), (dict(x=0), "null"), (dict(y=0), "null"), (dict(y_type=3), "null"),
    (dict(y_type=4, y_pitch=32), "null"), (dict(x=P + 2), "aligned"), (dict(y=P + 2), "aligned"), (dict(gamma=P + 2), "aligned"), (dict(res=P + 1), "aligned"), (dict(res=P, total=P + 2), "aligned"),
    (dict(y_type=3, scales=P + 1), "aligned"), (dict(x_pitch=-1), "pitch"), (dict(y_pitch=63), "pitch"), (dict(y_type=4, scales=P, y_pitch=31), "pitch"), (dict(res=P, res_pitch=-64), "pitch"),
    (dict(res=P, total=P, sum_pitch=63), "pitch"), (dict(x_pitch=1 << 61), "address range"), (dict(m=1 << 39, x_pitch=0, y_pitch=64), "address range")])
def test_rms_norm_refuses(lib, bad, text):
    refused(lib, lambda: norm(lib, **bad), -1, text)


def test_null_blocks(lib):
    refused(lib, lambda: lib.tsb_rms_norm(None, None), -1, "null")
    refused(lib, lambda: lib.tsb_inner_prod_mxfp4(None, None, 0, None), -1, "null")
    assert lib.tsb_inner_prod_mxfp4_workspace_bytes(None) == 0


def test_nothing_to_do(lib):
    assert quantize(lib, m=0, x=None, q=None, scales=None) == 0 and dequantize(lib, m=0, q=None, y=None, scales=None) == 0
    assert product(lib, m=0) == 0 and product(lib, n=0) == 0 and norm(lib, m=0, x=0, y=0) == 0


def test_argument_blocks_match_the_header():
    from tennis_b200 import _lib
    text = re.sub(r"/\*.*?\*/", "", open(ROOT + "/include/tennis_b200.h").read(), flags=re.S)
    for name, packed in (("tsb_inner_prod_mxfp4_args", _lib.INNER_PROD_MXFP4_ARGS), ("tsb_rms_norm_desc", _lib.RMS_NORM_DESC)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, flags=re.S).group(1)
        codes = []
        for line in body.split(";"):
            if line.strip():
                kind = "P" if "*" in line else {"int64_t": "q", "double": "d", "int": "i", "float": "f"}[line.split()[0]]
                codes += [kind] * len(line.split(","))
        assert "".join(codes) == "".join(c * int(k or 1) for k, c in re.findall(r"(\d*)([qPdif])", packed.format)), name
        assert packed.size % 8 == 0


def test_operators_refuse_host_tensors():
    from tennis_b200 import ops
    x, q, s = torch.zeros((2, 64)), torch.zeros((2, 32), dtype=torch.uint8), torch.zeros((1, 1, 32, 4, 4), dtype=torch.uint8)
    for call in (lambda: ops.quantize_rows_mxfp4(x), lambda: ops.dequantize_rows_mxfp4(q, s), lambda: ops.inner_prod_mxfp4(x, None, q, s), lambda: ops.rms_norm(x)):
        with pytest.raises(ops.EjectionException, match="is_cuda"):
            call()


def test_the_module_of_ordinary_calls():
    """It takes nothing that is not ordinary."""
    from tennis_b200 import ops
    native, x = ops._ordinary(), torch.zeros((2, 64))
    assert native.quantize_rows_mxfp4(x) is None and native.quantize_rows_mxfp4("x") is None and native.quantize_rows_mxfp4() is None
    assert native.dequantize_rows_mxfp4(*[None] * 4) is None and native.dequantize_rows_mxfp4(x, x, None, torch.float32) is None and native.dequantize_rows_mxfp4(x) is None
    assert native.inner_prod_mxfp4(*[None] * 10) is None and native.inner_prod_mxfp4(x, None, x, x, None, None, 0, 0.0, None, False) is None
    assert native.rms_norm(*[None] * 5) is None and native.rms_norm(x, None, None, 1e-6, None) is None and native.rms_norm() is None


def test_scale_tiles():
    """The order of tiles, against places worked out one by one."""
    from tennis_b200 import ops
    for m, groups in ((1, 1), (5, 4), (128, 4), (129, 5), (300, 33)):
        s = np.random.RandomState(m).randint(1, 255, (m, groups)).astype(np.uint8)
        t = ops.mxfp4_scale_tiles(torch.from_numpy(s))
        assert t.dtype == torch.float8_e8m0fnu and t.shape == ((m + 127) // 128, (groups + 3) // 4, 32, 4, 4) and t.is_contiguous()
        assert np.array_equal(t.view(torch.uint8).numpy().reshape(-1), plain.tiles(s)) and np.array_equal(plain.from_tiles(plain.tiles(s), m, groups), s)
        into = torch.empty(tuple(t.shape), dtype=torch.uint8)
        assert ops.mxfp4_scale_tiles(torch.from_numpy(s).view(torch.float8_e8m0fnu), out=into) is into and torch.equal(into, t.view(torch.uint8))
    for bad in (torch.zeros((2, 2)), torch.zeros(4, dtype=torch.uint8), torch.zeros((2, 2), dtype=torch.int8)):
        with pytest.raises(ops.EjectionException):
            ops.mxfp4_scale_tiles(bad)


def test_plain_rows():
    """The plain form itself, on values worked out by hand."""
    x = np.zeros((3, 40))
    x[0, :10] = [4.0, 0.25, 0.75, -1.25, 1.75, 2.5, -3.5, 5.0, 7.0, -0.2]      # scale 1
    x[0, 32] = 12.0                                                            # scale 2
    x[1, 0], x[2, 1] = np.nan, 2.0 ** -140
    codes, scales = plain.quantize(x)
    assert codes[0, :10].tolist() == [6, 0, 2, 8 + 2, 4, 4, 8 + 6, 6, 7, 8] and codes[0, 32] == 7 and scales.tolist() == [[127, 128], [255, 0], [0, 0]]
    assert plain.values(codes, scales)[0, [0, 3, 8, 32]].tolist() == [4.0, -1.0, 6.0, 12.0] and np.isnan(plain.values(codes, scales)[1, :32]).all()
    assert np.array_equal(plain.unpack(plain.pack(codes)), codes)


def test_plain_norm_and_product():
    x = torch.tensor([[3.0, 4.0, 0.0, 0.0]])
    v, h = plain.rms_norm(x, torch.tensor([1.0, 2.0, 1.0, 1.0]), torch.tensor([[0.0, 0.0, 0.0, 0.0]]), eps=0.0)
    assert np.allclose(v, [[1.2, 3.2, 0.0, 0.0]]) and torch.equal(h, x)
    y, _ = plain.inner_prod(np.array([[1.0, 2.0]]), np.array([[3.0, -4.0], [1.0, 1.0]]), bias=np.array([0.0, 1.0]), act=1)
    assert y.tolist() == [[0.0, 4.0]]


def test_every_wait_code_has_a_name_of_its_own(lib):
    from tennis_b200 import _lib
    kernel = "".join(open(ROOT + "/tennis_b200/csrc/inner_prod_mxfp4_%s.cu" % name).read() for name in ("tc", "few"))
    codes = sorted({int(c) for c in re.findall(r"give_up\((\d+)\)", kernel)})
    assert codes == list(range(1, len(codes) + 1))
    names = set()
    for code in codes:
        assert lib.tsb_inner_prod_mxfp4_status_decode(code) == _lib.ERR_DEVICE_TIMEOUT
        names.add(re.search(r"the wait for (.*) ran out;", lib.tsb_last_error().decode()).group(1))
    assert len(names) == len(codes) and "an unknown event" not in names
    assert lib.tsb_inner_prod_mxfp4_status_decode(codes[-1] + 1) == _lib.ERR_DEVICE_TIMEOUT and "an unknown event" in lib.tsb_last_error().decode()
    assert lib.tsb_inner_prod_mxfp4_status_decode(0) == 0
    assert "code (1..%d, which wait) in it" % codes[-1] in open(ROOT + "/include/tennis_b200.h").read()


OLDER = """
import sys, torch
del torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
sys.path.insert(0, %r)
import tennis_b200
from tennis_b200 import ops, nets
s = torch.arange(2 * 5, dtype=torch.uint8).view(2, 5)
t = ops.mxfp4_scale_tiles(s)
assert t.dtype == torch.uint8 and t.shape == (1, 2, 32, 4, 4) and t[0, 1, 1, 0, 0] == 9
for call in (lambda: ops.quantize_rows_mxfp4(torch.zeros(2, 64)), lambda: ops.rms_norm(torch.zeros(2, 64), out_dtype=torch.uint8)):
    try:
        call()
    except ops.EjectionException as e:
        assert "is_cuda" in str(e)
    else:
        raise AssertionError("a host tensor was taken")
"""


def test_the_package_needs_no_4_bit_types():
    """A PyTorch without the types of 4-bit values and their scales: the package imports, and works on their bytes."""
    import subprocess
    import sys
    done = subprocess.run([sys.executable, "-c", OLDER % ROOT], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert done.returncode == 0, done.stdout[-2000:]
