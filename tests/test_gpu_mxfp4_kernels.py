"""Every kernel of inner_prod_mxfp4 by itself and beside the others, and 4-bit layers whose tensors lie among NaN."""
import pytest
import torch

import mxfp4_layers as plain
from mxfp4_kernels import ALL, FLOATING
from test_gpu_inner_prod_mxfp4 import FLOATS, call, case
from test_gpu_rms_norm import FP4, check as check_norm, features, weights
import test_gpu_mxfp4_rows as four

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [size for size, *_ in ALL])
def test_every_kernel(m, n, k):
    """Each output type, with a residual and without: sums are exact, so a product of doubles has the very bits behind the fp32 steps."""
    from tennis_b200 import ops
    d = case(m, n, k, torch.float32, m + n + k)
    x, w = ops.dequantize_rows_mxfp4(d["x"], d["xs"]).double(), ops.dequantize_rows_mxfp4(d["w"], d["ws"]).double()
    want = (x @ w.t()).float() + d["bias"]
    for out in FLOATS:
        r = d["residual"].to(out)
        assert torch.equal(call(dict(d, residual=None), out_dtype=out), want.to(out))
        assert torch.equal(call(dict(d, residual=r), out_dtype=out), (want + r.float()).to(out))
    ops.inner_prod_mxfp4_status()


@pytest.mark.parametrize("m,n,k", [size for size, _ in FLOATING])
def test_every_kernel_of_floating_rows(m, n, k):
    """What quantizes its rows itself has the bits of a product of 4-bit rows."""
    from tennis_b200 import ops
    for dtype in FLOATS:
        d = case(m, n, k, dtype, m)
        x = torch.randn((m, k), device="cuda", generator=torch.Generator(device="cuda").manual_seed(k)).to(dtype)
        q, s = ops.quantize_rows_mxfp4(x)
        got = ops.inner_prod_mxfp4(x, None, d["w"], d["ws"], d["bias"], d["residual"], 4)
        assert got.dtype == dtype and torch.equal(got, ops.inner_prod_mxfp4(q, s, d["w"], d["ws"], d["bias"], d["residual"], 4, out_dtype=dtype))


def test_every_kernel_beside_the_others():
    """Clusters that share tiles, pairs, kept weights, whole tiles, few tokens, and the int8 product's pairs and splits, on four streams at once: CTAs that hold tensor memory while
    they wait for their cluster share multiprocessors with all the others.  Every call has the bits that it has alone."""
    from tennis_b200 import ops
    sizes = [(2500, 2304, 4096), (130, 512, 4112), (128, 1024, 14336), (50000, 24, 500), (7, 1000, 4096), (64, 10000, 1100), (600, 40000, 300), (90, 161, 8000), (25, 2000, 2048), (1000, 1000, 1000)]
    cases = [case(m, n, k, torch.bfloat16, i) for i, (m, n, k) in enumerate(sizes)]
    calls = [lambda stream=None, d=d: call(d, out_dtype=torch.bfloat16, stream=stream) for d in cases]
    x = torch.randn((5, 4096), device="cuda").bfloat16()
    d = case(1, 1000, 4096, torch.bfloat16, 3)
    calls.append(lambda stream=None: ops.inner_prod_mxfp4(x, None, d["w"], d["ws"], d["bias"], stream=stream))
    for m, n, k in ((2048, 4096, 4096), (64, 2048, 8192)):
        a, b = (ops.quantize_rows(torch.randn(shape, device="cuda").bfloat16()) for shape in ((m, k), (n, k)))
        calls.append(lambda stream=None, a=a, b=b: ops.inner_prod_quantized(*a, *b, out_dtype=torch.bfloat16, stream=stream))
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in range(4)]
    for turn in range(12):
        got = []
        for side in streams:
            side.wait_stream(torch.cuda.current_stream())
        for i in range(2 * len(calls)):
            at = (i * 5 + turn) % len(calls)
            got.append((at, calls[at](streams[i % 4])))
        for side in streams:
            torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(y, want[at]) for at, y in got)
    ops.inner_prod_mxfp4_status()
    ops.inner_prod_status()


def among(t, fill=float("nan")):
    """t on a boundary of 16 bytes between values that must not be read: NaN, or bytes of `fill`."""
    if t.element_size() == 1:
        room = torch.full((t.numel() + 8192,), fill, dtype=torch.uint8, device="cuda")
        return room[4096:4096 + t.numel()].view(t.dtype).view(t.shape).copy_(t)
    return torch.full((t.numel() + 4096,), fill, dtype=t.dtype, device="cuda")[2048:2048 + t.numel()].view(t.shape).copy_(t)


@pytest.mark.parametrize("k", [4, 8, 40, 64, 100, 264, 320, 520, 1000, 1032, 4104, 8200, 16392, 40008])
def test_a_norm_among_nan(k):
    """Rows, residual and gamma between NaN: every value and every byte of scales, those of tiles behind the last group too."""
    from tennis_b200 import ops
    for m in (1, 3, 300):
        for dtype in FLOATS:
            x, r, gamma = among(features(m, k, dtype, k)), among(features(m, k, dtype, k + 1)), among(weights(k))
            for out in (dtype, torch.int8, FP4):
                check_norm(ops.rms_norm(x, gamma, out_dtype=out), x, gamma, None, out)
                check_norm(ops.rms_norm(x, gamma, r, out_dtype=out), x, gamma, r, out)


@pytest.mark.parametrize("m,k", [(1, 8), (3, 40), (130, 64), (5, 1000), (200, 104), (2, 16392)])
def test_rows_among_nan(m, k):
    from tennis_b200 import ops
    for dtype in FLOATS:
        x = among(four.features(m, k, dtype, k))
        q, s = ops.quantize_rows_mxfp4(x)
        four.check(x, q, s)
        want = ops.dequantize_rows_mxfp4(q, s, k, dtype)
        assert not want.isnan().any() and torch.equal(ops.dequantize_rows_mxfp4(among(q.view(torch.uint8), 0x77), among(s.view(torch.uint8), 255), k, dtype), want)


@pytest.mark.parametrize("m,n,k", [(1, 100, 200), (20, 130, 288), (40, 1000, 1100), (100, 130, 300), (130, 512, 4112), (129, 130, 16384), (2500, 2300, 1024), (50000, 24, 500)])
def test_a_product_among_nan(m, n, k):
    """Operands between codes of 6 and scales of NaN, bias and residual between NaN."""
    from tennis_b200 import ops
    for out in FLOATS:
        d = case(m, n, k, out, m)
        there = {"x": among(d["x"].view(torch.uint8), 0x77), "w": among(d["w"].view(torch.uint8), 0x77), "xs": among(d["xs"].view(torch.uint8), 255), "ws": among(d["ws"].view(torch.uint8), 255),
                 "bias": among(d["bias"]), "residual": among(d["residual"])}
        want = call(d, out_dtype=out)
        assert not want.isnan().any() and torch.equal(call(there, out_dtype=out), want)
