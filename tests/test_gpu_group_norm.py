"""group_norm_nhwc against the norm in 64 bits, at sizes, values and layouts where it can go wrong."""
import numpy as np
import pytest
import torch

import int8_layers as plain

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def tensors(shape, dtype, seed=0, shift=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[-1]
    x = torch.randn(shape, device="cuda", generator=g) * (0.5 + torch.rand(c, device="cuda", generator=g)) + shift * torch.randn(c, device="cuda", generator=g)
    return x.to(dtype), 1.0 + 0.3 * torch.randn(c, device="cuda", generator=g), 0.3 * torch.randn(c, device="cuda", generator=g)


def numbers(t):
    return None if t is None else t.float().cpu().double().numpy()


def check(got, x, groups, gamma=None, beta=None, eps=1e-5, act=0, leaky=0.0):
    want, bound = plain.group_norm(numbers(x), groups, numbers(gamma), numbers(beta), eps, act, leaky)
    plain.assert_close(got, want, bound, got.dtype)


SIZES = [(1, 1, 1, 2, 1), (1, 1, 1, 64, 4), (2, 7, 7, 64, 32), (1, 16, 16, 128, 32), (3, 5, 9, 12, 4), (2, 13, 11, 30, 3), (1, 33, 17, 320, 32), (2, 8, 8, 96, 6), (5, 3, 3, 7, 7),
         (1, 64, 64, 32, 1), (4, 28, 28, 256, 32), (1, 1, 5000, 16, 2), (1, 100, 100, 3, 1), (2, 4, 4, 2048, 32), (1, 2, 2, 4100, 41), (1, 56, 56, 64, 64), (40, 2, 3, 24, 8),
         (1, 128, 128, 40, 8), (2, 40, 40, 640, 32), (1, 200, 200, 8, 8), (1, 9, 7, 1000, 8), (200, 4, 4, 16, 4), (1, 160, 160, 256, 32), (2, 96, 96, 1024, 32)]


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("n,h,w,c,groups", SIZES)
def test_sizes(n, h, w, c, groups, dtype):
    from tennis_b200 import ops
    x, gamma, beta = tensors((n, h, w, c), dtype, n + h + w + c)
    got = ops.group_norm_nhwc(x, groups, gamma, beta)
    assert got.shape == x.shape and got.dtype == dtype
    check(got, x, groups, gamma, beta)
    assert torch.equal(got, ops.group_norm_nhwc(x, groups, gamma, beta))       # and the same bits again


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("act,leaky", [(1, 0.0), (2, 0.1), (3, 0.0), (4, 0.0)])
def test_activations_and_missing_vectors(dtype, act, leaky):
    from tennis_b200 import ops
    for shape, groups in (((2, 9, 10, 48), 4), ((1, 70, 70, 128), 32)):
        x, gamma, beta = tensors(shape, dtype, act)
        check(ops.group_norm_nhwc(x, groups, gamma, beta, 1e-3, act, leaky), x, groups, gamma, beta, 1e-3, act, leaky)
        check(ops.group_norm_nhwc(x, groups, None, beta, activation=act, leaky=leaky), x, groups, None, beta, act=act, leaky=leaky)
        check(ops.group_norm_nhwc(x, groups, gamma, activation=act, leaky=leaky), x, groups, gamma, None, act=act, leaky=leaky)
        check(ops.group_norm_nhwc(x, groups, activation=act, leaky=leaky), x, groups, act=act, leaky=leaky)


@pytest.mark.parametrize("shape,groups", [((2, 11, 11, 64), 8), ((1, 90, 90, 96), 32)])
def test_values_far_from_zero(shape, groups):
    """A mean of thousands of deviations, a constant image (variance zero), values near the type's largest."""
    from tennis_b200 import ops
    x, gamma, beta = tensors(shape, torch.float32, 1)
    check(ops.group_norm_nhwc(x + 5000.0, groups, gamma, beta), x + 5000.0, groups, gamma, beta)
    same = torch.full(shape, 3.25, device="cuda")
    check(ops.group_norm_nhwc(same, groups, gamma, beta), same, groups, gamma, beta)
    big = (x * 1e30).contiguous()
    check(ops.group_norm_nhwc(big, groups, gamma, beta), big, groups, gamma, beta)
    small = (x * 1e-20).contiguous()
    check(ops.group_norm_nhwc(small, groups, gamma, beta, 1e-5), small, groups, gamma, beta)
    check(ops.group_norm_nhwc(small, groups, gamma, beta, 0.0), small, groups, gamma, beta, 0.0)


@pytest.mark.parametrize("mean", [1e4, -1e6, 1e7])
@pytest.mark.parametrize("shape,groups", [((2, 11, 11, 64), 8), ((1, 90, 90, 96), 32), ((1, 9, 9, 15), 3)])
def test_means_of_many_deviations(shape, groups, mean):
    """The variance's relative error, (mean / deviation)^2 2^-52 or a small multiple of it (counted here with 2^-49), beside the rounded mean's."""
    from tennis_b200 import ops
    x, gamma, beta = tensors(shape, torch.float32, 3, shift=0.0)
    x = x + mean
    want, bound = plain.group_norm(numbers(x), groups, numbers(gamma), numbers(beta))
    plain.assert_close(ops.group_norm_nhwc(x, groups, gamma, beta), want, bound + np.abs(want - numbers(beta)) * (mean / 0.5) ** 2 * 2.0 ** -49, torch.float32)


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("shape,groups", [((2, 8, 8, 64), 8), ((2, 16, 8, 32), 8), ((1, 256, 256, 256), 32), ((1, 256, 256, 128), 32)])
def test_steps_are_rounded_one_by_one(shape, groups, dtype):
    """Whole numbers, of which every group has a power of two: sums, mean and variance are exact in 64 bits whatever their order, so the steps behind
    mean and reciprocal deviation (each rounded to fp32) can be compared bit for bit."""
    from tennis_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(groups)
    _, gamma, beta = tensors(shape, dtype, 9)
    x = torch.randint(-60, 100, shape, device="cuda", generator=g).to(dtype)
    t = x.double().view(shape[0], -1, groups, shape[-1] // groups)
    mean = t.mean((1, 3), keepdim=True)
    rstd = 1.0 / ((t * t).mean((1, 3), keepdim=True) - mean * mean + 1e-5).sqrt()
    v = ((t.float() - mean.float()) * rstd.float()).view(shape) * gamma + beta
    assert torch.equal(ops.group_norm_nhwc(x, groups, gamma, beta), v.to(dtype))
    assert torch.equal(ops.group_norm_nhwc(x, groups, gamma, beta, activation=1), v.clamp(min=0.0).to(dtype))


def test_deviation_and_gamma_whose_product_no_number_holds():
    """eps = 0, deviations of 10^-25 and gammas of 10^20: their quotient is beyond fp32, the results are not."""
    from tennis_b200 import ops
    for shape in ((2, 8, 8, 32), (2, 90, 90, 64), (1, 7, 9, 33)):
        x, gamma, beta = tensors(shape, torch.float32, 4)
        x, gamma = (x * 1e-25).to(torch.bfloat16), gamma * 1e20
        got = ops.group_norm_nhwc(x, shape[-1] // (8 if shape[-1] % 8 == 0 else 11), gamma, beta, 0.0)
        assert torch.isfinite(got).all()
        check(got, x, shape[-1] // (8 if shape[-1] % 8 == 0 else 11), gamma, beta, 0.0)


def test_nan_and_infinity_stay_in_their_group():
    from tennis_b200 import ops
    for shape in ((3, 8, 8, 32), (3, 80, 80, 32)):
        x, gamma, beta = tensors(shape, torch.bfloat16, 2)
        clean = ops.group_norm_nhwc(x, 4, gamma, beta)
        x[1, 3, 4, 9] = float("nan")
        x[2, 0, 0, 31] = float("inf")
        got = ops.group_norm_nhwc(x, 4, gamma, beta)
        touched = torch.zeros(shape, dtype=torch.bool, device="cuda")
        touched[1, ..., 8:16] = True
        touched[2, ..., 24:32] = True
        assert torch.equal(got[~touched], clean[~touched]) and torch.isnan(got[touched]).all()


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("n,h,w,c,groups", [(1, 5, 5, 16, 4), (2, 7, 9, 24, 3), (3, 14, 14, 64, 8), (2, 6, 7, 75, 5), (1, 3, 5, 3, 1), (4, 56, 56, 64, 32), (1, 100, 100, 130, 10), (16, 28, 28, 256, 32)])
def test_int8_output(dtype, n, h, w, c, groups):
    """quantize() of the floating result of an fp32 copy of the input, which has the same bits before quantize; padding channels zero."""
    from tennis_b200 import _lib, ops
    x, gamma, beta = tensors((n, h, w, c), dtype, n + c)
    v = ops.group_norm_nhwc(x.float(), groups, gamma, beta, activation=_lib.ACT_RELU)
    for scales in ([20.0], [20.0 + i for i in range(n)]):
        got = ops.group_norm_nhwc(x, groups, gamma, beta, activation=_lib.ACT_RELU, out_dtype=torch.int8, requant_scales=scales)
        assert got.shape == (n, h, w, ops.padded_channels(c)) and (got[..., c:] == 0).all()
        nchw = v.permute(0, 3, 1, 2).contiguous()
        want = torch.empty_like(nchw, dtype=torch.int8)
        _lib.check(_lib.load().tsb_quantize_f32_i8(ops._ptr(nchw), ops._ptr(want), nchw.numel(), _lib.float_array(scales), len(scales), ops._stream_ptr()))
        assert torch.equal(got[..., :c], want.permute(0, 2, 3, 1))


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("hw", [9, 60])
def test_layouts(dtype, hw):
    """Slices of channels, pixels and images, a channels-last view of NCHW, tokens of a sequence, outputs of the caller's, in place."""
    from tennis_b200 import ops
    x, gamma, beta = tensors((3, hw, hw, 72), dtype, 5)
    gamma, beta = gamma[:48].contiguous(), beta[:48].contiguous()
    nchw = x[..., :48].permute(0, 3, 1, 2).contiguous(memory_format=torch.channels_last)
    for t in (x[..., 8:56], x[..., 5:53], x[:, :, :5, :48], x[1:, 2:7, :, 16:64], x[:, :, :1, :48], x[:, :1, :, 3:51], nchw.permute(0, 2, 3, 1), x[..., :48].flatten(1, 2),
              x[0:1].expand(4, hw, hw, 72)[..., 1:49], x.permute(0, 2, 1, 3)[..., :48]):
        got = ops.group_norm_nhwc(t, 8, gamma, beta, activation=1)
        assert got.is_contiguous()
        check(got, t, 8, gamma, beta, act=1)
        room = torch.full(t.shape[:-1] + (61,), 7.0, dtype=dtype, device="cuda")
        out = room[..., 3:51]
        assert ops.group_norm_nhwc(t, 8, gamma, beta, activation=1, out=out) is out and torch.equal(out, got)
        assert (room[..., :3] == 7).all() and (room[..., 51:] == 7).all()
        if 0 not in t.stride():
            mine = x.clone()
            view = mine.as_strided(t.shape, t.stride(), t.storage_offset()) if t.data_ptr() != nchw.data_ptr() else nchw.clone().permute(0, 2, 3, 1)
            if ops._pixel_step(view) is not None:
                ops.group_norm_nhwc(view, 8, gamma, beta, activation=1, out=view)
                assert torch.equal(view, got)


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("act", [3, 4])
def test_bits_of_a_value_are_its_own(dtype, act):
    """Activations give the same bits by vectors and value by value (a view that starts off 16 bytes), resident and swept."""
    from tennis_b200 import ops
    for shape in ((3, 30, 30, 72), (2, 200, 200, 136)):
        x, gamma, beta = tensors(shape, dtype, 13)
        c = shape[-1] - 8
        gamma, beta = gamma[:c].contiguous(), beta[:c].contiguous()
        odd = x[..., 5:5 + c]
        assert torch.equal(ops.group_norm_nhwc(odd, 8, gamma, beta, activation=act), ops.group_norm_nhwc(odd.contiguous(), 8, gamma, beta, activation=act))


def test_far_offsets():
    from tennis_b200 import ops
    step = (1 << 32) // 63 + 8
    x, gamma, beta = tensors((1, 8, 8, 32), torch.bfloat16, 6)
    far = torch.empty(63 * step + 64, dtype=torch.bfloat16, device="cuda").as_strided((1, 64, 32), (64 * step, step, 1))
    far.copy_(x.view(1, 64, 32))
    check(ops.group_norm_nhwc(far, 4, gamma, beta), far, 4, gamma, beta)
    ops.group_norm_nhwc(far, 4, gamma, beta, out=far)
    check(far, x.view(1, 64, 32), 4, gamma, beta)


def test_streams_and_graphs():
    """Two graphs and an eager call on a third stream at once: no call uses another's memory."""
    from tennis_b200 import ops
    for hw in (8, 100):
        x, gamma, beta = tensors((3, hw, hw, 128), torch.float16, 7)
        want = ops.group_norm_nhwc(x, 32, gamma, beta)
        graphs, outs = [], []
        for i in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(ops.group_norm_nhwc(x[i:i + 1], 32, gamma, beta))
            graphs.append(graph)
        streams = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        for _ in range(10):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
            eager = ops.group_norm_nhwc(x[2:], 32, gamma, beta, stream=streams[2])
        torch.cuda.synchronize()
        for i, got in enumerate(outs + [eager]):
            assert torch.equal(got, want[i:i + 1])


def test_refusals():
    from tennis_b200 import ops
    x, gamma, beta = tensors((1, 4, 4, 16), torch.float32, 8)
    for call in (lambda: ops.group_norm_nhwc(x, 4, requant_scales=[1.0]), lambda: ops.group_norm_nhwc(x, 4, out_dtype=torch.int8), lambda: ops.group_norm_nhwc(x[0, 0], 4),
                 lambda: ops.group_norm_nhwc(x.double(), 4), lambda: ops.group_norm_nhwc(x, 4, gamma[:8]), lambda: ops.group_norm_nhwc(x, 4, gamma, beta.double()),
                 lambda: ops.group_norm_nhwc(x, 4, out_dtype=torch.float16), lambda: ops.group_norm_nhwc(x, 4, out=x[..., :8]),
                 lambda: ops.group_norm_nhwc(x, 4, out=torch.empty((1, 4, 4, 16, 2), device="cuda")[..., 0])):
        with pytest.raises(ops.EjectionException, match="Check failed"):
            call()
    with pytest.raises(RuntimeError, match="do not make 5 groups"):
        ops.group_norm_nhwc(x, 5)


def test_empty():
    from tennis_b200 import ops
    for shape in ((0, 4, 4, 8), (2, 0, 4, 8)):
        assert ops.group_norm_nhwc(torch.empty(shape, device="cuda"), 2).shape == shape


def test_into_a_convolution_and_an_inner_product():
    """A residual block of group norms, the way a network runs it: norm -> int8 -> 3x3 convolution -> norm -> quantize_rows -> product over
    the pixels with the input as its residual; against the same operators one by one and against the plain forms."""
    from tennis_b200 import _lib, ops
    n, h, w, c = 2, 20, 18, 64
    x, gamma, beta = tensors((n, h, w, c), torch.float32, 11)
    g = torch.Generator(device="cuda").manual_seed(12)
    weight = torch.randint(-127, 128, (c, c, 3, 3), device="cuda", generator=g, dtype=torch.int8)
    dq = torch.rand(c, device="cuda", generator=g) * 1e-4
    proj, ps = ops.quantize_rows(torch.randn((c, c), device="cuda", generator=g) / 8)
    scales = [30.0] * n
    q = ops.group_norm_nhwc(x, 32, gamma, beta, activation=_lib.ACT_SILU, out_dtype=torch.int8, requant_scales=scales)
    plan = ops.ConvPlan((n, c, h, w), (c, c, 3, 3), (1, 1, 1, 1), (1, 1), (1, 1))
    plan.set_weights(weight)
    y = torch.empty((n, h, w, c), device="cuda")
    plan.run(q, _lib.LAYOUT_NHWC_PAD, dq, out_f32=y, out_f32_layout=_lib.LAYOUT_NHWC_PAD)
    plan.status()
    want = torch.nn.functional.conv2d(q[..., :c].permute(0, 3, 1, 2).double(), weight.double(), padding=1).permute(0, 2, 3, 1) * dq.double()
    assert torch.allclose(y.double(), want, rtol=1e-6, atol=1e-6)
    z = ops.group_norm_nhwc(y, 32, gamma, beta, activation=_lib.ACT_SILU)
    check(z, y, 32, gamma, beta, act=3)
    out = ops.inner_prod_quantized(z, None, proj, ps, residual=x)
    zq, zs = ops.quantize_rows(z)
    assert torch.equal(out, ops.inner_prod_quantized(zq, zs, proj, ps, residual=x))
    ref, bound = plain.inner_prod(zq.reshape(-1, c).cpu().numpy(), numbers(zs).reshape(-1), proj.cpu().numpy(), numbers(ps), residual=numbers(x).reshape(-1, c))
    plain.assert_close(out.view(-1, c), ref, bound, torch.float32)
