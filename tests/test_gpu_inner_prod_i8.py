"""inner_prod_quantized against the product in 64 bits, at sizes, layouts and epilogues where it can go wrong."""
import struct

import numpy as np
import pytest
import torch

import int8_layers as plain

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def int8(m, k, gen, pitch=None, at=0):
    """An int8 matrix whose rows lie `pitch` apart, all of [-128, 127] in it."""
    pitch = pitch or (k + 15) // 16 * 16
    room = torch.empty(m * pitch + at + 16, dtype=torch.int8, device="cuda").random_(-128, 128, generator=gen)
    return room[at:].as_strided((m, k), (pitch, 1))


def case(m, n, k, out, seed=0, residual=True, bias=True, **layout):
    g = torch.Generator(device="cuda").manual_seed(seed)
    d = dict(x=int8(m, k, g, layout.get("x_pitch"), layout.get("x_at", 0)), w=int8(n, k, g, layout.get("w_pitch"), layout.get("w_at", 0)),
             xs=torch.empty(m, device="cuda").uniform_(0.5, 2.0, generator=g), ws=torch.empty(n, device="cuda").uniform_(0.5, 2.0, generator=g) / (5000.0 * k ** 0.5),
             bias=torch.randn(n, device="cuda", generator=g) if bias else None,
             residual=torch.randn((m, n), device="cuda", generator=g).to(out) if residual else None)
    return d


def numbers(t):
    return None if t is None else t.float().cpu().double().numpy()


def check(got, d, act=0, leaky=0.0, after=False):
    want, bound = plain.inner_prod(d["x"].cpu().numpy(), d["xs"].cpu().numpy(), d["w"].cpu().numpy(), d["ws"].cpu().numpy(), numbers(d["bias"]), numbers(d["residual"]),
                                   act, leaky, after)
    plain.assert_close(got, want, bound, got.dtype)


SIZES = [(1, 1, 1), (1, 8, 16), (1, 1000, 2048), (1, 37, 4099), (2, 129, 64), (3, 64, 100), (4, 1024, 1024), (5, 4096, 512), (7, 333, 8192), (8, 250, 1040),
         (9, 65, 333), (16, 1000, 2048), (17, 128, 128), (24, 511, 192), (31, 2048, 272), (32, 96, 4096), (33, 100, 48), (63, 777, 130), (64, 1000, 2048),
         (65, 257, 1000), (100, 130, 4096), (127, 64, 127), (128, 128, 128), (129, 256, 256), (130, 512, 4112), (200, 40, 96), (255, 300, 144), (256, 256, 1024),
         (257, 255, 2048), (300, 1024, 512), (500, 1000, 500), (700, 512, 640), (1000, 96, 64), (1025, 513, 1009), (2049, 64, 32), (4096, 200, 128), (333, 777, 1021),
         (2300, 1300, 400), (6000, 16, 16)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_sizes(m, n, k):
    """Every size with the layout that quantize_rows gives, with contiguous (odd) rows and with each output type."""
    from tennis_b200 import ops
    for i, out in enumerate(FLOATS):
        d = case(m, n, k, out, m + n + k + i, residual=i != 1, bias=i != 2)
        got = ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], d["bias"], d["residual"], out_dtype=out)
        assert got.dtype == out and got.shape == (m, n)
        check(got, d)
    d["x"], d["w"] = d["x"].contiguous(), d["w"].contiguous()
    check(ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], d["bias"], d["residual"], out_dtype=out), d)


@pytest.mark.parametrize("m,n,k", [(1, 200, 512), (12, 200, 512), (40, 200, 500), (150, 200, 512), (400, 520, 1024)])
@pytest.mark.parametrize("act,leaky", [(0, 0.0), (1, 0.0), (2, 0.1), (2, -0.25), (3, 0.0), (4, 0.0)])
def test_activations(m, n, k, act, leaky):
    from tennis_b200 import ops
    for out in FLOATS:
        for after in (False, True):
            d = case(m, n, k, out, act)
            got = ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], d["bias"], d["residual"], act, leaky, out, residual_after_activation=after)
            check(got, d, act, leaky, after)


@pytest.mark.parametrize("m", [1, 12, 40, 150, 400])
@pytest.mark.parametrize("act", [1, 3, 4])
def test_activations_of_the_largest_values(m, act):
    """Values to the ends of fp32, infinities and NaN, side by side: what is far below zero becomes zero (an infinity NaN, 0 times it, as
    the formulas say), and none changes its neighbour.  Sums of zero leave the bias itself."""
    from tennis_b200 import ops
    ends = [-1e4, 3.0, -1e30, -3.3e38, -44.0, -43.0, float("nan"), -1.0, -float("inf"), -2.0, float("inf"), -90.0, 3.3e38, -200.0, 1e-30, -3.3e38]
    for n in (16, 200):
        bias = torch.tensor((ends * 13)[:n], device="cuda")
        v = bias.double().cpu()
        want = v.clamp(min=0.0).nan_to_num(nan=0.0, posinf=float("inf")) if act == 1 else v / (1.0 + torch.exp(-v)) if act == 3 else 0.5 * v * (1.0 + torch.erf(v * 0.5 ** 0.5))
        for out in FLOATS:
            d = case(m, n, 48, out, 3)
            got = ops.inner_prod_quantized(torch.zeros_like(d["x"]), d["xs"], d["w"], d["ws"], bias, activation=act, out_dtype=out).cpu()
            # fp32: silu by 8 half steps of its value, gelu by 24 of 1; one rounding to 16 bits; 10^-17 as plain.activation's quotient
            torch.testing.assert_close(got.double(), want.to(out).double().expand(m, n), rtol=2 * torch.finfo(out).eps + 8 * plain.EPS32,
                                       atol=24 * plain.EPS32 if act == 4 else 1e-17, equal_nan=True)


@pytest.mark.parametrize("m", [1, 6, 30, 140, 700])
def test_kernels_agree_bit_for_bit(m):
    """The result's bits depend neither on the kernel nor on the rows that are computed with a row."""
    from tennis_b200 import _lib, ops
    d = case(m, 330, 1056, torch.float32, m)
    args = (d["x"], d["xs"], d["w"], d["ws"], d["bias"], d["residual"], _lib.ACT_SILU)
    got = ops.inner_prod_quantized(*args)
    assert torch.equal(got, ops.inner_prod_quantized(*args, kernel=_lib.KERNEL_DIRECT))
    assert torch.equal(got[m // 2:], ops.inner_prod_quantized(d["x"][m // 2:], d["xs"][m // 2:], *args[2:5], d["residual"][m // 2:], _lib.ACT_SILU))


@pytest.mark.parametrize("out", FLOATS, ids=str)
@pytest.mark.parametrize("act,leaky", [(0, 0.0), (1, 0.0), (2, 0.1), (3, 0.0), (4, 0.0)])
def test_bits_of_a_value_are_its_own(out, act, leaky):
    """They depend on a row of x, a row of w and what is added: not on the kernel, on the rows or channels beside it (on either side of the 32
    rows at which kernels change), or on the call.  An odd number of channels: the last one has no neighbour."""
    from tennis_b200 import _lib, ops
    for m, n, k in ((900, 1001, 64), (300, 776, 1056)):
        for after in (False, True):
            d = case(m, n, k, out, act)

            def call(rows=slice(None), channels=slice(None), **kw):
                return ops.inner_prod_quantized(d["x"][rows], d["xs"][rows], d["w"][channels], d["ws"][channels], d["bias"][channels], d["residual"][rows, channels].contiguous(), act, leaky,
                                                out, residual_after_activation=after, **kw)
            got = call()
            assert torch.equal(got, call(kernel=_lib.KERNEL_DIRECT))
            for rows in (slice(0, 1), slice(5, 37), slice(5, 38), slice(40, 140), slice(m // 2, m)):
                assert torch.equal(got[rows], call(rows))
            assert torch.equal(got[:, 1:], call(channels=slice(1, n)))
            assert torch.equal(got[7:39, 1:], call(slice(7, 39), slice(1, n)))
            for _ in range(3):
                assert torch.equal(got, call())


@pytest.mark.parametrize("m,n,k", [(4096, 2560, 2048), (2500, 2304, 4096), (9472, 256, 4096), (2049, 4097, 2176), (2430, 2432, 8192), (4097, 2080, 1920)])
def test_large_products(m, n, k):
    """Sizes of many tiles a multiprocessor, of one and of two CTAs: int32 sums do not depend on their order, so a product of doubles has the
    very bits of what is left to do in fp32."""
    from tennis_b200 import ops
    d = case(m, n, k, torch.float32, m, residual=False)
    want = (d["x"].double() @ d["w"].double().t()).float() * d["ws"] * d["xs"][:, None] + d["bias"]
    for out in FLOATS:
        got = ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], d["bias"], out_dtype=out)
        assert torch.equal(got, want.to(out))
    ops.inner_prod_status()


def after_the_sums(d, acc, act, after):
    """The fp32 steps behind the sums (whole numbers, exact in `acc`), one by one as the header lists them."""
    v = acc.float() * d["ws"] * d["xs"][:, None] + d["bias"]
    r = d["residual"].float()
    if not after:
        v = v + r
    if act == 1:
        v = v.clamp(min=0.0)
    return v + r if after else v


@pytest.mark.parametrize("m,n,k", [(2048, 4096, 4096), (4992, 2560, 2048), (2430, 2432, 8192), (3201, 2056, 4096), (1152, 4096, 4096), (4096, 2560, 2048), (2049, 4097, 2176)])
@pytest.mark.parametrize("act,after", [(0, False), (1, False), (1, True)])
def test_large_products_with_a_residual(m, n, k, act, after):
    """Tiles of two CTAs (the first four: also an odd number of 128 tokens, tokens and channels that fill no tile) and of one, many a
    multiprocessor: the very bits of a product of doubles and the fp32 steps behind it."""
    from tennis_b200 import ops
    for out in FLOATS:
        d = case(m, n, k, out, m + act)
        want = after_the_sums(d, d["x"].double() @ d["w"].double().t(), act, after).to(out)
        got = ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], d["bias"], d["residual"], act, out_dtype=out, residual_after_activation=after)
        assert torch.equal(got, want)
    ops.inner_prod_status()


@pytest.mark.parametrize("m,n,k", [(2048, 4096, 4096), (4992, 2560, 2048), (2049, 4097, 2176)])
def test_large_products_onto_their_residual(m, n, k):
    """The residual is the output: every element is read before it is written."""
    from tennis_b200 import ops
    for out in FLOATS:
        d = case(m, n, k, out, m + 7)
        want = after_the_sums(d, d["x"].double() @ d["w"].double().t(), 0, False).to(out)
        y = d["residual"].clone()
        assert ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], d["bias"], y, out=y) is y
        assert torch.equal(y, want)
    ops.inner_prod_status()


@pytest.mark.parametrize("x_pitch,x_at,w_pitch,w_at", [(512, 0, 512, 0), (512, 0, 500, 0), (501, 0, 512, 0), (512, 1, 512, 0), (512, 0, 512, 4), (520, 8, 504, 8), (1024, 16, 640, 32)])
@pytest.mark.parametrize("m", [1, 13, 50, 300])
def test_layouts(m, x_pitch, x_at, w_pitch, w_at):
    from tennis_b200 import ops
    d = case(m, 150, 500, torch.float16, x_pitch, x_pitch=x_pitch, x_at=x_at, w_pitch=w_pitch, w_at=w_at)
    check(ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], d["bias"], d["residual"], out_dtype=torch.float16), d)


@pytest.mark.parametrize("out", FLOATS, ids=str)
@pytest.mark.parametrize("m,n,pitch,at", [(1, 100, 100, 0), (9, 100, 112, 0), (40, 99, 99, 0), (200, 128, 128, 0), (200, 128, 129, 1), (300, 250, 256, 8), (300, 256, 512, 3)])
def test_outputs_of_the_callers(m, n, pitch, at, out):
    """Rows anywhere: nothing between or behind them is written; the residual may be the output."""
    from tennis_b200 import ops
    d = case(m, n, 272, out, m)
    room = torch.full((m * pitch + at + 64,), 7.0, dtype=out, device="cuda")
    y = room[at:].as_strided((m, n), (pitch, 1))
    y.copy_(d["residual"])
    got = ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], d["bias"], y, out=y)
    assert got is y
    check(got, d)
    written = torch.zeros_like(room, dtype=torch.bool)
    written[at:].as_strided((m, n), (pitch, 1)).fill_(True)
    assert (room[~written] == 7.0).all()


def test_shapes_and_scales():
    """More than two dimensions, transposed weights, one scale for all rows, broadcast rows."""
    from tennis_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    x = int8(2 * 5 * 7, 48, g, pitch=64).as_strided((2, 5, 7, 48), (35 * 64, 7 * 64, 64, 1))
    w = int8(48, 24, g).t()
    ws = torch.rand(24, device="cuda", generator=g) * 1e-3
    for xs in (torch.rand((2, 5, 7), device="cuda", generator=g), torch.full((1,), 0.25, device="cuda")):
        got = ops.inner_prod_quantized(x, xs, w, ws)
        assert got.shape == (2, 5, 7, 24) and got.dtype == torch.float32
        want, bound = plain.inner_prod(x.reshape(70, 48).cpu().numpy(), xs.expand(2, 5, 7).cpu().numpy().reshape(-1), w.cpu().numpy(), ws.cpu().numpy())
        plain.assert_close(got.view(70, 24), want, bound, torch.float32)
    one = int8(1, 48, g).expand(20, 48)
    got = ops.inner_prod_quantized(one, torch.rand(1, device="cuda"), w, ws)
    assert (got == got[0]).all()
    vec = ops.inner_prod_quantized(one[0], torch.ones(1, device="cuda"), w, ws)
    assert vec.shape == (24,)


@pytest.mark.parametrize("k", [131071, 131056])
def test_largest_sums(k):
    """k at its limit and every product the largest there is: -128 x -128 and -128 x 127."""
    from tennis_b200 import ops
    for m in (1, 20, 200):
        x = torch.full((m, (k + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :k]
        w = torch.full((70, (k + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :k]
        w[35:] = 127
        got = ops.inner_prod_quantized(x, torch.ones(m, device="cuda"), w, torch.ones(70, device="cuda"))
        want = torch.tensor([float(np.float32(k * 16384))] * 35 + [float(np.float32(-k * 128 * 127))] * 35, device="cuda")
        assert torch.equal(got, want.expand(m, 70))


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 300, 1000), (1, 64, 16), (2, 300, 4096), (3, 77, 333), (4, 128, 8192), (8, 1000, 2048), (11, 256, 130), (16, 512, 16384), (33, 300, 512), (150, 200, 300)])
def test_floating_rows(dtype, m, n, k):
    """Bit for bit what quantize_rows and the product on its result give; rows of zeros and NaN as that says."""
    from tennis_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x = (torch.randn((m, k), device="cuda", generator=g) * 2).to(dtype)
    if m > 2:
        x[1] = 0
        x[2, k // 3] = float("nan")
    d = case(m, n, k, dtype, 5)
    q, s = ops.quantize_rows(x)
    for rows in (x, torch.cat([x, x], 1)[:, :k], torch.cat([x[:, :1], x], 1)[:, 1:]):
        got = ops.inner_prod_quantized(rows, None, d["w"], d["ws"], d["bias"], d["residual"])
        want = ops.inner_prod_quantized(q, s, d["w"], d["ws"], d["bias"], d["residual"], out_dtype=dtype)
        assert got.dtype == dtype and torch.equal(got.nan_to_num(-5.0), want.nan_to_num(-5.0))
        assert m <= 2 or (torch.isnan(got[2]).all() and not torch.isnan(got[0]).any())


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("k", [24, 1000, 4096, 20000, 40000])
def test_one_floating_row(dtype, k):
    """The row that is quantized inside the product: ordinary, of zeros, with a NaN, with an infinity, near the type's largest, misaligned."""
    from tennis_b200 import ops
    d = case(1, 300, k, dtype, 7, residual=False)
    g = torch.Generator(device="cuda").manual_seed(k)
    room = torch.randn(k + 1, device="cuda", generator=g).to(dtype)
    for at in (0, 1):
        for spoil in (None, "zero", "nan", "inf", "large"):
            x = room.clone()[at:at + k].view(1, k)
            if spoil == "zero":
                x.zero_()
            elif spoil == "nan":
                x[0, k // 2] = float("nan")
            elif spoil == "inf":
                x[0, k - 1] = -float("inf")
            elif spoil == "large":
                x.mul_(0.0).add_(torch.finfo(dtype).max)
            q, s = ops.quantize_rows(x)
            want = ops.inner_prod_quantized(q, s, d["w"], d["ws"], d["bias"], out_dtype=dtype)
            got = ops.inner_prod_quantized(x, None, d["w"], d["ws"], d["bias"])
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(3.0), want.nan_to_num(3.0))
            assert torch.isnan(got).all() == (spoil == "nan")


def test_far_offsets():
    """Outputs and operands whose offsets pass 32 bits, of elements and of bytes."""
    from tennis_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    for m in (3, 150):
        pitch = ((1 << 32) // (m - 1) + 64) // 64 * 64
        d = case(m, 40, 64, torch.bfloat16, 1, residual=False)
        x = torch.empty((m - 1) * pitch + 64, dtype=torch.int8, device="cuda").as_strided((m, 64), (pitch, 1))
        x.copy_(d["x"])
        y = torch.empty((m - 1) * pitch + 64, dtype=torch.bfloat16, device="cuda").as_strided((m, 40), (pitch, 1))
        check(ops.inner_prod_quantized(x, d["xs"], d["w"], d["ws"], d["bias"], out=y), d)


def test_streams_and_graphs():
    """Two graphs of the same layer and an eager call on a third stream, all at once: no call uses another's memory."""
    from tennis_b200 import ops
    for m in (1, 16, 200):
        g = torch.Generator(device="cuda").manual_seed(3)
        d = case(m, 512, 1024, torch.float32, 3, residual=False)
        xs = [torch.randn((m, 1024), device="cuda", generator=g) for _ in range(3)]
        want = [ops.inner_prod_quantized(x, None, d["w"], d["ws"], d["bias"]) for x in xs]
        graphs, outs = [], []
        for x in xs[:2]:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = x
                for _ in range(4):
                    y = ops.inner_prod_quantized(x, None, d["w"], d["ws"], d["bias"])
            graphs.append(graph)
            outs.append(y)
        streams = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        for _ in range(10):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
            eager = ops.inner_prod_quantized(xs[2], None, d["w"], d["ws"], d["bias"], stream=streams[2])
        torch.cuda.synchronize()
        for got, ref in zip(outs + [eager], want):
            assert torch.equal(got, ref)


def test_operands_that_the_tensor_cores_cannot_read():
    from tennis_b200 import _lib, ops
    d = case(20, 64, 100, torch.float32, 1, x_pitch=100)
    with pytest.raises(_lib.TsbError, match="16 bytes"):
        ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], kernel=_lib.KERNEL_TCGEN05)
    ops.inner_prod_status()


@pytest.mark.parametrize("lead", [(5,), (2, 3), (1, 2, 2)])
def test_ordinary_and_general_calls_agree(lead):
    """The module for ordinary calls and the Python behind it give the same tensors, for each operator and type."""
    from tennis_b200 import ops
    here = dict(stream=torch.cuda.current_stream())
    g = torch.Generator(device="cuda").manual_seed(1)
    for dtype in FLOATS:
        x = torch.randn(lead + (96,), device="cuda", generator=g).to(dtype)
        w, ws = ops.quantize_rows(torch.randn((40, 96), device="cuda", generator=g))
        bias, res = torch.randn(40, device="cuda", generator=g), torch.randn(lead + (40,), device="cuda", generator=g)
        for one, other in zip(ops.quantize_rows(x), ops.quantize_rows(x, **here)):
            assert torch.equal(one, other) and one.stride() == other.stride()
        q, s = ops.quantize_rows(x)
        for args in ((x, None, w, ws), (x, None, w, ws, bias), (q, s, w, ws, bias, res, 3), (q, s.flatten()[:1].contiguous(), w, ws), (q, s, w, ws, None, None, 2, 0.1)):
            one, other = ops.inner_prod_quantized(*args), ops.inner_prod_quantized(*args, **here)
            assert torch.equal(one, other) and one.dtype == other.dtype and one.shape == other.shape == lead + (40,)
        assert torch.equal(ops.inner_prod_quantized(q, s, w, ws, bias, res, 1, residual_after_activation=True),
                           ops.inner_prod_quantized(q, s, w, ws, bias, res, 1, residual_after_activation=True, **here))
        image = torch.randn((2, 6, 5, 48), device="cuda", generator=g).to(dtype)
        gamma, beta = torch.randn(48, device="cuda", generator=g), torch.randn(48, device="cuda", generator=g)
        for kw in (dict(), dict(gamma=gamma, beta=beta, eps=1e-3, activation=2, leaky=0.2), dict(out_dtype=torch.int8, requant_scales=[9.0, 11.0]), dict(out_dtype=dtype)):
            one, other = ops.group_norm_nhwc(image, 6, **kw), ops.group_norm_nhwc(image, 6, **kw, **here)
            assert torch.equal(one, other) and one.dtype == other.dtype


class Nothing:
    """In the place of the module of ordinary calls: takes no call, and counts those that come."""

    def __init__(self):
        self.calls = 0

    def __getattr__(self, name):
        def take(*args):
            self.calls += 1
        return take


@pytest.mark.parametrize("lead", [(), (1,), (5,), (40,), (2, 3), (3, 1, 15), (1, 2, 2)])
@pytest.mark.parametrize("k,n", [(96, 40), (33, 37), (16, 1)])
def test_the_module_of_ordinary_calls_and_the_general_way(monkeypatch, lead, k, n):
    """The same tensors by both, for each operator, type and number of dimensions; on a stream and with outputs of the caller's too."""
    from tennis_b200 import ops
    native, nothing = ops._ordinary(), Nothing()

    def both(call, *args, **kw):
        monkeypatch.setattr(ops, "_native", native)
        one = call(*args, **kw)
        monkeypatch.setattr(ops, "_native", nothing)
        before = nothing.calls
        other = call(*args, **kw)
        assert nothing.calls == before + 1
        elsewhere = call(*args, stream=torch.cuda.current_stream(), **kw)
        assert nothing.calls == before + 2
        for a, b, c in zip(*(v if isinstance(v, tuple) else (v,) for v in (one, other, elsewhere))):
            assert torch.equal(a, b) and torch.equal(a, c) and a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() == c.stride()
        return one

    g = torch.Generator(device="cuda").manual_seed(1)
    for dtype in FLOATS:
        x = torch.randn(lead + (k,), device="cuda", generator=g).to(dtype)
        w, ws = both(ops.quantize_rows, torch.randn((n, k), device="cuda", generator=g))
        bias = torch.randn(n, device="cuda", generator=g)
        q, s = both(ops.quantize_rows, x)
        one = s.flatten()[:1].contiguous()
        for out in FLOATS:
            res = torch.randn(lead + (n,), device="cuda", generator=g).to(out)
            for args, kw in (((x, None, w, ws), {}), ((x, None, w, ws, bias, res), {}), ((q, s, w, ws, bias, res, 3), {}), ((q, one, w, ws), {}), ((q, s, w, ws, None, None, 2, 0.1), {}),
                             ((q, s, w, ws, bias, res, 4), dict(residual_after_activation=True)), ((x, None, w.contiguous(), ws, bias), {})):
                y = both(ops.inner_prod_quantized, *args, out_dtype=out, **kw)
                assert y.dtype == out and y.shape == lead + (n,)
                room = torch.empty_like(y)
                assert ops.inner_prod_quantized(*args, out_dtype=out, out=room, **kw) is room and torch.equal(room, y)
        assert both(ops.inner_prod_quantized, x, None, w, ws).dtype == dtype and both(ops.inner_prod_quantized, q, s, w, ws).dtype == torch.float32
    for dtype in FLOATS:
        image = torch.randn((2,) + lead + (5, 3 * n), device="cuda", generator=g).to(dtype)
        gamma, beta = torch.randn(3 * n, device="cuda", generator=g), torch.randn(3 * n, device="cuda", generator=g)
        for kw in (dict(), dict(gamma=gamma, beta=beta, eps=1e-3, activation=2, leaky=0.2), dict(out_dtype=torch.int8, requant_scales=[9.0, 11.0]),
                   dict(gamma=gamma, out_dtype=torch.int8, requant_scales=[9.0]), dict(beta=beta, out_dtype=dtype, activation=3)):
            y = both(ops.group_norm_nhwc, image, 3, **kw)
            assert y.shape == image.shape[:-1] + (ops.padded_channels(3 * n) if "requant_scales" in kw else 3 * n,)


def test_refusals():
    from tennis_b200 import ops
    d = case(6, 32, 64, torch.float32, 1)
    x, xs, w, ws, bias, res = (d[v] for v in ("x", "xs", "w", "ws", "bias", "residual"))
    call = ops.inner_prod_quantized
    for bad in (lambda: call(x.float(), xs, w, ws), lambda: call(x, None, w, ws), lambda: call(x.double(), None, w, ws), lambda: call(x, xs, w.float(), ws),
                lambda: call(x, xs, w[0], ws), lambda: call(x[:, :48], xs, w, ws), lambda: call(x, xs[:5], w, ws), lambda: call(x, xs.double(), w, ws),
                lambda: call(x, xs, w, ws[:31]), lambda: call(x, xs, w, ws, bias[:31]), lambda: call(x, xs, w, ws, bias.half()), lambda: call(x, xs, w, ws, bias, res.half()),
                lambda: call(x, xs, w, ws, bias, res[:, :31]), lambda: call(x, xs, w, ws, out_dtype=torch.int8), lambda: call(x, xs, w, ws, out=res.t()),
                lambda: call(x, xs, w, ws, out=res, out_dtype=torch.float16), lambda: call(x, xs, w.cpu(), ws), lambda: call(x[:, :0], xs, w[:, :0], ws)):
        with pytest.raises(ops.EjectionException, match="Check failed"):
            bad()
    with pytest.raises(RuntimeError, match="activation 9"):
        call(x, xs, w, ws, activation=9)


def test_numbers_beyond_an_argument():
    """Numbers of which an int's 32 bits would be valid ones."""
    from tennis_b200 import ops
    d = case(6, 32, 64, torch.float32, 1)
    for bad in (1 << 32, (1 << 32) + 1, -(1 << 32)):
        with pytest.raises((struct.error, RuntimeError)):
            ops.inner_prod_quantized(d["x"], d["xs"], d["w"], d["ws"], activation=bad)
        with pytest.raises((struct.error, RuntimeError)):
            ops.group_norm_nhwc(torch.ones((1, 2, 2, 16), device="cuda"), 4, activation=bad)


def test_empty():
    from tennis_b200 import ops
    w, ws = torch.ones((8, 16), dtype=torch.int8, device="cuda"), torch.ones(8, device="cuda")
    assert ops.inner_prod_quantized(torch.empty((0, 16), device="cuda"), None, w, ws).shape == (0, 8)
    assert ops.inner_prod_quantized(torch.ones((3, 16), device="cuda"), None, w[:0], ws[:0]).shape == (3, 0)
