"""inner_prod_mxfp4 against the product in 64 bits, at sizes, layouts and epilogues where it can go wrong."""
import numpy as np
import pytest
import torch

import int8_layers as int8
import mxfp4_layers as plain

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def rows(m, k, gen, around=127, spread=3, pitch=None, at=0):
    """A 4-bit matrix of all codes, rows `pitch` bytes apart, with scales 2^(around - 127 + 0..spread - 1)."""
    groups = (k + 31) // 32
    codes = torch.randint(0, 16, (m, groups * 32), dtype=torch.uint8, device="cuda", generator=gen)
    codes[:, k:] = 0
    pitch = pitch or groups * 16
    room = torch.zeros(m * pitch + at, dtype=torch.uint8, device="cuda")
    q = room[at:].as_strided((m, groups * 16), (pitch, 1))
    q.copy_(codes[:, 0::2] | codes[:, 1::2] << 4)
    scales = torch.randint(around, around + spread, (m, groups), dtype=torch.uint8, device="cuda", generator=gen)
    from tennis_b200 import ops
    return q.view(torch.float4_e2m1fn_x2), ops.mxfp4_scale_tiles(scales)


def case(m, n, k, out, seed=0, residual=True, bias=True, around=127, spread=3, **layout):
    """Sums are multiples of a quarter of the smallest two scales' product and, of scales that spread over two powers of two each, below 2^24
    of that for k up to 8192 (36 * 16 * 4 * 8192 = 2^24.2 is reached by no random sum): exact in fp32 in any order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, xs = rows(m, k, g, around, spread, layout.get("x_pitch"), layout.get("x_at", 0))
    w, ws = rows(n, k, g, 127 - int(np.log2(k) / 2) - 4, spread, layout.get("w_pitch"), layout.get("w_at", 0))
    return dict(x=x, xs=xs, w=w, ws=ws, bias=torch.randn(n, device="cuda", generator=g) if bias else None,
                residual=torch.randn((m, n), device="cuda", generator=g).to(out) if residual else None)


def check(got, d, act=0, leaky=0.0, after=False, exact_sums=True):
    want, bound = plain.inner_prod(plain.decode(d["x"], d["xs"]), plain.decode(d["w"], d["ws"]), plain.numbers(d["bias"]), plain.numbers(d["residual"]), act, leaky, after, exact_sums)
    int8.assert_close(got, want, bound, got.dtype)


def call(d, **kw):
    from tennis_b200 import ops
    return ops.inner_prod_mxfp4(d["x"], d["xs"], d["w"], d["ws"], d["bias"], d["residual"], **kw)


SIZES = [(1, 1, 1), (1, 8, 16), (1, 1000, 2048), (1, 37, 4099), (2, 129, 64), (3, 64, 100), (4, 1024, 1024), (5, 4096, 512), (7, 333, 8192), (8, 250, 1040),
         (9, 65, 333), (16, 1000, 2048), (17, 128, 128), (24, 511, 192), (31, 2048, 272), (32, 96, 4096), (33, 100, 48), (63, 777, 130), (64, 1000, 2048),
         (65, 257, 1000), (100, 130, 4096), (127, 64, 127), (128, 128, 128), (129, 256, 256), (130, 512, 4112), (200, 40, 96), (255, 300, 144), (256, 256, 1024),
         (257, 255, 2048), (300, 1024, 512), (500, 1000, 500), (700, 512, 640), (1000, 96, 64), (1025, 513, 1009), (2049, 64, 32), (4096, 200, 128), (333, 777, 1021),
         (2300, 1300, 400), (6000, 16, 16), (1, 4096, 8192), (12, 5000, 2304), (48, 2000, 96), (2, 19000, 64)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_sizes(m, n, k):
    """Every size with each output type, with and without residual and bias."""
    for i, out in enumerate(FLOATS):
        d = case(m, n, k, out, m + n + k + i, residual=i != 1, bias=i != 2)
        got = call(d, out_dtype=out)
        assert got.dtype == out and got.shape == (m, n)
        check(got, d)


@pytest.mark.parametrize("m,n,k", [(1, 200, 512), (12, 200, 512), (40, 200, 500), (150, 200, 512), (400, 520, 1024)])
@pytest.mark.parametrize("act,leaky", [(0, 0.0), (1, 0.0), (2, 0.1), (2, -0.25), (3, 0.0), (4, 0.0)])
def test_activations(m, n, k, act, leaky):
    for out in FLOATS:
        for after in (False, True):
            d = case(m, n, k, out, act)
            check(call(d, activation=act, leaky=leaky, out_dtype=out, residual_after_activation=after), d, act, leaky, after)


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
            got = ops.inner_prod_mxfp4(torch.zeros_like(d["x"].view(torch.uint8)), d["xs"], d["w"], d["ws"], bias, activation=act, out_dtype=out).cpu()
            # fp32: silu by 8 half steps of its value, gelu by 24 of 1; one rounding to 16 bits; 10^-17 as plain.activation's quotient
            torch.testing.assert_close(got.double(), want.to(out).double().expand(m, n), rtol=2 * torch.finfo(out).eps + 8 * plain.EPS32,
                                       atol=24 * plain.EPS32 if act == 4 else 1e-17, equal_nan=True)


@pytest.mark.parametrize("out", FLOATS, ids=str)
def test_gelu_between(out):
    """gelu from -7 to 7: within |v| 2^-22 (the formula of 16-bit results is off by 1.5e-7 |v| / 2, its fp32 steps by some 2^-23 |v|; erff's form by as much) and one rounding."""
    from tennis_b200 import ops
    n = 4096
    bias = torch.linspace(-7.0, 7.0, n, device="cuda")
    v = bias.double().cpu()
    want = 0.5 * v * torch.erfc(-v * 0.5 ** 0.5)
    for m in (1, 40, 300):
        d = case(m, n, 48, out, 3)
        got = ops.inner_prod_mxfp4(torch.zeros_like(d["x"].view(torch.uint8)), d["xs"], d["w"], d["ws"], bias, activation=4, out_dtype=out).cpu().double()
        room = v.abs() * 2.0 ** -22 + (0.0 if out == torch.float32 else want.abs() * torch.finfo(out).eps / 2 + (2.0 ** -25 if out == torch.float16 else 0.0))
        assert ((got - want).abs() <= room).all()


@pytest.mark.parametrize("m", [1, 6, 30, 60, 140, 700])
def test_kernels_agree(m):
    """Exact sums: the kernels have the same bits, whatever rows are computed with a row."""
    from tennis_b200 import _lib, ops
    d = case(m, 330, 1056, torch.float32, m)
    args = (d["x"], d["xs"], d["w"], d["ws"], d["bias"])
    got = ops.inner_prod_mxfp4(*args, d["residual"], _lib.ACT_SILU)
    assert torch.equal(got, ops.inner_prod_mxfp4(*args, d["residual"], _lib.ACT_SILU, kernel=_lib.KERNEL_DIRECT))
    for _ in range(3):
        assert torch.equal(got, ops.inner_prod_mxfp4(*args, d["residual"], _lib.ACT_SILU))
    if m >= 140:
        some = (d["x"][:128], d["xs"][:1])
        assert torch.equal(got[:128], ops.inner_prod_mxfp4(*some, *args[2:], d["residual"][:128], _lib.ACT_SILU))


@pytest.mark.parametrize("m,n,k", [(4096, 2560, 2048), (2500, 2304, 4096), (9472, 256, 4096), (2049, 4097, 2176), (2430, 2432, 8192), (4097, 2080, 1920)])
def test_large_products(m, n, k):
    """Sizes of many tiles a multiprocessor, of one and of two CTAs: exact sums, so a product of doubles has the very bits."""
    from tennis_b200 import ops
    d = case(m, n, k, torch.float32, m, residual=False)
    x, w = ops.dequantize_rows_mxfp4(d["x"], d["xs"]).double(), ops.dequantize_rows_mxfp4(d["w"], d["ws"]).double()
    want = (x @ w.t()).float() + d["bias"]
    for out in FLOATS:
        assert torch.equal(call(d, out_dtype=out), want.to(out))
    r = torch.randn((m, n), device="cuda", dtype=torch.bfloat16)
    assert torch.equal(ops.inner_prod_mxfp4(d["x"], d["xs"], d["w"], d["ws"], d["bias"], r, out_dtype=torch.bfloat16), (want + r.float()).bfloat16())
    ops.inner_prod_mxfp4_status()


@pytest.mark.parametrize("m,n,k", [(1, 500, 4096), (20, 300, 8192), (50, 260, 1500), (200, 300, 4096), (900, 1100, 8192)])
def test_scales_of_any_size(m, n, k):
    """Scales over twenty powers of two: sums are rounded.  As a whole they are as near as fp32 sums of k / 64 steps are, each off by up to 2^-23
    of a sum like the last one or smaller, were all of one sign: k / 64 * 2^-23 of the result's root mean square."""
    d = case(m, n, k, torch.float32, k, spread=20, around=117)
    got = call(d)
    check(got, d, exact_sums=False)
    want = plain.decode(d["x"], d["xs"]) @ plain.decode(d["w"], d["ws"]).T
    off = plain.numbers(got) - plain.numbers(d["bias"]) - plain.numbers(d["residual"]) - want
    assert np.sqrt((off ** 2).mean()) <= (k / 64 + 8) * 2.0 ** -23 * np.sqrt((want ** 2).mean()) + 2.0 ** -22


@pytest.mark.parametrize("m", [1, 20, 50, 200, 900])
def test_scales_at_the_ends(m):
    """Scales whose product leaves fp32 or comes back to it, zero codes under any scale, and groups that are not finite: NaN in their row and
    column alone."""
    from tennis_b200 import ops
    n, k = 300, 256
    g = torch.Generator(device="cuda").manual_seed(m)
    d = case(m, n, k, torch.float32, m, residual=False, bias=False)
    xs, ws = torch.full((m, 8), 240, dtype=torch.uint8, device="cuda"), torch.full((n, 8), 5, dtype=torch.uint8, device="cuda")
    d["xs"], d["ws"] = ops.mxfp4_scale_tiles(xs), ops.mxfp4_scale_tiles(ws)
    check(call(d), d)                                         # 2^113 times 2^-122
    xs[:, 3], ws[:, 5] = 255, 255
    xs[m // 2, 3], xs[:m // 2, 3], xs[m // 2 + 1:, 3] = 255, 240, 240
    ws[:, 5] = 5
    ws[7, 5] = ws[n - 1, 5] = 255
    d["xs"], d["ws"] = ops.mxfp4_scale_tiles(xs), ops.mxfp4_scale_tiles(ws)
    got = call(d).cpu()
    want = torch.from_numpy(plain.decode(d["x"], d["xs"]) @ plain.decode(d["w"], d["ws"]).T)
    assert torch.equal(got.isnan(), want.isnan()) and got.isnan().sum() == n + 2 * (m - 1)
    assert torch.equal(got.nan_to_num(nan=0.0).double(), want.nan_to_num(nan=0.0))
    xs.fill_(254), ws.fill_(250)                              # 2^127 times 2^123
    d["xs"], d["ws"] = ops.mxfp4_scale_tiles(xs), ops.mxfp4_scale_tiles(ws)
    d["x"], d["w"] = d["x"].view(torch.uint8).clone(), d["w"].view(torch.uint8).clone()
    d["x"][:, :] = 0x22                                       # ones
    d["w"][:, :] = 0x22
    d["w"][::2] = 0
    got = call(d)
    assert (got[:, ::2] == 0).all() and (got[:, 1::2] == float("inf")).all()
    del g


@pytest.mark.parametrize("m,n,k", [(1, 300, 200), (20, 300, 512), (60, 128, 130), (300, 260, 640)])
def test_layouts(m, n, k):
    """Rows a pitch apart and rows that start anywhere, residuals likewise, more dimensions, results into room of the caller's and into the residual."""
    from tennis_b200 import ops
    row = (k + 31) // 32 * 16
    for out in FLOATS:
        want = None
        for layout in (dict(), dict(x_pitch=row + 16, w_pitch=row + 48), dict(x_pitch=row + 1, w_pitch=row + 3, x_at=1, w_at=5), dict(w_at=8), dict(x_at=2, x_pitch=row + 16)):
            d = case(m, n, k, out, 5, **layout)
            got = call(d, out_dtype=out)
            check(got, d)
            assert want is None or torch.equal(got, want)
            want = got
        d = case(m, n, k, out, 5)
        r = d["residual"]
        wide, more = (torch.full((m, n + 11), 5.0, dtype=out, device="cuda") for _ in range(2))
        for at in (0, 1, 8):
            to, there = wide[:, at:at + n], more[:, at:at + n]
            wide.fill_(5.0)
            there.copy_(r)
            assert call(d, out=to) is to and torch.equal(to, want) and (wide[:, :at] == 5.0).all() and (wide[:, at + n:] == 5.0).all()
            assert torch.equal(call(dict(d, residual=there), out_dtype=out), want)
            assert call(dict(d, residual=there), out=there) is there and torch.equal(there, want)
        one = r[:1].expand(m, n)
        got = ops.inner_prod_mxfp4(d["x"], d["xs"], d["w"], d["ws"], d["bias"], one, out_dtype=out)
        check(got, dict(d, residual=one))
        if m % 20 == 0:
            x = d["x"].view(torch.uint8).view(4, m // 4, row)
            assert torch.equal(ops.inner_prod_mxfp4(x, d["xs"], d["w"], d["ws"], d["bias"], r.view(4, m // 4, n), out_dtype=out), want.view(4, m // 4, n))
        x = d["x"].view(torch.uint8)[:1].expand(m, row)       # one row for all
        xs = ops.mxfp4_scale_tiles(torch.full((m, row // 16), 127, dtype=torch.uint8, device="cuda"))
        got = ops.inner_prod_mxfp4(x, xs, d["w"], d["ws"], out_dtype=out)
        assert torch.equal(got, got[:1].expand(m, n))
        check(got, dict(x=x, xs=xs, w=d["w"], ws=d["ws"], bias=None, residual=None))


@pytest.mark.parametrize("m,n,k", [(1, 300, 32), (1, 4096, 4096), (1, 100, 1111), (2, 500, 777), (5, 2048, 8192), (8, 64, 96), (9, 333, 500), (30, 1024, 2048), (33, 200, 100), (64, 640, 4096), (130, 130, 130),
                                   (600, 512, 1000)])
def test_floating_rows(m, n, k):
    """The same bits as a call of quantize_rows_mxfp4 in front, of every type, also of rows that start anywhere."""
    from tennis_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    for dtype in FLOATS:
        d = case(1, n, k, dtype, 3)
        wide = (torch.randn((m, k + 9), device="cuda", generator=g) * torch.exp2(torch.randint(-3, 4, (m, 1), device="cuda", generator=g).float())).to(dtype)
        for x in (wide[:, :k].contiguous(), wide[:, :k], wide[:, 1:k + 1], wide[:, 8:k + 8], wide[:1, :k].expand(m, k)):
            q, s = ops.quantize_rows_mxfp4(x)
            for out in FLOATS:
                r = torch.randn((m, n), device="cuda", generator=g).to(out)
                got = ops.inner_prod_mxfp4(x, None, d["w"], d["ws"], d["bias"], r, 3, out_dtype=out)
                assert torch.equal(got, ops.inner_prod_mxfp4(q, s, d["w"], d["ws"], d["bias"], r, 3, out_dtype=out))
        assert ops.inner_prod_mxfp4(x, None, d["w"], d["ws"]).dtype == dtype
        x = wide[:, :k].clone()
        x[m // 2, k // 2] = float("nan")
        got = ops.inner_prod_mxfp4(x, None, d["w"], d["ws"]).isnan()
        assert got[m // 2].all() and got.sum() == n


@pytest.mark.parametrize("m", [1, 24, 300])
def test_norm_and_products_together(m):
    """A block of a network in 4 bits, as it runs: norm of the residual stream, two products with an activation between them, the stream carried on;
    the same with int8 rows beside it."""
    from tennis_b200 import _lib, ops
    k, n = 512, 1408
    g = torch.Generator(device="cuda").manual_seed(m)
    x, stream = (torch.randn((m, k), device="cuda", generator=g).bfloat16() for _ in range(2))
    gamma = torch.rand(k, device="cuda", generator=g) + 0.5
    up, down = torch.randn((n, k), device="cuda", generator=g) / k ** 0.5, torch.randn((k, n), device="cuda", generator=g) / n ** 0.5
    v, h64 = plain.rms_norm(x, gamma, stream)

    def block(quantize_w, product, fmt, form):
        (wu, su), (wd, sd) = quantize_w(up), quantize_w(down)
        q, s, h = ops.rms_norm(x, gamma, stream, out_dtype=fmt)
        t = product(q, s, wu, su, activation=_lib.ACT_SILU, out_dtype=torch.bfloat16)
        y = product(t, None, wd, sd, residual=h)
        a = form(v.astype(np.float64)) @ form(plain.numbers(up)).T
        assert int8_close(t, a / (1 + np.exp(-a)))
        assert int8_close(y, form(plain.numbers(t)) @ form(plain.numbers(down)).T + plain.numbers(h64))
        assert torch.equal(h.cpu(), h64) and y.dtype == torch.bfloat16

    def int8_close(got, want):
        # sums of at most 1408 fp32 steps (2^-23 of a magnitude of at most sqrt(k) results), the steps behind them, one rounding to bf16
        return np.all(np.abs(plain.numbers(got) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -9)

    def as_int8(t):
        q, s = int8.quantize_rows(torch.from_numpy(t))
        return q.astype(np.float64) * s.astype(np.float32).astype(np.float64)[:, None]

    block(ops.quantize_rows_mxfp4, ops.inner_prod_mxfp4, torch.float4_e2m1fn_x2, lambda t: plain.values(*plain.quantize(t)))
    block(ops.quantize_rows, ops.inner_prod_quantized, torch.int8, as_int8)


def test_nothing_to_do():
    from tennis_b200 import ops
    d = case(3, 5, 64, torch.float32)
    assert ops.inner_prod_mxfp4(d["x"][:0], d["xs"][:0], d["w"], d["ws"]).shape == (0, 5)
    assert ops.inner_prod_mxfp4(d["x"], d["xs"], d["w"][:0], d["ws"][:0]).shape == (3, 0)
    assert ops.inner_prod_mxfp4(torch.empty((0, 64), device="cuda"), None, d["w"], d["ws"]).shape == (0, 5)


@pytest.mark.parametrize("m", [1, 30, 300])
def test_streams_and_graphs(m):
    """Another stream than the current one; two captured calls with workspaces of their own, replayed behind each other and at once; two calls at once."""
    from tennis_b200 import ops
    d = case(m, 500, 1000, torch.bfloat16)
    xs = [torch.randn((m, 1000), device="cuda").bfloat16() for _ in range(2)]
    want = [ops.inner_prod_mxfp4(x, None, d["w"], d["ws"], d["bias"]) for x in xs]
    sides = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for x, side in zip(xs, sides):
            side.wait_stream(torch.cuda.current_stream())
            got.append(ops.inner_prod_mxfp4(x, None, d["w"], d["ws"], d["bias"], stream=side))
        for side in sides:
            torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, got = [torch.cuda.CUDAGraph() for _ in xs], []
    for x, graph in zip(xs, graphs):
        with torch.cuda.graph(graph):
            got.append(ops.inner_prod_mxfp4(x, None, d["w"], d["ws"], d["bias"]))
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, side, t in zip(graphs, sides, got):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                t.zero_()
                graph.replay()
        for side in sides:
            torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    from tennis_b200 import _lib, ops
    d = case(4, 40, 64, torch.float32)
    x, xs, w, ws, b, r = d["x"], d["xs"], d["w"], d["ws"], d["bias"], d["residual"]
    f = torch.zeros((4, 64), device="cuda")
    for call in (lambda: ops.inner_prod_mxfp4(x, None, w, ws), lambda: ops.inner_prod_mxfp4(f, xs, w, ws), lambda: ops.inner_prod_mxfp4(f.double(), None, w, ws),
                 lambda: ops.inner_prod_mxfp4(f[:, :32], None, w, ws), lambda: ops.inner_prod_mxfp4(x[:, :16], xs, w, ws), lambda: ops.inner_prod_mxfp4(x, xs, w.view(torch.int8), ws),
                 lambda: ops.inner_prod_mxfp4(x, xs, w[:, :24], ws), lambda: ops.inner_prod_mxfp4(x, xs, w[0], ws), lambda: ops.inner_prod_mxfp4(x, xs, w.cpu(), ws),
                 lambda: ops.inner_prod_mxfp4(x, xs, w, ws.cpu()), lambda: ops.inner_prod_mxfp4(x, xs, w, ws[..., :2]), lambda: ops.inner_prod_mxfp4(x, xs.view(torch.int8), w, ws),
                 lambda: ops.inner_prod_mxfp4(x, b[:4], w, ws), lambda: ops.inner_prod_mxfp4(x, xs, w, ws, b[:39]), lambda: ops.inner_prod_mxfp4(x, xs, w, ws, b.half()),
                 lambda: ops.inner_prod_mxfp4(x, xs, w, ws, b, r[:, :39]), lambda: ops.inner_prod_mxfp4(x, xs, w, ws, b, r.half()), lambda: ops.inner_prod_mxfp4(x, xs, w, ws, out_dtype=torch.int8),
                 lambda: ops.inner_prod_mxfp4(x, xs, w, ws, out=torch.empty((4, 41), device="cuda")), lambda: ops.inner_prod_mxfp4(x, xs, w, ws, out=torch.empty((40, 4), device="cuda").t())):
        with pytest.raises(ops.EjectionException):
            call()
    for kw, text in ((dict(activation=5), "activation 5"), (dict(activation=-1), "activation -1"), (dict(kernel=9), "kernel 9")):
        with pytest.raises(_lib.TsbError, match=text):
            ops.inner_prod_mxfp4(x, xs, w, ws, **kw)


FIRST = """
import sys, torch
sys.path.insert(0, %r)
from tennis_b200 import ops
dev = torch.device("cuda")
w, ws = torch.zeros((512, 64), dtype=torch.uint8, device=dev), torch.zeros((4, 1, 32, 4, 4), dtype=torch.uint8, device=dev)
w.fill_(0x22), ws.fill_(127)
x, gamma = torch.full((%d, 128), 2.0, device=dev, dtype=torch.bfloat16), torch.ones(128, device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q, s, h = ops.rms_norm(x, gamma, x, 0.0, torch.float4_e2m1fn_x2)
    y = ops.inner_prod_mxfp4(q, s, w, ws)
    z = ops.inner_prod_mxfp4(x, None, w, ws)
    v = ops.dequantize_rows_mxfp4(*ops.quantize_rows_mxfp4(x))
graph.replay()
torch.cuda.synchronize()
assert (y == 128.0).all() and (z == 256.0).all() and (v == 2.0).all() and (h == 4.0).all()
ops.inner_prod_mxfp4_status()
"""


@pytest.mark.parametrize("m", [3, 40, 300])
def test_first_calls_of_a_process_may_be_captured(m):
    import subprocess
    import sys
    from conftest import ROOT
    done = subprocess.run([sys.executable, "-c", FIRST % (ROOT, m)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert done.returncode == 0, done.stdout[-2000:]


def test_kernels_beside_each_other():
    """Calls of every kernel on four streams at once: they share multiprocessors, and their tensor memory."""
    from tennis_b200 import ops
    sizes = [(2048, 2048, 512), (16, 4096, 1024), (128, 4096, 1024), (100, 512, 2048), (1, 1000, 4096), (600, 600, 600), (40, 300, 300), (4096, 512, 256)]
    cases = [case(m, n, k, torch.bfloat16, i) for i, (m, n, k) in enumerate(sizes)]
    want = [call(d, out_dtype=torch.bfloat16) for d in cases]
    streams = [torch.cuda.Stream() for _ in range(4)]
    for round in range(10):
        got = []
        for side in streams:
            side.wait_stream(torch.cuda.current_stream())
        for i, d in enumerate(cases * 2):
            got.append(call(cases[(i * 3 + round) % len(cases)], out_dtype=torch.bfloat16, stream=streams[i % 4]))
        for side in streams:
            torch.cuda.current_stream().wait_stream(side)
        for i, y in enumerate(got):
            assert torch.equal(y, want[(i * 3 + round) % len(cases)])
    ops.inner_prod_mxfp4_status()


def test_a_timed_out_wait_is_reported_once_and_named():
    """No kernel is made to time out: the code that a timed-out wait would leave is looked up on the host (the library decodes it), and a healthy device has none."""
    from tennis_b200 import _lib, ops
    call(case(300, 300, 300, torch.float32))
    ops.inner_prod_mxfp4_status()
    ops.inner_prod_mxfp4_status(torch.device("cuda"), torch.cuda.current_stream())
    with pytest.raises(_lib.TsbError, match="a stage to be loaded"):
        _lib.check(_lib.load().tsb_inner_prod_mxfp4_status_decode(2))


@pytest.mark.parametrize("m,n", [(5, 256), (40, 264), (300, 256), (700, 136)])
def test_what_lies_around_the_result_stays(m, n):
    """Rows above and below y, and columns beside it, at widths that copies write whole and at others."""
    for out in FLOATS:
        for odd in (0, 1):
            d = case(m, n - odd, 640, out, m)
            tall = torch.full((m + 9, n + 16), 7.0, dtype=out, device="cuda")
            to = tall[3:m + 3, 8:8 + n - odd]
            assert torch.equal(call(d, out=to), call(d, out_dtype=out))
            tall[3:m + 3, 8:8 + n - odd] = 7.0
            assert (tall == 7.0).all()


def test_offsets_beyond_32_bits():
    """A result of more than 2^31 values and operands of more than 2^31 bytes: the rows at the end are those of a call for them alone."""
    from tennis_b200 import ops
    d = case(300, 8192, 64, torch.bfloat16, 1, residual=False)
    m = 270000                                                  # 128 rows' tiles of scales again and again, so a row's lie where they should
    x = d["x"].view(torch.uint8)[:128].repeat(m // 128 + 1, 1)[:m]
    xs = d["xs"].view(torch.uint8)[:1].repeat(m // 128 + 1, 1, 1, 1, 1)
    y = ops.inner_prod_mxfp4(x, xs, d["w"], d["ws"], d["bias"], out_dtype=torch.bfloat16)
    assert y.numel() > 2 ** 31
    want = ops.inner_prod_mxfp4(d["x"][:128], d["xs"][:1], d["w"], d["ws"], d["bias"], out_dtype=torch.bfloat16)
    assert torch.equal(y[:128], want) and torch.equal(y[m - m % 128:], want[:m % 128]) and torch.equal(y[128 * 2000:128 * 2001], want)
    del y
    d = case(300, 24, 8192, torch.float32, 2, residual=False)
    m = 128 * 4200
    x = d["x"].view(torch.uint8)[:128].repeat(m // 128, 1)
    xs = d["xs"].view(torch.uint8)[:1].repeat(m // 128, 1, 1, 1, 1)
    assert x.numel() > 2 ** 31
    y = ops.inner_prod_mxfp4(x, xs, d["w"], d["ws"], d["bias"])
    want = ops.inner_prod_mxfp4(d["x"][:128], d["xs"][:1], d["w"], d["ws"], d["bias"])
    assert torch.equal(y.view(-1, 128, 24), want.expand(m // 128, 128, 24))


@pytest.mark.parametrize("m", [1, 20, 50, 200])
def test_scales_at_the_ends_of_operands_off_16_bytes(m):
    """A value under its own scale may lie beyond fp32 where the product does not: every kernel has the sums' very bits.  Sums are multiples of a quarter of the smallest two
    scales' product and, of scales that spread over six powers of two together, below 36 * 256 * 2^6 = 2^19.2 times that: exact in fp32 in any order."""
    from tennis_b200 import _lib, ops
    n, k = 130, 256
    for low, high in ((250, 0), (0, 250), (251, 3), (5, 248)):
        g = torch.Generator(device="cuda").manual_seed(m + low)
        for layout in (dict(), dict(x_at=8), dict(w_at=1), dict(x_pitch=k // 2 + 1, w_pitch=k // 2 + 3)):
            x, _ = rows(m, k, g, pitch=layout.get("x_pitch"), at=layout.get("x_at", 0))
            w, _ = rows(n, k, g, pitch=layout.get("w_pitch"), at=layout.get("w_at", 0))
            xs, ws = (torch.randint(at, at + 4, (count, k // 32), dtype=torch.uint8, device="cuda", generator=g) for at, count in ((low, m), (high, n)))
            xs[m // 2, 3], ws[7, 5] = 255, 255                # (not finite: NaN in their row and column alone)
            xt, wt = ops.mxfp4_scale_tiles(xs), ops.mxfp4_scale_tiles(ws)
            want = torch.from_numpy(plain.decode(x, xt) @ plain.decode(w, wt).T)
            assert want.isnan().sum() == m + n - 1
            for kernel in (_lib.KERNEL_AUTO, _lib.KERNEL_DIRECT):
                got = ops.inner_prod_mxfp4(x, xt, w, wt, kernel=kernel).cpu()
                assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.double().nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
    x, w = (torch.full((count, k // 2), 0x22, dtype=torch.uint8, device="cuda") for count in (m, n))      # ones
    w[::2] = 0
    xt, wt = (ops.mxfp4_scale_tiles(torch.full((count, k // 32), byte, dtype=torch.uint8, device="cuda")) for count, byte in ((m, 254), (n, 250)))
    got = ops.inner_prod_mxfp4(x, xt, w, wt, kernel=_lib.KERNEL_DIRECT)      # 2^127 times 2^123, and times nothing
    assert (got[:, ::2] == 0).all() and (got[:, 1::2] == float("inf")).all()


@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16], ids=str)
def test_gelu_of_short_results_far_below_zero(out):
    """gelu of 16-bit results is off by 2^-15 of itself before it is rounded, below zero too, where it is far smaller than its argument: so by (1 + 2^-8) times that and half a step behind
    it, of fp16's smallest numbers 2^-25.  From v = -13 on; what is below -13.3 is less than 2^-126 and becomes zero."""
    from tennis_b200 import ops
    v = torch.cat([torch.linspace(-13.0, 0.0, 6000), torch.linspace(0.0, 8.0, 2000), -torch.logspace(-6, -1, 180), torch.tensor([-13.4, -16.0, -17.0, -40.0, -1e3, -1e30, 16.0, 1e3, 6e4, 0.0])]).cuda()
    n = v.numel()
    assert n % 8 == 6
    x = v.double().cpu()
    want = 0.5 * x * torch.erfc(-x * 0.5 ** 0.5)
    want[x < -13.3] = 0.0
    room = want.abs() * (torch.finfo(out).eps / 2 + 2.0 ** -15 * (1 + 2.0 ** -8)) + (2.0 ** -25 if out == torch.float16 else 2.0 ** -134)
    for m in (1, 40, 300):
        d = case(m, n, 48, out, 3)
        got = ops.inner_prod_mxfp4(torch.zeros_like(d["x"].view(torch.uint8)), d["xs"], d["w"], d["ws"], v, activation=4, out_dtype=out).cpu().double()
        assert ((got - want).abs() <= room).all(), float(((got - want).abs() / room).max())
