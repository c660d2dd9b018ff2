"""quantize_rows_mxfp4, dequantize_rows_mxfp4 and mxfp4_scale_tiles: every bit against the plain form, at sizes, layouts and values where they can go wrong."""
import numpy as np
import pytest
import torch

import mxfp4_layers as plain

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]
SIZES = [(1, 1), (1, 31), (1, 32), (1, 33), (1, 4096), (2, 64), (3, 100), (5, 127), (7, 128), (31, 129), (32, 96), (33, 160), (127, 200), (128, 256), (129, 255), (130, 1000),
         (255, 32), (257, 8), (300, 416), (640, 64), (1000, 36), (97, 1111), (2, 8191), (1, 16384), (70, 4100)]


def features(m, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((m, k), device="cuda", generator=g) * torch.exp2(torch.randint(-9, 9, (m, (k + 31) // 32), device="cuda", generator=g).repeat_interleave(32, 1)[:, :k].float())
    return x.to(dtype)


def check(x, q, s):
    """q's bytes and every byte of s."""
    codes, scales = plain.quantize(plain.numbers(x.reshape(-1, x.shape[-1])))
    assert q.dtype == torch.float4_e2m1fn_x2 and s.dtype == torch.float8_e8m0fnu
    got = plain.bytes_of(q).reshape(codes.shape[0], -1)
    fine = np.repeat(scales != 255, 16, 1)
    assert np.array_equal(got[fine], plain.pack(codes)[fine])
    assert np.array_equal(plain.bytes_of(s).reshape(-1), plain.tiles(scales))


@pytest.mark.parametrize("m,k", SIZES)
def test_sizes(m, k):
    from tennis_b200 import ops
    for i, dtype in enumerate(FLOATS):
        x = features(m, k, dtype, m + k + i)
        q, s = ops.quantize_rows_mxfp4(x)
        assert q.shape == (m, (k + 31) // 32 * 16) and s.shape == ((m + 127) // 128, (k + 127) // 128, 32, 4, 4)
        check(x, q, s)
        want = plain.decode(q, s)[:, :k]
        for out in FLOATS:
            y = ops.dequantize_rows_mxfp4(q, s, k, out)
            assert y.dtype == out and y.shape == (m, k)
            assert torch.equal(y.cpu(), torch.from_numpy(want).to(out))
        if k % 32 == 0:
            assert torch.equal(ops.dequantize_rows_mxfp4(q, s), y.float() if out == torch.float32 else ops.dequantize_rows_mxfp4(q, s, k))


def test_rounding():
    """Every midpoint between two codes, and the numbers next to it, at scales from one end of fp32 to the other."""
    from tennis_b200 import ops
    v = torch.tensor([6.0, 7.9, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 0.0])
    v = torch.cat([v, torch.nextafter(v, v - 1), torch.nextafter(v, v + 1).clamp(max=7.9999), torch.zeros(16)])
    v = torch.cat([v, -v]).view(4, 32)
    v[1::2, 0] = torch.tensor([6.0, -6.0])
    x = torch.cat([v * 2.0 ** e for e in (-140, -126, -125, -120, -40, -1, 0, 1, 30, 100, 124, 125)])
    check(x, *ops.quantize_rows_mxfp4(x.cuda()))
    for dtype in (torch.float16, torch.bfloat16):
        y = torch.cat([v * 2.0 ** e for e in (-24, -14, -3, 0, 5, 12)]).to(dtype)
        check(y, *ops.quantize_rows_mxfp4(y.cuda()))


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
def test_ends_of_the_range(dtype):
    """Zeros of both signs, the smallest and the largest numbers, infinities and NaN: what is not finite stays within its group."""
    from tennis_b200 import ops
    f = torch.finfo(dtype)
    x = features(6, 200, dtype)
    x[0, :40] = 0.0
    x[0, 3] = -0.0
    x[1, 32:64] = f.tiny * torch.linspace(-1, 1, 32, device="cuda").to(dtype)
    x[2, 64:96] = f.smallest_normal / 1024
    x[3, 5], x[3, 6], x[3, 7] = f.max, -f.max, f.max / 3
    x[4, 33], x[4, 199], x[4, 100] = float("nan"), float("inf"), -float("inf")
    q, s = ops.quantize_rows_mxfp4(x)
    check(x, q, s)
    y = ops.dequantize_rows_mxfp4(q, s, 200).cpu()
    gone = torch.isnan(y[4])
    assert gone[32:64].all() and gone[96:128].all() and gone[192:200].all() and gone.sum() == 72 and torch.isfinite(y[:4]).all() and torch.isfinite(y[5]).all()


def test_every_code_and_scale():
    """256 scales times 16 codes, to each type: one rounding, infinities where it has no number."""
    from tennis_b200 import ops
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    scales = np.arange(256, dtype=np.uint8).reshape(256, 1)
    q = torch.from_numpy(plain.pack(codes)).cuda()
    s = ops.mxfp4_scale_tiles(torch.from_numpy(scales).cuda())
    assert s.dtype == torch.float8_e8m0fnu and np.array_equal(plain.bytes_of(s).reshape(-1), plain.tiles(scales))
    want = torch.from_numpy(plain.values(codes, scales))
    for dtype in FLOATS:
        for packed in (q, q.view(torch.float4_e2m1fn_x2)):
            for t in (s, s.view(torch.uint8)):
                got = ops.dequantize_rows_mxfp4(packed, t, dtype=dtype).cpu()
                assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=0.0, posinf=float("inf"), neginf=-float("inf")), want.float().to(dtype).nan_to_num(
                    nan=0.0, posinf=float("inf"), neginf=-float("inf")))


@pytest.mark.parametrize("k", [32, 100, 512])
def test_layouts(k):
    """Rows a pitch apart, rows that start anywhere, one row for all, transposes, more dimensions, outputs of the caller's with room around them."""
    from tennis_b200 import ops
    for dtype in FLOATS:
        wide = features(70, k + 13, dtype)
        for x in (wide[:, :k], wide[:, 1:k + 1], wide[::3, 8:8 + k], wide[:1, :k].expand(70, k), features(k, 70, dtype).t(), features(70, k, dtype).view(7, 10, k),
                  features(1, k, dtype).view(k), features(70, k, dtype).view(2, 5, 7, k).transpose(0, 1)):
            q, s = ops.quantize_rows_mxfp4(x)
            check(x, q, s)
            row = (k + 31) // 32 * 16
            y = ops.dequantize_rows_mxfp4(q, s, k, dtype)
            assert y.shape == x.shape
            for room_dtype in (torch.uint8, torch.float4_e2m1fn_x2):
                for at, pitch in ((0, row + 16), (3, row + 5), (4, row + 12)):
                    m = x.numel() // k
                    room = torch.full((m * pitch + 40,), 77, dtype=torch.uint8, device="cuda")
                    to = room[at:].as_strided((m, row), (pitch, 1)).view(room_dtype).view(q.shape)
                    around = torch.ones_like(room, dtype=torch.bool)
                    around[at:].as_strided((m, row), (pitch, 1)).fill_(False)
                    tiles = torch.full(tuple(s.shape), 99, dtype=torch.uint8, device="cuda")
                    got, got_s = ops.quantize_rows_mxfp4(x, out=to, scales=tiles)
                    assert got is to and got_s is tiles and torch.equal(tiles, s.view(torch.uint8)) and torch.equal(to.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8))
                    assert (room[around] == 77).all()
                    assert torch.equal(ops.dequantize_rows_mxfp4(to, tiles, k, dtype), y)
            some = torch.full((m, k + 5), 3.0, dtype=dtype, device="cuda")
            to = some[:, 2:k + 2].unflatten(0, x.shape[:-1]) if x.dim() > 2 else some[:, 2:k + 2] if x.dim() == 2 else some[0, 2:k + 2]
            assert ops.dequantize_rows_mxfp4(q, s, k, out=to) is to and torch.equal(to, y)
            assert (some[:, :2] == 3.0).all() and (some[:, k + 2:] == 3.0).all()


def test_nothing_to_do():
    from tennis_b200 import ops
    for shape in ((0, 64), (3, 0, 64)):
        q, s = ops.quantize_rows_mxfp4(torch.empty(shape, device="cuda"))
        assert q.shape == shape[:-1] + (32,) and s.shape == (0, 1, 32, 4, 4)
        assert ops.dequantize_rows_mxfp4(q, s).shape == shape


def test_streams_and_graphs():
    from tennis_b200 import ops
    x = features(300, 500, torch.bfloat16)
    want = [t.view(torch.uint8) for t in ops.quantize_rows_mxfp4(x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, s = ops.quantize_rows_mxfp4(x, stream=side)
    y = ops.dequantize_rows_mxfp4(q, s, 500, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(q.view(torch.uint8), want[0]) and torch.equal(s.view(torch.uint8), want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gq, gs = ops.quantize_rows_mxfp4(x)
        gy = ops.dequantize_rows_mxfp4(gq, gs, 500)
    x.neg_()
    graph.replay()
    assert torch.equal(gy, -y) and torch.equal(gs.view(torch.uint8), want[1])


def test_refusals():
    from tennis_b200 import ops
    x = features(4, 64, torch.float32)
    q, s = ops.quantize_rows_mxfp4(x)
    for call in (lambda: ops.quantize_rows_mxfp4(x.double()), lambda: ops.quantize_rows_mxfp4(x.int()), lambda: ops.quantize_rows_mxfp4(x[:, :0]), lambda: ops.quantize_rows_mxfp4(x[0, 0]),
                 lambda: ops.quantize_rows_mxfp4(x, out=torch.empty((4, 33), dtype=torch.uint8, device="cuda")), lambda: ops.quantize_rows_mxfp4(x, out=torch.empty((4, 32), device="cuda")),
                 lambda: ops.quantize_rows_mxfp4(x, out=q.cpu()), lambda: ops.quantize_rows_mxfp4(x, scales=s[..., :2]), lambda: ops.quantize_rows_mxfp4(x, scales=s.cpu()),
                 lambda: ops.quantize_rows_mxfp4(x, scales=torch.empty((1, 1, 32, 4, 8), dtype=torch.uint8, device="cuda")[..., ::2]),
                 lambda: ops.quantize_rows_mxfp4(x, scales=torch.empty((1, 2, 32, 4, 4), dtype=torch.uint8, device="cuda")),
                 lambda: ops.dequantize_rows_mxfp4(q, s, 65), lambda: ops.dequantize_rows_mxfp4(q, s, 32), lambda: ops.dequantize_rows_mxfp4(q, s, 0), lambda: ops.dequantize_rows_mxfp4(q, s, -1),
                 lambda: ops.dequantize_rows_mxfp4(q[:, :8], s), lambda: ops.dequantize_rows_mxfp4(x, s), lambda: ops.dequantize_rows_mxfp4(q, s, dtype=torch.float64),
                 lambda: ops.dequantize_rows_mxfp4(q, s, dtype=torch.int8), lambda: ops.dequantize_rows_mxfp4(q, s.view(torch.int8)), lambda: ops.dequantize_rows_mxfp4(q[:, :0], s),
                 lambda: ops.dequantize_rows_mxfp4(q, s, out=torch.empty((4, 63), device="cuda")), lambda: ops.mxfp4_scale_tiles(s), lambda: ops.mxfp4_scale_tiles(x)):
        with pytest.raises(ops.EjectionException):
            call()


def test_long_rows_and_many_rows():
    """Rows of more values than a block's turn, more rows than a grid's dimension, and offsets beyond 2^31 bytes."""
    from tennis_b200 import ops
    x = features(3, 70001, torch.float16)
    check(x, *ops.quantize_rows_mxfp4(x))
    row = features(1, 64, torch.bfloat16)
    m = 40 * 1000 * 1000
    x = row.expand(m, 64)
    q, s = ops.quantize_rows_mxfp4(x)
    one, t = ops.quantize_rows_mxfp4(row)
    assert (q.view(torch.int64) == one.view(torch.int64)).all()
    assert (s.view(torch.int32).view(-1) == t.view(torch.int32).view(-1)[0]).all()
    assert torch.equal(ops.dequantize_rows_mxfp4(q[-5:], s[-1:].clone() if m % 128 == 5 else ops.quantize_rows_mxfp4(x[-5:])[1], 64, torch.bfloat16), ops.dequantize_rows_mxfp4(one, t, 64, torch.bfloat16).expand(5, 64))
    del x, q, s
    y = ops.dequantize_rows_mxfp4(one.expand(m, 32), torch.full(((m + 127) // 128, 1, 32, 4, 4), 127, dtype=torch.uint8, device="cuda"), dtype=torch.bfloat16)
    assert (y == ops.dequantize_rows_mxfp4(one, torch.full((1, 1, 32, 4, 4), 127, dtype=torch.uint8, device="cuda"), dtype=torch.bfloat16)).all()
