"""rms_norm: every bit against the plain form in 64 bits, at sizes, layouts and values where it can go wrong."""
import numpy as np
import pytest
import torch

import int8_layers as int8
import mxfp4_layers as plain

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]
FP4 = torch.float4_e2m1fn_x2
SIZES = [(1, 1), (1, 16), (2, 31), (3, 32), (1, 100), (5, 127), (7, 256), (31, 257), (33, 512), (130, 513), (2, 1000), (129, 1024), (300, 64), (700, 33), (1, 4096), (310, 2048), (4, 4104), (3, 8191),
         (1, 8192), (300, 8192), (2, 16384), (5, 16392), (1, 32768), (2, 32777), (3, 40000), (2, 70001)]


def features(m, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((m, k), device="cuda", generator=g)
    x *= torch.where(torch.rand(k, device="cuda", generator=g) < 0.02, 12.0, 1.0)
    return (x * torch.exp2(torch.randint(-4, 5, (m, 1), device="cuda", generator=g).float())).to(dtype)


def weights(k, seed=1):
    return torch.empty(k, device="cuda").normal_(1.0, 0.3, generator=torch.Generator(device="cuda").manual_seed(seed))


def bits(t):
    return t.contiguous().view(torch.uint8) if t.dtype in (FP4, torch.float8_e8m0fnu) else t


def check(got, x, gamma, residual, out, eps=1e-6):
    """All results of a call.  64-bit sums in another order are off by 2^-45 or so: the rounded reciprocal deviation differs once in a million rows."""
    v, h = plain.rms_norm(x, gamma, residual, eps)
    got = got if isinstance(got, tuple) else (got,)
    if residual is not None:
        assert got[-1].dtype == x.dtype and torch.equal(got[-1].cpu().isnan(), h.isnan()) and torch.equal(got[-1].cpu().nan_to_num(nan=-7.0), h.nan_to_num(nan=-7.0))
        got = got[:-1]
    v = torch.from_numpy(v)
    if out == torch.int8:
        q, s = int8.quantize_rows(v)
        assert got[0].dtype == torch.int8 and got[1].dtype == torch.float32
        assert np.array_equal(got[0].cpu().numpy(), q)
        assert np.array_equal(got[1].cpu().numpy(), s.astype(np.float32), equal_nan=True)
    elif out == FP4:
        codes, scales = plain.quantize(v.double().numpy())
        fine = np.repeat(scales != 255, 16, 1)
        assert got[0].dtype == FP4 and got[1].dtype == torch.float8_e8m0fnu
        assert np.array_equal(plain.bytes_of(got[0])[fine], plain.pack(codes)[fine])
        assert np.array_equal(plain.bytes_of(got[1]).reshape(-1), plain.tiles(scales))
    else:
        assert got[0].dtype == x.dtype and torch.equal(got[0].cpu().nan_to_num(nan=-7.0), v.to(x.dtype).nan_to_num(nan=-7.0)) and torch.equal(got[0].cpu().isnan(), v.isnan())


@pytest.mark.parametrize("m,k", SIZES)
def test_sizes(m, k):
    from tennis_b200 import ops
    for i, dtype in enumerate(FLOATS):
        x, r, gamma = features(m, k, dtype, m + k), features(m, k, dtype, m + k + 1), weights(k)
        for out in (dtype, torch.int8, FP4):
            for residual in (None, r):
                for g in (gamma, None):
                    check(ops.rms_norm(x, g, residual, out_dtype=None if out == dtype and i else out), x, g, residual, out)


def test_shapes_of_results():
    from tennis_b200 import ops
    x, g = features(12, 100, torch.float16), weights(100)
    for shape in ((100,), (12, 100), (3, 4, 100), (2, 3, 2, 100)):
        t = x[0] if len(shape) == 1 else x.view(shape)
        assert ops.rms_norm(t, g).shape == shape
        y, h = ops.rms_norm(t, g, t)
        assert y.shape == h.shape == shape
        q, s = ops.rms_norm(t, g, out_dtype=torch.int8)
        assert q.shape == shape and s.shape == shape[:-1] and (q.stride(-2) % 16 == 0 if len(shape) > 1 else True)
        q, s, h = ops.rms_norm(t, g, t, out_dtype=FP4)
        assert q.shape == shape[:-1] + (64,) and s.shape == (1, 1, 32, 4, 4) and h.shape == shape


@pytest.mark.parametrize("k", [32, 100, 768, 2000, 40000])
def test_layouts(k):
    """Rows a pitch apart, rows that start anywhere, one row for all, more dimensions; results in place and with room around them."""
    from tennis_b200 import ops
    gamma = weights(k + 1)[1:]              # (off 16 bytes)
    for dtype in FLOATS:
        wide, more = features(9, k + 13, dtype), features(9, k + 13, dtype, 5)
        for x, r in ((wide[:, :k], more[:, 8:k + 8]), (wide[:, 1:k + 1], more[:, :k]), (wide[:1, :k].expand(9, k), more[:, :k]), (wide[:, :k], more[:1, 8:k + 8].expand(9, k)),
                     (wide[::3, 8:k + 8].contiguous()[:3], more[::3, :k]), (features(k, 9, dtype).t(), more[:, :k])):
            for out in (dtype, torch.int8, FP4):
                check(ops.rms_norm(x, gamma.contiguous(), r, out_dtype=out), x, gamma, r, out)
                check(ops.rms_norm(x, gamma.clone(), None, out_dtype=out), x, gamma, None, out)
        x, r = wide[:, :k], more[:, 3:k + 3]
        want = ops.rms_norm(x, gamma.contiguous(), r)
        # the sum in the place of the residual, of x; the norm in the place of x and of the residual
        for sum_in, y_in in (("r", None), ("x", None), (None, "x"), (None, "r"), ("r", "x"), ("x", "r")):
            a, b = wide.clone()[:, :k], more.clone()[:, 3:k + 3]
            here = {"x": a, "r": b, None: None}
            y, h = ops.rms_norm(a, gamma.contiguous(), b, sum_out=here[sum_in], out=here[y_in])
            assert torch.equal(y, want[0]) and torch.equal(h, want[1])
            assert (here[sum_in] is None or h is here[sum_in]) and (here[y_in] is None or y is here[y_in])
        y = wide.clone()
        assert torch.equal(ops.rms_norm(y[:, :k], gamma.contiguous(), out=y[:, :k]), ops.rms_norm(x, gamma.contiguous())) and torch.equal(y[:, k:], wide[:, k:])
        # 8 and 4 bits into room of the caller's
        m, row = 9, (k + 31) // 32 * 16
        for out, cols in ((torch.int8, k), (torch.uint8, row)):
            q, s, _ = ops.rms_norm(x, gamma.contiguous(), r, out_dtype=torch.int8 if out == torch.int8 else FP4)
            for at, pitch in ((0, (cols + 31) // 16 * 16), (5, cols + 3), (4, (cols + 7) // 4 * 4)):
                room = torch.full((m * pitch + 64,), 77, dtype=out, device="cuda")
                to = room[at:].as_strided((m, cols), (pitch, 1))
                around = torch.ones_like(room, dtype=torch.bool)
                around[at:].as_strided((m, cols), (pitch, 1)).fill_(False)
                scales = torch.empty(m, device="cuda") if out == torch.int8 else torch.full(tuple(s.shape), 9, dtype=torch.uint8, device="cuda")
                got = ops.rms_norm(x, gamma.contiguous(), r, out=to, scales=scales)
                assert got[0] is to and got[1] is scales and torch.equal(bits(to), bits(q)) and torch.equal(bits(scales), bits(s)) and (room[around] == 77).all()


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
def test_ends_of_the_range(dtype):
    """Rows of zeros (eps alone, and no eps: 0 / 0), of the smallest and the largest numbers, with infinities and NaN: each row is its own."""
    from tennis_b200 import ops
    f = torch.finfo(dtype)
    x = features(8, 300, dtype)
    x[1] = 0.0
    x[2] = f.tiny
    x[3] = f.max
    x[4, 7] = float("inf")
    x[5, 9] = float("nan")
    x[6, 299] = -f.max
    gamma = weights(300)
    for eps in (1e-6, 0.0, 1e30):
        for out in (dtype, torch.int8, FP4):
            check(ops.rms_norm(x, gamma, None, eps, out), x, gamma, None, out, eps)
    y = torch.zeros_like(x)
    y[3] = f.max            # the sum becomes infinite
    check(ops.rms_norm(x, gamma, y), x, gamma, y, dtype)


def test_nothing_to_do():
    from tennis_b200 import ops
    x = torch.empty((0, 64), device="cuda")
    assert ops.rms_norm(x).shape == (0, 64)
    y, h = ops.rms_norm(x, None, x)
    assert y.shape == h.shape == (0, 64)
    q, s = ops.rms_norm(x, out_dtype=torch.int8)
    assert q.shape == (0, 64) and s.shape == (0,)
    q, s = ops.rms_norm(x, out_dtype=FP4)
    assert q.shape == (0, 32) and s.shape == (0, 1, 32, 4, 4)


def test_streams_and_graphs():
    from tennis_b200 import ops
    x, r, g = features(300, 1000, torch.bfloat16), features(300, 1000, torch.bfloat16, 3), weights(1000)
    want = ops.rms_norm(x, g, r, out_dtype=FP4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ops.rms_norm(x, g, r, out_dtype=FP4, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rms_norm(x, g, r, out_dtype=torch.int8)
    x.copy_(features(300, 1000, torch.bfloat16, 9))
    graph.replay()
    check(got, x, g, r, torch.int8)


def last_in_memory(t):
    """t as the last bytes of an allocation."""
    room = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")[-t.numel() * t.element_size():].view(t.dtype).view(t.shape)
    return room.copy_(t)


@pytest.mark.parametrize("k", [8, 64, 264, 320, 520, 1000, 1032, 4104, 8200])
def test_nothing_is_read_behind_the_ends(k):
    """Rows of whole vectors whose scales' tiles, and whose threads, reach beyond them."""
    from tennis_b200 import ops
    for dtype in FLOATS:
        x, r, gamma = (last_in_memory(t) for t in (features(3, k, dtype, k), features(3, k, dtype, k + 1), weights(k)))
        for out in (dtype, torch.int8, FP4):
            check(ops.rms_norm(x, gamma, out_dtype=out), x, gamma, None, out)
            check(ops.rms_norm(x, gamma, r, out_dtype=out), x, gamma, r, out)


def test_many_rows():
    """Offsets beyond 2^31 bytes."""
    from tennis_b200 import ops
    row, g = features(1, 64, torch.bfloat16), weights(64)
    m = 20 * 1000 * 1000
    q, s = ops.rms_norm(row.expand(m, 64), g, out_dtype=torch.int8)
    one, t = ops.rms_norm(row, g, out_dtype=torch.int8)
    assert (q.view(torch.int64) == one.view(torch.int64)).all() and (s == t).all()
    y, h = ops.rms_norm(row.expand(m, 64), g, row.expand(m, 64))
    one, t = ops.rms_norm(row, g, row)
    assert (y.view(torch.int64) == one.view(torch.int64)).all() and (h.view(torch.int64) == t.view(torch.int64)).all()


def test_refusals():
    from tennis_b200 import ops
    x, g = features(4, 64, torch.float32), weights(64)
    for call in (lambda: ops.rms_norm(x.double()), lambda: ops.rms_norm(x[:, :0]), lambda: ops.rms_norm(x[0, 0]), lambda: ops.rms_norm(x, g[:63]), lambda: ops.rms_norm(x, g.half()),
                 lambda: ops.rms_norm(x, g.cpu()), lambda: ops.rms_norm(x, g, x[:3]), lambda: ops.rms_norm(x, g, x.half()), lambda: ops.rms_norm(x, g, x.cpu()),
                 lambda: ops.rms_norm(x, g, out_dtype=torch.float16), lambda: ops.rms_norm(x, g, out_dtype=torch.uint8), lambda: ops.rms_norm(x, g, sum_out=x),
                 lambda: ops.rms_norm(x, g, x, sum_out=x.half()), lambda: ops.rms_norm(x, g, x, sum_out=torch.empty((64, 4), device="cuda").t()), lambda: ops.rms_norm(x, g, scales=g),
                 lambda: ops.rms_norm(x, g, out=torch.empty((4, 63), device="cuda")), lambda: ops.rms_norm(x, g, out=torch.empty((4, 64), device="cuda", dtype=torch.float16)),
                 lambda: ops.rms_norm(x, g, out_dtype=torch.int8, scales=g), lambda: ops.rms_norm(x, g, out_dtype=FP4, scales=g[:4])):
        with pytest.raises(ops.EjectionException):
            call()
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(Exception, match="eps"):
            ops.rms_norm(x, g, eps=eps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_rows_longer_than_2_to_the_30(dtype):
    """One row whose gamma, and of fp32 whose values, lie beyond 2^32 bytes: every result, the end's and the beginning's.  Values are small whole numbers, so the squares'
    sum is exact in 64 bits in any order and the reciprocal deviation is one fp32 number; v is its two fp32 products."""
    from tennis_b200 import ops
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("40 GB of memory")
    k, piece, dev = (1 << 30) + 1_000_003, 1 << 26, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(k)
    x, r = (torch.empty((1, k), dtype=torch.int8, device=dev).random_(-3, 4, generator=g).to(dtype) for _ in range(2))
    gamma = torch.rand(k, device=dev, generator=g).add_(0.5)

    def pieces(total):
        return [slice(at, min(at + piece, total)) for at in range(0, total, piece)]

    for residual in (None, r):
        def h_of(at):
            return x[0, at].float() if residual is None else x[0, at].float() + r[0, at].float()

        squares = sum(float((h_of(at).double() ** 2).sum()) for at in pieces(k))
        by = np.float32(1.0 / np.sqrt(squares / k + 1e-6))

        def v_of(at):
            return h_of(at) * float(by) * gamma[at]

        largest = max(float(v_of(at).abs().max()) for at in pieces(k))
        for out in (dtype, torch.int8, FP4):
            got = ops.rms_norm(x, gamma, residual, 1e-6, out)
            got = got if isinstance(got, tuple) else (got,)
            if residual is not None:
                assert all(torch.equal(got[-1][0, at], h_of(at).to(dtype)) for at in pieces(k))
            if out == dtype:
                assert all(torch.equal(got[0][0, at], v_of(at).to(dtype)) for at in pieces(k))
            elif out == torch.int8:
                assert got[1].item() == np.float32(largest) / np.float32(127)
                factor = float(np.float32(127) / np.float32(largest))
                assert all(torch.equal(got[0][0, at], (v_of(at) * factor).round().to(torch.int8)) for at in pieces(k))
            else:
                q, s = bits(got[0]), bits(got[1]).view(-1, 128, 4)
                for at in pieces(k):
                    want_q, want_s = (bits(t) for t in ops.quantize_rows_mxfp4(v_of(at).view(1, -1)))
                    first = at.start // 128
                    assert torch.equal(q[0, at.start // 2:][:want_q.shape[1]], want_q[0]) and torch.equal(s[first:first + want_s.shape[1]], want_s.view(-1, 128, 4))
            del got
