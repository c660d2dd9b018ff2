"""quantize_rows against its definition: whole values and scales, at sizes and values where it can go wrong."""
import numpy as np
import pytest
import torch

import int8_layers as plain

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


def check(x, q, s):
    want_q, want_s = plain.quantize_rows(x.cpu())
    assert np.array_equal(q.cpu().numpy(), want_q)
    got = s.cpu().double().numpy()
    # a / 127 is rounded once
    with np.errstate(invalid="ignore"):
        same = (got == want_s) | (np.isnan(got) & np.isnan(want_s)) | (np.abs(got - want_s) <= np.abs(want_s) * plain.EPS32)
    assert same.all()


def values(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * 3).to(dtype)


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 7), (3, 8), (2, 16), (5, 31), (1, 2048), (7, 1000), (33, 1023), (4, 4096), (3, 4104), (2, 8192), (2, 8200),
                                 (3, 16384), (2, 40000), (1, 70001), (5000, 24), (1030, 257), (20000, 3), (300, 128), (257, 64), (65, 520)])
def test_sizes(m, k, dtype):
    from tennis_b200 import ops
    x = values((m, k), dtype, m + k)
    q, s = ops.quantize_rows(x)
    assert q.shape == (m, k) and s.shape == (m,) and (m == 1 or q.stride(0) % 16 == 0)
    check(x, q, s)


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
@pytest.mark.parametrize("k", [5, 64, 1000, 5000, 20000])
def test_special_rows(dtype, k):
    from tennis_b200 import ops
    x = values((12, k), dtype, 3)
    x[0] = 0.0
    x[1] = -0.0
    x[2, k // 2] = float("nan")
    x[3, k - 1] = float("inf")
    x[4, 0] = -float("inf")
    x[5] = 2.0 ** -24                        # the smallest fp16
    x[6] = torch.finfo(dtype).max
    x[7] = -torch.finfo(dtype).max
    x[8] = 0.0
    x[8, k - 1] = -1.0
    x[9] = torch.arange(k, device="cuda").remainder(255).sub(127).to(dtype) * 0.5     # halves: ties once scaled by 2
    x[9, 0] = 63.5
    if dtype != torch.float16:
        x[10] = 1e-31                        # counts as zero
        x[11] = 1e-30                        # does not
    q, s = ops.quantize_rows(x)
    check(x, q, s)
    assert s[0] == 0 and s[1] == 0 and torch.isnan(s[2]) and torch.isinf(s[3]) and torch.isinf(s[4])
    assert (q[2] == -128).all() and q[3, k - 1] == -128 and q[4, 0] == -128
    assert (q[6] == 127).all() and (q[7] == -127).all() and q[8, k - 1] == -127


@pytest.mark.parametrize("dtype", FLOATS, ids=str)
def test_layouts(dtype):
    """Pitches, misaligned starts, broadcast rows, transposes, more than two dimensions, outputs of the caller's."""
    from tennis_b200 import ops
    wide = values((40, 517), dtype, 1)
    for x in (wide[:, 3:500], wide[:, 8:264], wide[::2, 1:257], wide[5:6].expand(9, 517), wide.t(), wide.view(4, 10, 517), wide.view(4, 10, 517)[:, 2:5, 4:205],
              wide[3], wide[:1, :16]):
        q, s = ops.quantize_rows(x)
        k = x.shape[-1]
        assert q.shape == x.shape and s.shape == x.shape[:-1]
        check(x.reshape(-1, k), q.reshape(-1, k), s.reshape(-1))
    for pitch, at, k in ((517, 0, 517), (520, 1, 300), (528, 16, 512), (512, 0, 512), (531, 3, 512)):
        room = torch.full((40 * pitch + 64,), 77, dtype=torch.int8, device="cuda")
        out = room[at:].as_strided((40, k), (pitch, 1))
        scales = torch.zeros(40, device="cuda")
        q, s = ops.quantize_rows(wide[:, :k], out=out, scales=scales)
        assert q is out and s is scales
        check(wide[:, :k], q, s)
        written = torch.zeros_like(room, dtype=torch.bool)
        written[at:].as_strided((40, k), (pitch, 1)).fill_(True)
        assert (room[~written] == 77).all()           # nothing between or behind the rows


def test_far_offsets():
    """Rows whose offsets pass 32 bits, of elements and of bytes."""
    from tennis_b200 import ops
    pitch = (1 << 31) // 2 + 8
    room = torch.empty(4 * pitch + 64, dtype=torch.float16, device="cuda")
    x = room.as_strided((5, 64), (pitch, 1))
    x.copy_(values((5, 64), torch.float16, 9))
    y = torch.empty(4 * pitch + 64, dtype=torch.int8, device="cuda").as_strided((5, 64), (pitch, 1))
    q, s = ops.quantize_rows(x, out=y)
    check(x, q, s)


def test_streams_and_graphs():
    from tennis_b200 import ops
    x = values((64, 1000), torch.bfloat16, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, s = ops.quantize_rows(x, stream=side)
    side.synchronize()
    check(x, q, s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s = ops.quantize_rows(x)
    for seed in (5, 6):
        x.copy_(values((64, 1000), torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        check(x, q, s)


def test_refusals():
    from tennis_b200 import ops
    x = torch.ones((4, 8), device="cuda")
    for call in (lambda: ops.quantize_rows(x.double()), lambda: ops.quantize_rows(x[:, :0]), lambda: ops.quantize_rows(x.new_ones(())),
                 lambda: ops.quantize_rows(x, out=torch.empty((4, 8), device="cuda")), lambda: ops.quantize_rows(x, out=torch.empty((8, 4), dtype=torch.int8, device="cuda").t()),
                 lambda: ops.quantize_rows(x, scales=torch.ones(3, device="cuda")), lambda: ops.quantize_rows(x, scales=torch.ones(8, device="cuda")[::2]),
                 lambda: ops.quantize_rows(x.view(2, 2, 8), out=torch.empty((2, 3, 8), dtype=torch.int8, device="cuda")[:, :2])):
        with pytest.raises(ops.EjectionException, match="Check failed"):
            call()


def test_empty():
    from tennis_b200 import ops
    q, s = ops.quantize_rows(torch.empty((0, 8), device="cuda"))
    assert q.shape == (0, 8) and s.shape == (0,)
    q, s = ops.quantize_rows(torch.empty((3, 0, 8), device="cuda"))
    assert q.shape == (3, 0, 8) and s.shape == (3, 0)


@pytest.mark.parametrize("shape", [(0, 8), (3, 0, 8), (0, 3, 5)])
def test_empty_outputs_of_the_callers(shape):
    from tennis_b200 import ops
    out, scales = torch.empty(shape, dtype=torch.int8, device="cuda"), torch.empty(shape[:-1], device="cuda")
    q, s = ops.quantize_rows(torch.empty(shape, device="cuda"), out=out, scales=scales)
    assert q is out and s is scales
