"""The operators of networks whose layers are root-mean-square norms and matrix products in 4 bits, as cases that can be timed and compared.

* ``norm``    rms_norm: the residual's addition, the norm of the sum and a weight per column, to floats or to int8 with a scale per row;
* ``pack``    quantize_rows_mxfp4 and dequantize_rows_mxfp4: 4-bit floating-point values with a power of two for every 32 of a row, and
  the values that they stand for;
* ``prod``    inner_prod_mxfp4 on 4-bit rows: sums, bias, residual, activation;
* ``token``   inner_prod_mxfp4 on float rows: the same with the rows quantized in the call, as a served layer runs;
* ``layer``   rms_norm with a residual to 4 bits and inner_prod_mxfp4 of the result: the two together, as a network runs them.

A 4-bit matrix is held as bytes of two values (the lower half first), rows filled up with zeros to a multiple of 32 values, and its scales
as tiles of 128 rows x 4 scales, ``[rows / 128, columns / 128, 32, 4, 4]``: row r, group g at ``[r // 128, g // 4, r % 32, r % 128 // 32, g % 4]``.

A case is a dict of plain values.  ``listed()`` gives the standing ones, ``draw(rng)`` one more of the same ranges, ``prepare`` what
a program holds before the call, ``run`` one pass (``own``: through the framework, otherwise in elementary torch operations),
``work`` the bytes and operations that a pass cannot do without, ``exact`` the outputs by the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16, "int8": torch.int8}
_SIZE = {"float32": 4, "float16": 2, "bfloat16": 2, "int8": 1}
_ACTS = {"none": 0, "relu": 1, "leaky": 2, "silu": 3, "gelu": 4}      # the framework's ACT_* numbers
_LEAKY = 0.1
_EPS = 1e-6
_TINY = 2.0 ** -100        # int8 rows whose largest magnitude is below this count as zero
_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]                    # the magnitudes of the 4-bit codes 0 to 7
# no drawn case is dearer than the dearest listed ones
_MOST_VALUES = 1 << 27
_MOST_MACS = 1 << 39


def _norm(name, m, k, dtype, out, residual):
    return dict(name=name, kind="norm", m=m, k=k, dtype=dtype, out=out, residual=residual)


def _pack(name, m, k, dtype):
    return dict(name=name, kind="pack", m=m, k=k, dtype=dtype)


def _prod(name, kind, m, n, k, dtype, out, act="none", bias=True, residual=False):
    return dict(name=name, kind=kind, m=m, n=n, k=k, dtype=dtype, out=out, act=act, bias=bias, residual=residual)


def listed():
    return [
        # one token on its way into an int8 layer: all latency
        _norm("norm_token_4096_bf16_to_i8", 1, 4096, "bfloat16", "int8", True),
        # a ragged batch in fp32: rows that no vector width divides
        _norm("norm_ragged_997x1111_f32", 997, 1111, "float32", "float32", False),
        # a long prompt's activations between two int8 layers: memory traffic
        _norm("norm_prompt_16384x8192_bf16_to_i8", 16384, 8192, "bfloat16", "int8", True),
        # activations of odd width, to 4 bits and back
        _pack("pack_ragged_997x1111_f32", 997, 1111, "float32"),
        # a weight matrix as it is laid out: memory traffic
        _pack("pack_weights_8192x16384_bf16", 8192, 16384, "bfloat16"),
        # one token through a square layer, quantized in the call: the weights' bytes and latency
        _prod("token_1_4096x4096_bf16", "token", 1, 4096, 4096, "bfloat16", "bfloat16", bias=False),
        # thirty-two sequences decoded together through a wide layer
        _prod("token_32_8192x8192_bf16", "token", 32, 8192, 8192, "bfloat16", "bfloat16", residual=True),
        # sizes that fit no tile, as pruned layers have them
        _prod("prod_ragged_333x777x1021_f16", "prod", 333, 777, 1021, "mxfp4", "float16", act="gelu", residual=True),
        # a pointwise layer over the pixels of 32 images of 56 x 56: few channels, many rows
        _prod("prod_pixels_100352x256x64_bf16", "prod", 32 * 56 * 56, 256, 64, "mxfp4", "bfloat16", act="silu"),
        # a long prompt through a wide layer: arithmetic
        _prod("prod_prompt_8192x8192x8192_bf16", "prod", 8192, 8192, 8192, "mxfp4", "bfloat16"),
        # the residual stream of sixteen sequences into a layer
        _prod("layer_16_4096x4096_bf16", "layer", 16, 4096, 4096, "bfloat16", "bfloat16", bias=False),
        # the same of a prompt
        _prod("layer_2048x4096x4096_bf16", "layer", 2048, 4096, 4096, "bfloat16", "bfloat16", act="silu"),
    ]


def _log(rng, lo, hi):
    """An integer from lo to hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A width: mostly a multiple of 32 as networks have them, sometimes any number."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.35 or v < 32 else max(lo, v // 32 * 32)


def draw(rng):
    kind = rng.choice(["norm", "norm", "pack", "token", "prod", "prod", "layer"])
    floats = ["float32", "float16", "bfloat16", "bfloat16"]
    while True:
        if kind in ("norm", "pack"):
            case = dict(kind=kind, m=_log(rng, 1, 32768), k=_size(rng, 16, 16384), dtype=rng.choice(floats))
            if kind == "norm":
                case.update(out=rng.choice([case["dtype"], "int8"]), residual=rng.random() < 0.6)
            if case["m"] * case["k"] <= _MOST_VALUES:
                return case
        else:
            few = kind == "token" or (kind == "layer" and rng.random() < 0.5)
            dtype = rng.choice(floats)
            case = dict(kind=kind, m=_log(rng, 1, 64 if few else 32768), n=_size(rng, 8, 8192), k=_size(rng, 16, 8192),
                        dtype="mxfp4" if kind == "prod" else dtype, out=dtype, act=rng.choice(["none", "none", "relu", "leaky", "silu", "gelu"]),
                        bias=rng.random() < 0.6, residual=kind != "layer" and rng.random() < 0.3)
            if case["m"] * case["n"] * case["k"] <= _MOST_MACS and case["m"] * max(case["n"], case["k"]) <= _MOST_VALUES:
                return case


# ---- what a program holds before the call ---------------------------------------------------------------------------
def _features(shape, dtype, gen):
    """Activations as layers produce them: normal values, a few columns an order of magnitude larger than the rest."""
    x = torch.randn(shape, device="cuda", generator=gen)
    x.mul_(torch.rand(shape[-1], device="cuda", generator=gen).lt_(0.01).mul_(9.0).add_(1.0))
    return x.to(_DTYPES[dtype])


def _tiles(scales):
    """Scales [m, groups] as tiles; places that stand for nothing are zero."""
    m, g = scales.shape
    t = torch.zeros(((m + 127) // 128 * 128, (g + 3) // 4 * 4), dtype=scales.dtype, device=scales.device)
    t[:m, :g] = scales
    return t.view(t.shape[0] // 128, 4, 32, t.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def _mxfp4_rows(m, k, gen, around):
    """A 4-bit matrix of a size and its scales: exponents that differ by a few powers of two, codes as normal values have them."""
    groups = (k + 31) // 32
    codes = torch.empty((m, groups * 32), dtype=torch.uint8, device="cuda").random_(0, 16, generator=gen)
    codes[:, k:] = 0
    q = (codes[:, 1::2] << 4).add_(codes[:, 0::2])
    scales = torch.empty((m, groups), dtype=torch.uint8, device="cuda").random_(around - 1, around + 2, generator=gen)
    return q.view(torch.float4_e2m1fn_x2), _tiles(scales).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    kind, m, k = case["kind"], case["m"], case["k"]
    if kind in ("norm", "pack", "token", "layer"):
        st["x"] = _features((m, k), case["dtype"], gen)
        if m > 8 and kind in ("norm", "pack"):
            st["x"][m // 2].zero_()       # a padding token
    if kind in ("norm", "layer"):
        st["gamma"] = torch.empty(k, device="cuda").normal_(1.0, 0.2, generator=gen)
        st["stream"] = _features((m, k), case["dtype"], gen) if kind == "layer" or case["residual"] else None
    if kind in ("norm", "pack"):
        return st
    n = case["n"]
    # weights of a variance of about 1 / k: codes have one of some 8
    st["w"], st["ws"] = _mxfp4_rows(n, k, gen, 127 - int(round(math.log2(math.sqrt(8.0 * k)))))
    st["bias"] = torch.empty(n, device="cuda").normal_(0.0, 0.1, generator=gen) if case["bias"] else None
    st["residual"] = torch.randn((m, n), device="cuda", generator=gen).to(_DTYPES[case["out"]]) if case["residual"] else None
    if kind == "prod":
        st["x"], st["xs"] = _mxfp4_rows(m, k, gen, 126)
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------
def _plain_activation(v, act):
    if act == "relu":
        return v.clamp_min(0.0)
    if act == "leaky":
        return torch.where(v > 0, v, v * _LEAKY)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return v


def _plain_norm(st):
    """The norm in fp32, and the sum that it is the norm of."""
    h = st["x"]
    if st["stream"] is not None:
        h = (h.float() + st["stream"].float()).to(h.dtype)
    h64 = h.double()
    rstd = 1.0 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + _EPS)
    return h.float() * rstd.float() * st["gamma"], h


def _plain_quantize_rows(x):
    largest = x.abs().amax(1, keepdim=True)
    zero = largest < _TINY
    # (a tensor over a tensor is one rounded division; a number over a tensor would be a reciprocal and a product)
    by = torch.div(torch.full_like(largest, 127.0), largest.masked_fill(zero, 1.0))
    q = (x * by).round().masked_fill(zero, 0.0).to(torch.int8)
    return q, torch.div(largest, torch.full_like(largest, 127.0)).masked_fill(zero, 0.0).squeeze(1)


def _plain_mxfp4(x):
    """The values that x's 4-bit form stands for."""
    m, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(m, -1, 32)
    # the scale is the power of two two below the largest magnitude's, 2^-127 at least
    exponent = ((v.abs().amax(2, keepdim=True).view(torch.int32) >> 23) - 2).clamp_min(0)
    t = v.abs() * ((254 - exponent) << 23).view(torch.float32)
    # to the nearest of eight values, ties to the even one
    at = ((t > 0.25).int() + (t >= 0.75).int() + (t > 1.25).int() + (t >= 1.75).int() + (t > 2.5).int() + (t >= 3.5).int() + (t > 5.0).int())
    scale = torch.pow(2.0, (exponent - 127).double())
    t = torch.tensor(_VALUES, device=x.device)[at].copysign(v)
    return (t * scale).float().view(m, -1)[:, :k]


def _plain_values(q, scales):
    """The values of a 4-bit matrix."""
    q, scales = q.view(torch.uint8), scales.view(torch.uint8)
    m, groups = q.shape[0], q.shape[1] // 16
    s = scales.permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:m, :groups]
    code = torch.stack([q & 15, q >> 4], 2).view(m, groups, 32).long()
    table = torch.tensor(_VALUES + [-v for v in _VALUES], device=q.device)
    return (table[code] * torch.pow(2.0, s.int() - 127)[..., None]).view(m, -1)


def _plain_product(st, x):
    w = _plain_values(st["w"], st["ws"])
    v = torch.nn.functional.pad(x, (0, w.shape[1] - x.shape[1])) @ w.t()
    if st["bias"] is not None:
        v = v + st["bias"]
    if st["residual"] is not None:
        v = v + st["residual"].float()
    return _plain_activation(v, st["act"]).to(_DTYPES[st["out"]])


def run(state):
    st = state
    kind = st["kind"]
    if own:
        from tennis_b200 import ops
        if kind == "norm":
            return ops.rms_norm(st["x"], st["gamma"], residual=st["stream"], eps=_EPS, out_dtype=_DTYPES[st["out"]])
        if kind == "pack":
            q, s = ops.quantize_rows_mxfp4(st["x"])
            return ops.dequantize_rows_mxfp4(q, s, st["k"], _DTYPES[st["dtype"]])
        if kind == "layer":
            x, xs, h = ops.rms_norm(st["x"], st["gamma"], residual=st["stream"], eps=_EPS, out_dtype=torch.float4_e2m1fn_x2)
            return ops.inner_prod_mxfp4(x, xs, st["w"], st["ws"], bias=st["bias"], activation=_ACTS[st["act"]], leaky=_LEAKY,
                                        out_dtype=_DTYPES[st["out"]]), h
        return ops.inner_prod_mxfp4(st["x"], st.get("xs"), st["w"], st["ws"], bias=st["bias"], residual=st["residual"],
                                    activation=_ACTS[st["act"]], leaky=_LEAKY, out_dtype=_DTYPES[st["out"]])
    if kind == "norm":
        v, h = _plain_norm(st)
        y = _plain_quantize_rows(v) if st["out"] == "int8" else (v.to(_DTYPES[st["out"]]),)
        y = y + (h,) if st["stream"] is not None else y
        return y if len(y) > 1 else y[0]
    if kind == "pack":
        return _plain_mxfp4(st["x"]).to(_DTYPES[st["dtype"]])
    if kind == "layer":
        v, h = _plain_norm(st)
        return _plain_product(st, _plain_mxfp4(v)), h
    return _plain_product(st, _plain_mxfp4(st["x"]) if kind == "token" else _plain_values(st["x"], st["xs"]))


def _bytes4(rows, k):
    """Of a 4-bit matrix with its scales."""
    groups = (k + 31) // 32
    return rows * groups * 17


def work(case):
    kind, m, k = case["kind"], case["m"], case["k"]
    if kind == "norm":
        size = _SIZE[case["dtype"]]
        read = m * k * size * (2 if case["residual"] else 1) + 4 * k
        written = m * k * _SIZE[case["out"]] + (4 * m if case["out"] == "int8" else 0) + (m * k * size if case["residual"] else 0)
        return {"bytes": read + written, "flops": 6 * m * k}
    if kind == "pack":
        return {"bytes": 2 * m * k * _SIZE[case["dtype"]], "flops": 4 * m * k}
    n = case["n"]
    x = _bytes4(m, k) if kind == "prod" else m * k * _SIZE[case["dtype"]]
    if kind == "layer":
        x = 3 * x + 4 * k                   # the residual stream is read and written too
    y = m * n * _SIZE[case["out"]] * (2 if case["residual"] else 1)
    return {"bytes": x + _bytes4(n, k) + (4 * n if case["bias"] else 0) + y, "flops": 2 * m * n * k}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _exact_activation(v, act):
    if act == "relu":
        return np.maximum(v, 0.0)
    if act == "leaky":
        return np.where(v > 0, v, _LEAKY * v)
    if act == "silu":
        return v / (1.0 + np.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(torch.from_numpy(v / math.sqrt(2.0))).numpy())
    return v


def _exact_norm(case, host):
    """The norm by its 32-bit steps (sum, reciprocal deviation, two products), which steps in 64 bits that are rounded once equal, and in
    64 bits throughout."""
    h = host["x"]
    if host.get("stream") is not None:
        h = torch.from_numpy(h + host["stream"]).to(_DTYPES[case["dtype"]]).double().numpy()
    rstd = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + _EPS)
    steps = (h * rstd.astype(np.float32).astype(np.float64)).astype(np.float32).astype(np.float64)
    return (steps * host["gamma"]).astype(np.float32).astype(np.float64), h * rstd * host["gamma"], h


def _exact_mxfp4(x):
    """What the 4-bit form of x stands for: a step of a half, one or two by the size, halves of it to the even multiple."""
    m, k = x.shape
    v = np.pad(x, ((0, 0), (0, -k % 32))).reshape(m, -1, 32)
    largest = np.abs(v).max(2, keepdims=True)
    exponent = np.maximum(np.frexp(largest)[1] - 3, -127)
    t = np.ldexp(v, -exponent)
    step = np.where(np.abs(t) < 2.0, 0.5, np.where(np.abs(t) < 4.0, 1.0, 2.0))
    t = np.clip(np.rint(t / step) * step, -6.0, 6.0)
    return np.ldexp(t, exponent).reshape(m, -1)[:, :k]


def _exact_values(q, scales, k):
    q, scales = (v.view(torch.uint8).cpu().numpy() for v in (q, scales))
    m = q.shape[0]
    c = np.empty((m, q.shape[1] * 2), dtype=np.int64)
    c[:, 0::2], c[:, 1::2] = q & 15, q >> 4
    mantissa, exponent = c & 1, c >> 1 & 3
    v = np.where(exponent > 0, np.ldexp(1.0 + mantissa / 2.0, exponent - 1), mantissa / 2.0) * (1 - 2 * (c >> 3))
    r, g = np.arange(m)[:, None], np.arange(q.shape[1] // 16)[None, :]
    s = scales[r // 128, g // 4, r % 32, r % 128 // 32, g % 4].astype(np.int64) - 127
    return np.ldexp(v, np.repeat(s, 32, 1))[:, :k]


def exact(case, seed):
    kind, k = case["kind"], case["k"]
    if kind not in ("norm", "pack") and case["m"] * case["n"] * k > 1 << 36:
        return None
    st = prepare(case, seed)
    host = {name: v.cpu().double().numpy() for name, v in st.items() if isinstance(v, torch.Tensor) and v.element_size() > 1}
    if kind == "pack":
        return _exact_mxfp4(host["x"])
    if kind in ("norm", "layer"):
        steps, v, h = _exact_norm(case, host)
    if kind == "norm":
        if case["out"] == "int8":
            largest = np.abs(steps).max(1)
            by = np.array([127.0 / a if a >= _TINY else 0.0 for a in largest]).astype(np.float32).astype(np.float64)
            y = (np.rint((steps * by[:, None]).astype(np.float32)).astype(np.int8), np.where(largest >= _TINY, largest / 127.0, 0.0))
        else:
            y = (v,)
        y = y + (h,) if case["residual"] else y
        return y if len(y) > 1 else y[0]
    x = _exact_values(st["x"], st["xs"], k) if kind == "prod" else _exact_mxfp4(steps if kind == "layer" else host["x"])
    v = x @ _exact_values(st["w"], st["ws"], k).T
    if case["bias"]:
        v = v + host["bias"]
    if case["residual"]:
        v = v + host["residual"]
    v = _exact_activation(v, case["act"])
    return (v, h) if kind == "layer" else v
