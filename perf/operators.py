"""The operators of int8 networks built from matrix products and group norms, as cases that can be timed and compared.

* ``rows``    quantize_rows: int8 values of a float matrix with a scale for each row, taken from the row's largest magnitude;
* ``prod``    inner_prod_quantized on int8 rows: int8 x int8 -> int32 sums, times a scale per token and per output channel, bias,
  residual, activation;
* ``token``   inner_prod_quantized on float rows: the same with the rows quantized in the call, as a served layer runs;
* ``norm``    group_norm_nhwc: group norm and activation on channels-last images, float or int8 (for a convolution) out.

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
_EPS = 1e-5
_TINY = 2.0 ** -100        # rows whose largest magnitude is below this count as zero
# no drawn case is dearer than the dearest listed ones
_MOST_VALUES = 1 << 27
_MOST_MACS = 1 << 39


def _rows(name, m, k, dtype):
    return dict(name=name, kind="rows", m=m, k=k, dtype=dtype)


def _prod(name, kind, m, n, k, dtype, out, act="none", bias=True, residual=False):
    return dict(name=name, kind=kind, m=m, n=n, k=k, dtype=dtype, out=out, act=act, bias=bias, residual=residual)


def _norm(name, n, h, w, c, groups, dtype, out, act):
    return dict(name=name, kind="norm", n=n, h=h, w=w, c=c, groups=groups, dtype=dtype, out=out, act=act)


def listed():
    return [
        # one token on its way into a layer: all latency
        _rows("rows_token_2048_bf16", 1, 2048, "bfloat16"),
        # a ragged batch in fp32: rows that no vector width divides
        _rows("rows_ragged_997x1111_f32", 997, 1111, "float32"),
        # a long prompt's activations: memory traffic
        _rows("rows_prompt_32768x4096_f16", 32768, 4096, "float16"),
        # one token through a square layer, quantized in the call: the weights' bytes and latency
        _prod("token_1_4096x4096_bf16", "token", 1, 4096, 4096, "bfloat16", "bfloat16", bias=False),
        # sixteen sequences decoded together
        _prod("token_16_2048x8192_bf16", "token", 16, 2048, 8192, "bfloat16", "bfloat16", residual=True),
        # the classifier at the end of the residual network, 64 images: 2048 features, 1000 classes, fp32 out
        _prod("prod_classifier_64x1000x2048", "prod", 64, 1000, 2048, "int8", "float32"),
        # sizes that fit no tile, as pruned layers have them
        _prod("prod_ragged_333x777x1021_f16", "prod", 333, 777, 1021, "int8", "float16", act="gelu", residual=True),
        # a pointwise layer over the pixels of 32 images of 56 x 56: few channels, many rows
        _prod("prod_pixels_100352x256x64_bf16", "prod", 32 * 56 * 56, 256, 64, "int8", "bfloat16", act="silu"),
        # a long prompt through a wide layer: arithmetic
        _prod("prod_prompt_8192x8192x8192_bf16", "prod", 8192, 8192, 8192, "int8", "bfloat16"),
        # a deep stage of one image
        _norm("norm_16x16x128_f32", 1, 16, 16, 128, 32, "float32", "float32", "silu"),
        # in front of an int8 convolution: 16 images of the 56 x 56 stage, int8 out
        _norm("norm_56x56x256_b16_to_i8", 16, 56, 56, 256, 32, "bfloat16", "int8", "relu"),
        # a batch of large images: memory traffic
        _norm("norm_256x256x256_b8_bf16", 8, 256, 256, 256, 32, "bfloat16", "bfloat16", "silu"),
    ]


def _log(rng, lo, hi):
    """An integer from lo to hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A width: mostly a multiple of 16 as networks have them, sometimes any number."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.35 or v < 16 else max(lo, v // 16 * 16)


def draw(rng):
    kind = rng.choice(["rows", "token", "prod", "prod", "norm", "norm"])
    floats = ["float32", "float16", "bfloat16", "bfloat16"]
    while True:
        if kind == "rows":
            case = dict(kind=kind, m=_log(rng, 1, 32768), k=_size(rng, 16, 16384), dtype=rng.choice(floats))
            if case["m"] * case["k"] <= _MOST_VALUES:
                return case
        elif kind == "norm":
            groups = rng.choice([1, 2, 4, 8, 16, 32, 32, 32])
            per = _log(rng, 1, max(1, 1024 // groups))
            out = rng.choice(["same", "same", "int8"])
            dtype = rng.choice(floats)
            case = dict(kind=kind, n=_log(rng, 1, 32), h=_log(rng, 1, 256), w=_log(rng, 1, 256), c=groups * per, groups=groups, dtype=dtype,
                        out=dtype if out == "same" else out, act=rng.choice(["none", "relu"] if out == "int8" else ["none", "relu", "silu", "silu"]))
            values = case["n"] * case["h"] * case["w"] * case["c"]
            # (a group of a handful of values is no norm that a network has)
            if values <= _MOST_VALUES and case["h"] * case["w"] * per >= 32:
                return case
        else:
            case = dict(kind=kind, m=_log(rng, 1, 64 if kind == "token" else 32768), n=_size(rng, 8, 8192), k=_size(rng, 16, 8192),
                        dtype="int8" if kind == "prod" else rng.choice(floats), out=rng.choice(floats),
                        act=rng.choice(["none", "none", "relu", "leaky", "silu", "gelu"]), bias=rng.random() < 0.6, residual=rng.random() < 0.3)
            if case["m"] * case["n"] * case["k"] <= _MOST_MACS and case["m"] * case["n"] <= _MOST_VALUES:
                return case


# ---- what a program holds before the call ---------------------------------------------------------------------------
def _features(shape, dtype, gen):
    """Activations as layers produce them: normal values, a few columns an order of magnitude larger than the rest."""
    x = torch.randn(shape, device="cuda", generator=gen)
    x.mul_(torch.rand(shape[-1], device="cuda", generator=gen).lt_(0.01).mul_(9.0).add_(1.0))
    return x.to(_DTYPES[dtype])


def _int8_rows(m, k, gen):
    """An int8 matrix as quantize_rows lays it out: rows start 16 bytes apart or a multiple of that."""
    q = torch.empty((m, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda")
    q.random_(-127, 128, generator=gen)
    return q[:, :k]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    if case["kind"] == "rows":
        st["x"] = _features((case["m"], case["k"]), case["dtype"], gen)
        if case["m"] > 8:
            st["x"][case["m"] // 2].zero_()       # a padding token
        return st
    if case["kind"] == "norm":
        shape = (case["n"], case["h"], case["w"], case["c"])
        x = torch.randn(shape, device="cuda", generator=gen)
        x.mul_(torch.empty(case["c"], device="cuda").uniform_(0.5, 2.0, generator=gen))
        x.add_(torch.empty(case["c"], device="cuda").normal_(0.0, 1.0, generator=gen))
        st["x"] = x.to(_DTYPES[case["dtype"]])
        st["gamma"] = torch.empty(case["c"], device="cuda").normal_(1.0, 0.2, generator=gen)
        st["beta"] = torch.empty(case["c"], device="cuda").normal_(0.0, 0.2, generator=gen)
        st["scales"] = [127.0 / 6.0]
        return st
    m, n, k = case["m"], case["n"], case["k"]
    st["w"] = _int8_rows(n, k, gen)
    # weights of a variance of 1 / k, the largest of a row three to five deviations out
    st["ws"] = torch.empty(n, device="cuda").uniform_(3.0, 5.0, generator=gen).div_(127.0 * math.sqrt(k))
    st["bias"] = torch.empty(n, device="cuda").normal_(0.0, 0.1, generator=gen) if case["bias"] else None
    st["residual"] = torch.randn((m, n), device="cuda", generator=gen).to(_DTYPES[case["out"]]) if case["residual"] else None
    if case["kind"] == "token":
        st["x"] = _features((m, k), case["dtype"], gen)
        st["xs"] = None
    else:
        st["x"] = _int8_rows(m, k, gen)
        st["xs"] = torch.empty(m, device="cuda").uniform_(0.01, 0.05, generator=gen)
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


def _plain_quantize_rows(x):
    x = x.float()
    largest = x.abs().amax(1, keepdim=True)
    zero = largest < _TINY
    # (a tensor over a tensor is one rounded division; a number over a tensor would be a reciprocal and a product)
    by = torch.div(torch.full_like(largest, 127.0), largest.masked_fill(zero, 1.0))
    q = (x * by).round().masked_fill(zero, 0.0).to(torch.int8)
    return q, torch.div(largest, torch.full_like(largest, 127.0)).masked_fill(zero, 0.0).squeeze(1)


def _plain_product(st):
    x, xs = (st["x"], st["xs"]) if st["xs"] is not None else _plain_quantize_rows(st["x"])
    acc = (x.double() @ st["w"].double().t()).float()          # whole numbers: exact in 64 bits
    v = acc * st["ws"] * xs[:, None]
    if st["bias"] is not None:
        v = v + st["bias"]
    if st["residual"] is not None:
        v = v + st["residual"].float()
    return _plain_activation(v, st["act"]).to(_DTYPES[st["out"]])


def _plain_norm(st):
    n, h, w, c, g = (st[v] for v in ("n", "h", "w", "c", "groups"))
    x = st["x"].view(n, h * w, g, c // g)
    x64 = x.double()
    mean = x64.mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(((x64 - mean) * (x64 - mean)).mean((1, 3), keepdim=True) + _EPS)
    v = (x.float() - mean.float()) * rstd.float()
    v = v.view(n, h, w, c) * st["gamma"] + st["beta"]
    v = _plain_activation(v, st["act"])
    if st["out"] != "int8":
        return v.to(_DTYPES[st["out"]])
    # int8 for a convolution: channels padded with zeros to 16 or a multiple of 64; half to even, but the last count % 8 values in
    # channel-major order half away from zero
    t = (v * st["scales"][0]).permute(0, 3, 1, 2).reshape(-1)
    at = t.numel() // 8 * 8
    q = torch.cat([t[:at].round(), torch.trunc(t[at:].double() + torch.copysign(torch.full_like(t[at:].double(), 0.5), t[at:].double())).float()])
    q = q.clamp(-128.0, 127.0).to(torch.int8).view(n, c, h, w).permute(0, 2, 3, 1)
    out = torch.zeros((n, h, w, 16 if c <= 16 else (c + 63) // 64 * 64), dtype=torch.int8, device=q.device)
    out[..., :c] = q
    return out


def run(state):
    st = state
    if own:
        from tennis_b200 import ops
        if st["kind"] == "rows":
            return ops.quantize_rows(st["x"])
        if st["kind"] == "norm":
            return ops.group_norm_nhwc(st["x"], st["groups"], st["gamma"], st["beta"], eps=_EPS, activation=_ACTS[st["act"]],
                                       out_dtype=_DTYPES[st["out"]], requant_scales=st["scales"] if st["out"] == "int8" else None)
        return ops.inner_prod_quantized(st["x"], st["xs"], st["w"], st["ws"], bias=st["bias"], residual=st["residual"],
                                        activation=_ACTS[st["act"]], leaky=_LEAKY, out_dtype=_DTYPES[st["out"]])
    if st["kind"] == "rows":
        return _plain_quantize_rows(st["x"])
    return _plain_norm(st) if st["kind"] == "norm" else _plain_product(st)


def work(case):
    if case["kind"] == "rows":
        values = case["m"] * case["k"]
        return {"bytes": values * (_SIZE[case["dtype"]] + 1) + 4 * case["m"], "flops": 3 * values}
    if case["kind"] == "norm":
        pixels = case["n"] * case["h"] * case["w"]
        c = case["c"]
        written = c if case["out"] != "int8" else (16 if c <= 16 else (c + 63) // 64 * 64)
        return {"bytes": pixels * (c * _SIZE[case["dtype"]] + written * _SIZE[case["out"]]) + 8 * c, "flops": 8 * pixels * c}
    m, n, k = case["m"], case["n"], case["k"]
    x = m * k * _SIZE[case["dtype"]] + (4 * m if case["kind"] == "prod" else 0)
    y = m * n * _SIZE[case["out"]] * (2 if case["residual"] else 1)
    return {"bytes": x + n * k + 4 * n * (2 if case["bias"] else 1) + y, "flops": 2 * m * n * k}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _erf(v):
    return torch.erf(torch.from_numpy(v)).numpy()


def _exact_activation(v, act):
    if act == "relu":
        return np.maximum(v, 0.0)
    if act == "leaky":
        return np.where(v > 0, v, _LEAKY * v)
    if act == "silu":
        return v / (1.0 + np.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + _erf(v / math.sqrt(2.0)))
    return v


def _exact_rows(x):
    """The int8 values are defined by 32-bit steps (scale, product), which a product in 64 bits that is rounded once equals."""
    largest = np.abs(x).max(1)
    by = np.array([127.0 / a if a >= _TINY else 0.0 for a in largest]).astype(np.float32).astype(np.float64)
    q = np.rint((x * by[:, None]).astype(np.float32))
    return q, np.where(largest >= _TINY, largest / 127.0, 0.0)


def exact(case, seed):
    if case["kind"] in ("prod", "token") and case["m"] * case["n"] * case["k"] > 1 << 35:
        return None
    st = prepare(case, seed)
    host = {name: v.cpu().double().numpy() for name, v in st.items() if isinstance(v, torch.Tensor)}
    x = host["x"]
    if case["kind"] == "rows":
        q, s = _exact_rows(x)
        return q.astype(np.int8), s
    if case["kind"] == "norm":
        if case["out"] == "int8":
            return None
        n, c, g = case["n"], case["c"], case["groups"]
        out = np.empty_like(x)
        for i in range(n):                                       # image by image: a large batch in 64 bits is many GB
            xi = x[i].reshape(-1, g, c // g)
            mean = xi.mean((0, 2), keepdims=True)
            xi = xi - mean
            v = (xi / np.sqrt((xi * xi).mean((0, 2), keepdims=True) + _EPS)).reshape(x[i].shape)
            out[i] = _exact_activation(v * host["gamma"] + host["beta"], case["act"])
        return out
    xs = host.get("xs")
    if xs is None:
        x, xs = _exact_rows(x)
    v = (x @ host["w"].T) * host["ws"] * xs[:, None]
    if case["bias"]:
        v = v + host["bias"]
    if case["residual"]:
        v = v + host["residual"]
    return _exact_activation(v, case["act"])
