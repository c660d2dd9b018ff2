"""Plain forms in 64 bits of quantize_rows, inner_prod_quantized and group_norm_nhwc, and how far results may be off."""
import math

import numpy as np
import torch

TINY = 2.0 ** -100
EPS32 = 2.0 ** -24       # half a step of fp32, relative


def half_step(dtype):
    """The relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def quantize_rows(x):
    """(q, scales) of a float tensor [m, k] on the CPU.  The 32-bit steps belong to the definition; a product of two fp32 values is
    exact in 64 bits, so rounding it once to fp32 is the fp32 product."""
    x = x.float().double().numpy()
    with np.errstate(all="ignore"):
        a = np.abs(x).max(axis=1)                      # (NaN carries through)
        zero = a < TINY
        by = np.where(zero, 0.0, np.float64(127.0) / a).astype(np.float32)
        t = (x * by[:, None].astype(np.float64)).astype(np.float32)
        q = np.where(np.isfinite(t), np.clip(np.rint(t), -128, 127), -128.0).astype(np.int8)
        s = np.where(zero, 0.0, a / 127.0)
    return q, s


def activation(v, act, leaky):
    if act == 1:
        return np.where(v > 0, v, 0.0)
    if act == 2:
        return np.where(v > 0, v, v * leaky)
    if act == 3:
        with np.errstate(over="ignore"):
            return v / (1.0 + np.exp(-v))
    if act == 4:
        return 0.5 * v * (1.0 + torch.erf(torch.from_numpy(v) * math.sqrt(0.5)).numpy())
    return v


def inner_prod(q, xs, w, ws, bias=None, residual=None, act=0, leaky=0.0, after=False):
    """The product in 64 bits, and the bound of its fp32 evaluation's error: each rounded step adds half a step of the largest
    magnitude that it meets (int32 -> fp32, two scales, bias, residual: five), and an activation of slope at most 1.13 (gelu)
    passes that on and adds its own steps."""
    v = (q.astype(np.float64) @ w.astype(np.float64).T) * ws.astype(np.float64) * np.asarray(xs, dtype=np.float64).reshape(-1, 1)
    size = np.abs(v)
    if bias is not None:
        v = v + bias
        size = size + np.abs(bias)
    if residual is not None and not after:
        v = v + residual
        size = size + np.abs(residual)
    v = activation(v, act, leaky)
    if residual is not None and after:
        v = v + residual
        size = size + np.abs(residual)
    return v, size * 5 * 1.13 * EPS32 + transcendental(v, act)


def transcendental(v, act):
    """What silu and gelu add: expf and erff are within 2 units in the last place (4 half steps); of gelu the sum 1 + erf cancels
    for negative values, which leaves an error of a few half steps of |v| / 2 itself, so the bound goes by |v| before the activation
    where that is larger: |v| <= 6 wherever gelu(v) is not v or 0 to fp32, silu's factors have no cancellation."""
    if act == 3:
        return np.abs(v) * 8 * EPS32
    if act == 4:
        return (np.abs(v) * 4 + 6 * 4) * EPS32
    return 0.0


def group_norm(x, groups, gamma=None, beta=None, eps=1e-5, act=0, leaky=0.0):
    """Values in 64 bits of x [n, ..., c] (float64 numpy), and the bound of the fp32 evaluation's error: mean rounded once (half a step of
    |mean|, over the deviation), x - mean, the reciprocal deviation, the product with it, gamma, beta: six half steps in all."""
    n, c = x.shape[0], x.shape[-1]
    t = x.reshape(n, -1, groups, c // groups)
    mean = t.mean((1, 3), keepdims=True)
    rstd = 1.0 / np.sqrt(((t - mean) ** 2).mean((1, 3), keepdims=True) + eps)
    v = ((t - mean) * rstd).reshape(x.shape)
    off = ((np.abs(t - mean) * 4 + np.abs(mean)) * rstd).reshape(x.shape)
    if gamma is not None:
        v, off = v * gamma, off * np.abs(gamma)
    off = off + np.abs(v) * 2
    if beta is not None:
        v = v + beta
        off = off + np.abs(beta) + np.abs(v)
    y = activation(v, act, leaky)
    return y, off * 1.13 * EPS32 + transcendental(y, act)


def assert_close(got, want, bound, dtype):
    """got (a tensor of dtype) within the fp32 bound and one rounding to dtype of want; subnormal results of fp16 by its smallest step."""
    got = got.detach().float().cpu().double().numpy()
    room = bound + (0.0 if dtype == torch.float32 else half_step(dtype) * (np.abs(want) + bound) + (2.0 ** -25 if dtype == torch.float16 else 0.0)) + 1e-37
    bad = ~(np.abs(got - want) <= room)
    assert not bad.any(), "%d of %d off, by up to %g of their room (first at %s: %r, not %r)" % (
        bad.sum(), bad.size, float(np.max(np.abs(got - want) / room)), np.argwhere(bad)[0], got[tuple(np.argwhere(bad)[0])], want[tuple(np.argwhere(bad)[0])])
