"""Plain forms in 64 bits of the 4-bit rows and products and of rms_norm, and how far results may be off."""
import numpy as np
import torch

import int8_layers as int8

EPS32 = int8.EPS32
VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def numbers(t):
    """A tensor of any floating type on the host, in 64 bits."""
    return None if t is None else t.detach().cpu().float().double().numpy()


# ---- 4-bit rows -----------------------------------------------------------------------------------------------------
def quantize(x):
    """(codes [m, 32 groups], scale bytes [m, groups]) of x [m, k], an array in 64 bits.  A group that is not finite has byte 255 and codes of 0."""
    m, k = x.shape
    v = np.zeros((m, (k + 31) // 32 * 32))
    v[:, :k] = x
    v = v.reshape(m, -1, 32)
    largest = np.abs(v).max(2)
    fine = np.isfinite(largest)
    exponent = np.maximum(np.frexp(np.where(fine, largest, 0.0))[1] - 3, -127)       # frexp: the power of two above
    exponent = np.where(np.where(fine, largest, 0.0) == 0.0, -127, exponent)
    t = np.ldexp(np.where(fine[..., None], v, 0.0), -exponent[..., None])
    step = np.where(np.abs(t) < 2, 0.5, np.where(np.abs(t) < 4, 1.0, 2.0))
    size = np.minimum(np.abs(np.rint(t / step) * step), 6.0)
    codes = np.searchsorted(VALUES, size) + 8 * np.signbit(t)
    return codes.reshape(m, -1).astype(np.uint8), np.where(fine, exponent + 127, 255).astype(np.uint8)


def values(codes, scales):
    """What codes and scale bytes stand for; NaN of a group whose byte is 255."""
    with np.errstate(invalid="ignore"):
        by = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
        return VALUES[codes & 7] * np.where(codes & 8, -1.0, 1.0) * np.repeat(by, 32, 1)


def pack(codes):
    return codes[:, 0::2] | codes[:, 1::2] << 4


def unpack(q):
    codes = np.empty((q.shape[0], 2 * q.shape[1]), dtype=np.uint8)
    codes[:, 0::2], codes[:, 1::2] = q & 15, q >> 4
    return codes


def tiles(scales):
    """Scale bytes [m, groups] one by one to the places that the header names."""
    m, groups = scales.shape
    across = (groups + 3) // 4
    out = np.zeros((m + 127) // 128 * across * 512, dtype=np.uint8)
    for r in range(m):
        for g in range(groups):
            out[(r // 128 * across + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4] = scales[r, g]
    return out


def from_tiles(t, m, groups):
    r, g = np.arange(m)[:, None], np.arange(groups)[None, :]
    return t.reshape(-1)[(r // 128 * ((groups + 3) // 4) + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4]


def bytes_of(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def decode(q, scales):
    """The values of a 4-bit matrix [m, bytes] on the GPU and its tiles, as a host array [m, 2 bytes]."""
    q = bytes_of(q)
    return values(unpack(q), from_tiles(bytes_of(scales), q.shape[0], q.shape[1] // 16))


# ---- product --------------------------------------------------------------------------------------------------------
def inner_prod(x, w, bias=None, residual=None, act=0, leaky=0.0, after=False, exact_sums=True):
    """The product in 64 bits of the values x and w, and the bound of its fp32 evaluation's error.

    Where all sums of products are multiples of one power of two and smaller than 2^24 of it, any order of fp32 additions is exact
    (exact_sums); otherwise k additions, each off by at most 2^-23 of a sum that is at most that of the magnitudes.  Bias and
    residual add half a step each, and an activation of slope at most 1.13 (gelu) passes that on and adds its own steps."""
    v = x @ w.T
    off = 0.0 if exact_sums else x.shape[1] * 2 * EPS32 * (np.abs(x) @ np.abs(w).T)
    size = np.abs(v)
    if bias is not None:
        v = v + bias
        size = size + np.abs(bias)
    if residual is not None and not after:
        v = v + residual
        size = size + np.abs(residual)
    v = int8.activation(v, act, leaky)
    if residual is not None and after:
        v = v + residual
        size = size + np.abs(residual)
    return v, 1.13 * (off + size * 4 * EPS32) + int8.transcendental(v, act)


# ---- norm -----------------------------------------------------------------------------------------------------------
def rms_norm(x, gamma=None, residual=None, eps=1e-6):
    """(v, h) of a tensor x [m, k]: h as the definition rounds it, v by its fp32 steps -- products of two fp32 values are exact in 64 bits, so
    one rounding to fp32 each makes them the fp32 products."""
    h = x.detach().cpu()
    if residual is not None:
        h = (h.float() + residual.detach().cpu().float()).to(x.dtype)
    t = numbers(h)
    with np.errstate(all="ignore"):
        by = (1.0 / np.sqrt((t * t).sum(1, keepdims=True) / t.shape[1] + eps)).astype(np.float32)
        v = (t * by.astype(np.float64)).astype(np.float32)
        if gamma is not None:
            v = (v.astype(np.float64) * numbers(gamma)).astype(np.float32)
    return v, h
