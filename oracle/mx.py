"""The microscaled formats and their operators in numpy, in 64 bits, from their definitions.

Blocks of 32 values share a power of two; elements are e2m1 (4 bits) or e4m3 (8 bits). Written for checking:
decoding by each element's sign, exponent and mantissa, encoding by the step of a value's binade.
"""

from __future__ import annotations

import numpy as np

BLOCK, PAD = 32, 128
FORMATS = {4: (1, 1, 0, 6.0), 8: (3, 7, -6, 448.0)}     # mantissa bits, exponent bias, least exponent, largest value


def padded(k: int) -> int:
    return -(-k // PAD) * PAD


def _blocks(x):
    x = np.asarray(x, np.float64)
    wide = np.zeros((x.shape[0], padded(x.shape[1])))
    wide[:, :x.shape[1]] = x
    return wide.reshape(x.shape[0], -1, BLOCK)


def quantize(x, bits: int):
    """``(codes, scales)`` of rows: uint8 as they lie in memory."""
    b = _blocks(x)
    mantissa, bias, least, top = FORMATS[bits]
    bad = ~np.isfinite(b).all(2)
    b = np.where(bad[:, :, None], 0.0, b)
    largest = np.abs(b).max(2)
    exponent = np.frexp(largest)[1] - 1 - (2 if bits == 4 else 8)
    exponent = np.where(largest == 0, -127, np.maximum(exponent, -127))
    t = np.abs(b) / np.exp2(exponent.astype(np.float64))[:, :, None]
    step = np.exp2(np.maximum(np.frexp(t)[1] - 1, least) - float(mantissa))
    v = np.minimum(np.rint(t / step) * step, top)         # rint: ties to even
    e = np.maximum(np.frexp(v)[1] - 1, least)             # of the rounded value
    steps = np.rint(v / np.exp2(e - float(mantissa))).astype(np.int64)
    code = np.where(steps >= 1 << mantissa, ((e + bias) << mantissa) + steps - (1 << mantissa), steps)
    code = (code | np.signbit(b).astype(np.int64) << (bits - 1)).reshape(b.shape[0], -1).astype(np.uint8)
    code.reshape(b.shape)[bad] = 0
    if bits == 4:
        code = code[:, 0::2] | code[:, 1::2] << 4
    return np.ascontiguousarray(code), np.where(bad, 255, exponent + 127).astype(np.uint8)


def dequantize(codes, scales, k: int):
    """The values, float64 [rows, k]; NaN in a block of scale 255 (and for e4m3's NaN codes)."""
    bits = codes.shape[1] // scales.shape[1] // 4
    c = codes.astype(np.int64)
    if bits == 4:
        c = np.stack((c & 15, c >> 4), 2).reshape(c.shape[0], -1)
    mantissa, bias, least, _ = FORMATS[bits]
    e, f = (c >> mantissa) & ((1 << (bits - 1 - mantissa)) - 1), c & ((1 << mantissa) - 1)
    v = np.where(e > 0, f + (1 << mantissa), f) * np.exp2(np.maximum(e, 1) - bias - float(mantissa))
    if bits == 8:
        v = np.where(c & 127 == 127, np.nan, v)
    v = np.where(c >> (bits - 1) == 1, -v, v)
    power = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * np.repeat(power, BLOCK, 1))[:, :k]


def norm(x, delta, gamma, eps: float):
    """``(t, normed)`` float32: the sum of squares in 64 bits, its root's inverse rounded once, then float32
    products."""
    with np.errstate(all="ignore"):
        t = x if delta is None else (x + delta).astype(np.float32)
        t64 = t.astype(np.float64)
        r = (1 / np.sqrt((t64 * t64).sum(1, keepdims=True) / x.shape[1] + float(np.float32(eps)))).astype(np.float32)
        return t, ((t * r).astype(np.float32) * gamma).astype(np.float32)


def matmul(xq, xs, q, scales, bias=None, residual=None):
    """float64, and the sum of the magnitudes that were added (an error bound's scale)."""
    k = xs.shape[1] * BLOCK
    a, w = dequantize(xq, xs, k), dequantize(q, scales, k)
    y, size = a @ w.T, np.abs(a) @ np.abs(w).T
    for v in (bias, residual):
        if v is not None:
            y, size = y + v, size + np.abs(v)
    return y, size


def swiglu(xq, xs, qg, sg, qu, su):
    """float64 ``silu(gate) * up``, and the sums of magnitudes of gate and of up."""
    (g, gs), (u, us) = matmul(xq, xs, qg, sg), matmul(xq, xs, qu, su)
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u, (g, u, gs, us)
