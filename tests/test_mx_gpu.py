"""The microscaled operators on the GPU against their definitions in 64 bits.

Quantized rows and the norm's outputs are equal bit for bit: every step but the rounding to elements is exact, and
the norm's sum is taken in 64 bits. A product adds in float32: each matrix instruction and each addition is off by
at most half a step of what it adds, 2^-24 of the magnitudes, counted twice over for the instruction's inner sums
(2^-23 each). 128 values of k take one instruction where the activations have 4 bits and four where they have 8
(each takes 32 values), and there are at most 16 further additions (the waves' sums, bias, residual).
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import mx
from oracle import reference as R
from tests.conftest import bits as float_bits_of

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24


def activations(rng, m, k):
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[rng.random(x.shape) < 0.01] *= 20
    return x


def same_bits(a, b):
    """Equal bit for bit, any NaN for a NaN."""
    with np.errstate(over="ignore"):
        a, b = np.asarray(a, np.float32), np.asarray(b, np.float32)
    nan = np.isnan(a)
    return np.array_equal(nan, np.isnan(b)) and np.array_equal(float_bits_of(a)[~nan], float_bits_of(b)[~nan])


def shifted(array):
    """``array`` on the device one float past an aligned address."""
    from nanocompile_amd.hip import DeviceArray
    whole = DeviceArray((array.size + 1,), array.dtype)
    view = whole.view(array.shape, offset_bytes=array.itemsize)
    view.upload(array)
    return view


def guarded(nbytes, fill=0xA5):
    """A buffer of ``nbytes`` inside 64 bytes of a pattern on either side; and what checks and reads it."""
    from nanocompile_amd.hip import DeviceArray
    whole = DeviceArray.from_host(np.full(nbytes + 128, fill, np.uint8))

    def read():
        host = whole.numpy()
        assert (host[:64] == fill).all() and (host[64 + nbytes:] == fill).all(), "written outside"
        return host[64:64 + nbytes]
    return whole.ptr + 64, read


# -- the quantizer and its inverse ------------------------------------------------------------

ROWS = [(1, 1), (1, 31), (3, 32), (2, 33), (5, 127), (4, 128), (7, 129), (300, 896), (33, 1003), (2, 4864), (1, 70001)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m,k", ROWS)
def test_quantize_and_back(gpu, m, k, bits):
    from nanocompile_amd import hip, kernels
    print(f"quantize_mx m={m} k={k} bits={bits}", flush=True)
    rng = np.random.default_rng(m + k + bits)
    x = (rng.standard_normal((m, k)) * np.exp(5 * rng.standard_normal((m, 1)))).astype(np.float32)
    x[rng.random(x.shape) < 0.05] = 0
    codes, scales = mx.quantize(x, bits)
    for at in (x, shifted(x)):
        got = kernels.quantize_mx(at, bits)
        assert np.array_equal(got[0].numpy(), codes) and np.array_equal(got[1].numpy(), scales)
        assert same_bits(kernels.dequantize_mx(*got, k).numpy(), mx.dequantize(codes, scales, k))
    # nothing outside the outputs, which lie behind one another's guards
    (cp, cread), (sp, sread), (vp, vread) = (guarded(n) for n in (codes.size, scales.size, x.nbytes))
    hip.call("nc_quantize_mx", [cp, sp, shifted(x)], [m, k, bits])
    hip.call("nc_dequantize_mx", [vp, cp, sp], [m, k, bits])
    hip.sync()
    assert np.array_equal(cread(), codes.reshape(-1)) and np.array_equal(sread(), scales.reshape(-1))
    assert same_bits(vread().view(np.float32).reshape(m, k), mx.dequantize(codes, scales, k))


@pytest.mark.parametrize("bits", [4, 8])
def test_every_rounding_border(gpu, bits):
    """Every element, the middle of every two, and the floats next to both, in blocks of several scales."""
    from nanocompile_amd import kernels
    every = np.arange(127 if bits == 8 else 8, dtype=np.uint8)
    codes = np.zeros((1, 128 if bits == 8 else 64), np.uint8)
    codes[0, :every.size if bits == 8 else 4] = every if bits == 8 else every[0::2] | every[1::2] << 4
    values = mx.dequantize(codes, np.full((1, 4), 127, np.uint8), every.size)[0]
    points = np.concatenate([values, (values[1:] + values[:-1]) / 2, [values[-1] * 1.04, values[-1] * 1.14]])
    points = points.astype(np.float32)
    points = np.concatenate([points, np.nextafter(points, np.float32(1e9)), np.nextafter(points, np.float32(-1))])
    points = np.concatenate([points, -points])
    points = np.resize(points, -(-points.size // 31) * 31).reshape(-1, 31)
    rows = np.concatenate([np.full((points.shape[0], 1), values[-1], np.float32), points], 1)
    for power in (-100, -3, 0, 1, 90):
        x = (rows * np.float32(2.0 ** power)).astype(np.float32)
        got, want = kernels.quantize_mx(x, bits), mx.quantize(x, bits)
        assert np.array_equal(got[0].numpy(), want[0]) and np.array_equal(got[1].numpy(), want[1]), power


@pytest.mark.parametrize("bits", [4, 8])
def test_special_blocks(gpu, bits):
    """Zeros, subnormals, the largest float, infinities and NaN: each block by itself."""
    from nanocompile_amd import kernels
    top = np.finfo(np.float32).max
    x = np.ones((3, 9 * 32), np.float32)
    b = x.reshape(3, 9, 32)
    b[0, 0], b[0, 1], b[0, 2], b[0, 3, 5], b[0, 4, 0], b[0, 5, 31] = 0, 1e-45, 1.1e-38, np.nan, np.inf, -np.inf
    b[0, 6], b[0, 7], b[0, 8] = top, -0.0, 1.18e-38
    b[1, 0, 1:], b[1, 1], b[1, 2, 7] = 1e-45, 6e-39, -top
    got, want = kernels.quantize_mx(x, bits), mx.quantize(x, bits)
    assert np.array_equal(got[0].numpy(), want[0]) and np.array_equal(got[1].numpy(), want[1])
    assert same_bits(kernels.dequantize_mx(*got, x.shape[1]).numpy(), mx.dequantize(*want, x.shape[1]))


def test_every_code_and_scale_back(gpu):
    """Every element times every scale, among them values past float32's range and below its least."""
    from nanocompile_amd import kernels
    scales = np.repeat(np.arange(256, dtype=np.uint8), 8).reshape(-1, 8)
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    assert same_bits(kernels.dequantize_mx(codes, scales, 256).numpy(), mx.dequantize(codes, scales, 256))
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1)).reshape(256, 256)[:, :64]
    assert same_bits(kernels.dequantize_mx(codes, scales[:, :4], 128).numpy(),
                     mx.dequantize(codes, scales[:, :4], 128))


# -- the residual, the norm and the quantizer ----------------------------------------------------

NORMS = [(1, 1), (3, 7), (1, 896), (5, 896), (130, 129), (9, 1024), (6, 1025), (4, 2048), (3, 2049), (2, 4099), (2, 8192),
         (3, 8200), (2, 16390), (1, 32768)]


@pytest.mark.parametrize("mx_bits", [0, 4, 8])
@pytest.mark.parametrize("m,k", NORMS)
def test_norm_bit_for_bit(gpu, m, k, mx_bits):
    from nanocompile_amd import kernels
    print(f"add_rms_norm_quant m={m} k={k} mx_bits={mx_bits}", flush=True)
    rng = np.random.default_rng(m * 3 + k + mx_bits)
    x, delta = activations(rng, m, k), rng.standard_normal((m, k)).astype(np.float32)
    gamma = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    for d in (delta, None):
        t, n = mx.norm(x, d, gamma, 1e-6)
        q, qs = R.quantize_token(n) if mx_bits == 0 else mx.quantize(n, mx_bits)
        for up in (lambda a: a, shifted):
            got = kernels.add_rms_norm_quant(up(x), None if d is None else up(d), up(gamma), 1e-6, mx_bits, normed=True)
            got = [a.numpy() for a in got]
            assert same_bits(got[0], t) and same_bits(got[1], n)
            assert np.array_equal(got[2], q)
            assert same_bits(got[3], qs) if mx_bits == 0 else np.array_equal(got[3], qs)


@pytest.mark.parametrize("mx_bits", [0, 4, 8])
@pytest.mark.parametrize("m,k", [(5, 100), (2, 896), (3, 1500), (2, 9001)])
def test_norm_in_place_and_guards(gpu, m, k, mx_bits):
    """The new residual stream over either input; nothing written outside; the optional outputs left out."""
    from nanocompile_amd import hip, kernels
    from nanocompile_amd.hip import DeviceArray
    rng = np.random.default_rng(m + k)
    x, delta = activations(rng, m, k), rng.standard_normal((m, k)).astype(np.float32)
    gamma = (1 + 0.1 * rng.standard_normal(k)).astype(np.float32)
    t, n = mx.norm(x, delta, gamma, 1e-5)
    q, qs = R.quantize_token(n) if mx_bits == 0 else mx.quantize(n, mx_bits)
    for into in (0, 1, None):
        dx, dd, dg = (DeviceArray.from_host(a) for a in (x, delta, gamma))
        (qp, qread), (sp, sread) = guarded(q.nbytes), guarded(qs.nbytes)
        hip.call("nc_add_rms_norm_quant", [None if into is None else (dx, dd)[into], None, qp, sp, dx, dd, dg],
                 [m, k, kernels.float_bits(1e-5), mx_bits])
        hip.sync()
        assert np.array_equal(qread(), q.reshape(-1).view(np.uint8))
        assert np.array_equal(sread(), qs.reshape(-1).view(np.uint8))
        assert same_bits(dx.numpy(), t if into == 0 else x) and same_bits(dd.numpy(), t if into == 1 else delta)


@pytest.mark.parametrize("mx_bits", [0, 4, 8])
@pytest.mark.parametrize("k", [70, 3000])
def test_norm_of_zero_huge_and_bad_rows(gpu, mx_bits, k):
    """Zeros (with eps 0 too), values whose squares pass float32, a NaN and an infinity: each row by itself."""
    from nanocompile_amd import kernels
    x = np.ones((6, k), np.float32)
    x[0], x[1], x[2, k // 2], x[3, 0], x[4] = 0, 1e30, np.nan, np.inf, 1e-30
    gamma = np.ones(k, np.float32)
    for eps in (1e-6, 0.0):
        t, n = mx.norm(x, None, gamma, eps)
        got = [a.numpy() for a in kernels.add_rms_norm_quant(x, None, gamma, eps, mx_bits, normed=True)]
        with np.errstate(all="ignore"):
            assert same_bits(got[1], n)
            good = np.isfinite(n).all(1)
            if mx_bits:
                q, qs = mx.quantize(n, mx_bits)
                assert np.array_equal(got[2], q) and np.array_equal(got[3], qs)
            else:
                q, qs = R.quantize_token(n[good])
                assert np.array_equal(got[2][good], q) and same_bits(got[3][good], qs)
                assert np.isnan(got[3][~good]).all()


# -- the products ------------------------------------------------------------------------------------


def product_error(size, k, bits):
    """The most a sum of ``k`` products of the given magnitudes may be off."""
    return (mx.padded(k) // (128 if bits == 4 else 32) + 16) * 2 * HALF * size


def operands(rng, m, n, k, bits, weights=1):
    xq, xs = mx.quantize(activations(rng, m, k), bits)
    w = [mx.quantize((rng.standard_normal((n, k)) * 0.02 * np.exp(rng.standard_normal((n, 1)))).astype(np.float32), 4)
         for _ in range(weights)]
    return (xq, xs), w


def check_matmul(m, n, k, bits, seed=0):
    from nanocompile_amd import kernels
    print(f"matmul_mx m={m} n={n} k={k} bits={bits}", flush=True)
    rng = np.random.default_rng(m * 5 + n * 3 + k + bits + seed)
    x, (w,) = operands(rng, m, n, k, bits)
    bias, residual = rng.standard_normal(n).astype(np.float32), rng.standard_normal((m, n)).astype(np.float32)
    for b, r in ((None, None), (bias, None), (bias, residual)):
        want, size = mx.matmul(*x, *w, b, r)
        got = kernels.matmul_mx(*x, *w, b, r).numpy()
        assert (np.abs(got - want) <= product_error(size, k, bits)).all()


def check_swiglu(m, n, k, bits, seed=0):
    from nanocompile_amd import kernels
    print(f"matmul_mx_swiglu m={m} n={n} k={k} bits={bits}", flush=True)
    rng = np.random.default_rng(m * 5 + n * 3 + k + bits + seed)
    x, (wg, wu) = operands(rng, m, n, k, bits, 2)
    want, (g, u, gs, us) = mx.swiglu(*x, *wg, *wu)
    got = kernels.matmul_mx_swiglu(*x, *wg, *wu).numpy()
    dg, du = product_error(gs, k, bits), product_error(us, k, bits)
    # silu's slope is at most 1.1 and |silu(g)| <= |g|; its exponential, quotient and products: 8 roundings
    # of at most a step each
    most = 1.1 * dg * (np.abs(u) + du) + np.abs(g) * du + 16 * HALF * np.abs(want) + 1e-37
    assert (np.abs(got - want) <= most).all()


@pytest.mark.parametrize("m", [1, 1290])
def test_silu_over_its_range(gpu, m):
    """Gates that are one weight each, of either sign from 2^-127 to 6 * 2^100, exact; up 1: silu within 8 steps of
    float32, or of the gate times 2^-126 where the sigmoid is less than that."""
    from nanocompile_amd import kernels
    scales = np.arange(0, 228, dtype=np.uint8)
    n, k = 16 * len(scales), 520                       # 16 elements under every scale
    gate = np.zeros((n, 5 * 64), np.uint8), np.full((n, 5 * 4), 127, np.uint8)
    gate[0][:, 0], gate[1][:, 0] = np.arange(n) % 16, np.repeat(scales, 16)
    up = np.zeros_like(gate[0]), np.full_like(gate[1], 127)
    up[0][:, 0] = 2                                    # 1
    x = np.zeros((m, 5 * 128), np.uint8), np.full((m, 5 * 4), 127, np.uint8)
    x[0][:, 0] = 0x38                                  # 1
    g = mx.dequantize(*gate, k)[:, 0].astype(np.float64)
    with np.errstate(over="ignore"):
        want = g / (1 + np.exp(-g))
    got = kernels.matmul_mx_swiglu(*x, *gate, *up).numpy()
    assert (np.abs(got - want) <= 16 * HALF * np.abs(want) + 2.0 ** -126 * np.abs(g) + 2.0 ** -149).all()
    x4 = np.zeros((m, 5 * 64), np.uint8)
    x4[:, 0] = 2
    got = kernels.matmul_mx_swiglu(x4, x[1], *gate, *up).numpy()
    assert (np.abs(got - want) <= 16 * HALF * np.abs(want) + 2.0 ** -126 * np.abs(g) + 2.0 ** -149).all()


SHAPES = [(1, 1, 1), (1, 17, 32), (2, 16, 129), (3, 203, 100), (15, 64, 896), (16, 16, 128), (17, 33, 257), (31, 1, 640),
          (33, 130, 1040), (64, 96, 384), (65, 257, 1000), (130, 131, 512), (300, 65, 130), (1, 896, 4864), (5, 1152, 896),
          (129, 128, 4864), (257, 384, 896), (5, 4997, 1600), (16, 5000, 2177), (50, 1370, 1700), (1, 4513, 4100)]


# many outputs: ragged in rows, columns and steps of 128 (4 to 9 of them)
WIDE = [(1100, 1000, 513), (1030, 1024, 896), (1025, 1090, 768), (1089, 1030, 512), (1030, 1027, 1100), (300, 5003, 640),
        (4100, 4130, 520), (4097, 4099, 896), (4128, 4100, 1024)]


# few outputs and long k, whose k is split over four waves in pairs of steps: 12, 13, 17, 19, 20, 38 steps
LONG = [(330, 1000, 1500), (333, 1001, 1537), (321, 1003, 2176), (350, 997, 2305), (322, 1024, 2560), (352, 1025, 4864)]

# the same with short k
SHORT = [(330, 1001, 1100), (701, 700, 300), (355, 1003, 600)]

# many outputs again: 64 x 64 tiles of eight steps and more, the larger ones, their borders ragged
TILES = [(1300, 1000, 1024), (1281, 1025, 1100), (1300, 1030, 1153), (1281, 1000, 513), (1800, 1900, 1537), (1793, 1921, 2560),
         (3200, 3201, 1100), (3203, 3200, 1024), (3210, 3210, 1300), (3210, 3215, 1537), (2300, 2403, 1100),
         (1650, 1701, 900), (2301, 2400, 4100)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m,n,k", SHAPES + WIDE + LONG + SHORT + TILES)
def test_matmul(gpu, m, n, k, bits):
    check_matmul(m, n, k, bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m,n,k", SHAPES + WIDE + LONG + SHORT + TILES)
def test_swiglu(gpu, m, n, k, bits):
    check_swiglu(m, n, k, bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m", [1, 20, 200])
def test_every_position_of_k_counts_once(gpu, m, bits):
    """One nonzero product a row, at every k in turn, each block's scale its own: exact."""
    from nanocompile_amd import kernels
    k, n = 512, 33
    x, w = np.zeros((k, k), np.float32), np.zeros((n, k), np.float32)
    x[np.arange(k), np.arange(k)] = np.exp2(np.arange(k) // 32 - 8)
    w[:] = np.exp2(np.arange(k) % 4)[None, :] * np.exp2(np.arange(k) // 32 % 5)[None, :] * (1 + np.arange(n) % 2)[:, None]
    wq = mx.quantize(w, 4)
    assert np.array_equal(mx.dequantize(*wq, k), w)
    for first in range(0, k, m):
        rows = x[first:first + m]
        xq = mx.quantize(rows, bits)
        got = kernels.matmul_mx(*xq, *wq).numpy()
        assert np.array_equal(got, rows.astype(np.float64) @ w.T), first
        if first > 3 * m:
            break


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m,n,k", [(1, 100, 896), (40, 70, 300), (200, 300, 256), (1030, 1100, 640)])
def test_bad_blocks_stay_in_their_rows(gpu, m, n, k, bits):
    """A NaN block of x spoils its row of y, one of w its column, and no other output changes a bit."""
    from nanocompile_amd import kernels
    rng = np.random.default_rng(m)
    (xq, xs), (w, u) = operands(rng, m, n, k, bits, 2)
    clean = kernels.matmul_mx(xq, xs, *w).numpy(), kernels.matmul_mx_swiglu(xq, xs, *w, *u).numpy()
    xs, ws, us = xs.copy(), w[1].copy(), u[1].copy()
    xs[m // 2, 1] = ws[n // 3, 0] = us[n - 1, 5] = 255
    got = kernels.matmul_mx(xq, xs, w[0], ws).numpy(), kernels.matmul_mx_swiglu(xq, xs, w[0], ws, u[0], us).numpy()
    for i in range(2):
        bad = np.zeros((m, n), bool)
        bad[m // 2], bad[:, n // 3] = True, True
        if i:
            bad[:, n - 1] = True
        assert np.isnan(got[i][bad]).all()
        assert np.array_equal(float_bits_of(got[i][~bad]), float_bits_of(clean[i][~bad]))


@pytest.mark.parametrize("m,n,k", [(1, 50, 200), (20, 51, 896), (130, 260, 640), (1030, 1101, 640), (7, 4999, 1700)])
def test_residual_in_place_and_guards(gpu, m, n, k):
    """y over the residual, on an address of a float, and nothing written outside it."""
    from nanocompile_amd import hip, kernels
    from nanocompile_amd.hip import DeviceArray
    rng = np.random.default_rng(m)
    x, (w,) = operands(rng, m, n, k, 8)
    residual = rng.standard_normal((m, n)).astype(np.float32)
    bias = rng.standard_normal(n).astype(np.float32)
    want = kernels.matmul_mx(*x, *w, bias, residual).numpy()
    # one float of the buffer on either side besides the guards
    p, read = guarded(residual.nbytes + 8)
    DeviceArray((m, n), np.float32, ptr=p + 4, owner=False).upload(residual)
    dx, ds, dq, dw = (DeviceArray.from_host(a) for a in (*x, *w))
    hip.call("nc_matmul_mx", [p + 4, dx, ds, dq, dw, shifted(bias), p + 4], [m, n, k, 8])
    hip.sync()
    got = read()
    assert same_bits(got[4:-4].view(np.float32).reshape(m, n), want)
    assert (got[:4] == 0xA5).all() and (got[-4:] == 0xA5).all()


# a shape for each kernel of many outputs or long k: k split over waves, 64 x 64 by two steps and by four, the larger
# ones
KINDS = [(330, 1001, 1537), (1281, 1025, 513), (1281, 1025, 1100), (1793, 1921, 1537), (2301, 2403, 1030),
         (3203, 3201, 1030)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m,n,k", KINDS)
def test_every_kind_in_place_with_bad_blocks(gpu, m, n, k, bits):
    """y over the residual between guards, twice the same bits; NaN blocks in the first and the last step spoil their
    row or column and no other output."""
    from nanocompile_amd import hip, kernels
    from nanocompile_amd.hip import DeviceArray
    rng = np.random.default_rng(k)
    (xq, xs), (w, u) = operands(rng, m, n, k, bits, 2)
    residual = rng.standard_normal((m, n)).astype(np.float32)
    bias = rng.standard_normal(n).astype(np.float32)
    dx, dq, du, duq = (DeviceArray.from_host(a) for a in (xq, w[0], u[1], u[0]))
    db, r = DeviceArray.from_host(bias), DeviceArray.from_host(residual)
    clean = kernels.matmul_mx(dx, xs, dq, w[1], db, r).numpy()
    pair = kernels.matmul_mx_swiglu(dx, xs, dq, w[1], duq, du).numpy()
    xs2, ws2 = xs.copy(), w[1].copy()
    xs2[m - 1, (k - 1) // 32] = ws2[n - 1, 0] = xs2[m // 2, 0] = ws2[n // 3, (k - 1) // 32] = 255
    bad = np.zeros((m, n), bool)
    bad[[m // 2, m - 1]], bad[:, [n // 3, n - 1]] = True, True
    for scales in ((xs, w[1]), (xs, w[1]), (xs2, ws2)):
        held = [DeviceArray.from_host(a) for a in scales]
        p, read = guarded(residual.nbytes + 8)
        y = DeviceArray((m, n), np.float32, ptr=p + 4, owner=False)
        y.upload(residual)
        hip.call("nc_matmul_mx", [y, dx, held[0], dq, held[1], db, y], [m, n, k, bits])
        hip.sync()
        whole = read()
        assert (whole[:4] == 0xA5).all() and (whole[-4:] == 0xA5).all()
        got = whole[4:-4].view(np.float32).reshape(m, n)
        h = kernels.matmul_mx_swiglu(dx, held[0], dq, held[1], duq, du).numpy()
        for out, want in ((got, clean), (h, pair)):
            if scales[0] is xs:
                assert np.array_equal(float_bits_of(out), float_bits_of(want))
            else:
                assert np.isnan(out[bad]).all()
                assert np.array_equal(float_bits_of(out[~bad]), float_bits_of(want[~bad]))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m,n,k", KINDS)
def test_every_position_of_k_counts_once_in_every_kind(gpu, m, n, k, bits):
    """One nonzero product a row, row i's at k = i mod K and then at others till every k was: exact."""
    from nanocompile_amd import kernels
    w = np.exp2(np.arange(k) % 4 + np.arange(k) // 32 % 5)[None, :] * (1 + np.arange(n) % 2)[:, None]
    wq = mx.quantize(w.astype(np.float32), 4)
    assert np.array_equal(mx.dequantize(*wq, k), w)
    for first in range(0, k, m):
        at = (first + np.arange(m)) % k
        x = np.zeros((m, k), np.float32)
        x[np.arange(m), at] = np.exp2(at // 32 - 8)
        got = kernels.matmul_mx(*mx.quantize(x, bits), *wq).numpy()
        assert np.array_equal(got, np.exp2(at // 32 - 8)[:, None] * w.T[at]), first


# -- more workgroups than one row of the grid ----------------------------------------------------------


@pytest.mark.parametrize("bits", [4, 8])
def test_long_arrays_of_rows(gpu, bits):
    """140,003 rows of 1,000: the rows about the grid's first border and the last against the definition."""
    from nanocompile_amd import kernels
    from nanocompile_amd.hip import DeviceArray
    m, k = 140003, 1000
    rng = np.random.default_rng(bits)
    x = rng.standard_normal((m, k), dtype=np.float32)
    q, scales = kernels.quantize_mx(DeviceArray.from_host(x), bits)
    back = kernels.dequantize_mx(q, scales, k).numpy()
    q, scales = q.numpy(), scales.numpy()
    per_row = 1024
    for values in (8, 4):                              # a thread's, in one kernel and the other
        border = 65536 * 256 * values // per_row
        for rows in (slice(0, 3), slice(border - 2, border + 3), slice(m - 3, m)):
            want = mx.quantize(x[rows], bits)
            assert np.array_equal(q[rows], want[0]) and np.array_equal(scales[rows], want[1])
            assert same_bits(back[rows], mx.dequantize(*want, k))


@pytest.mark.parametrize("mx_bits", [0, 8])
def test_norm_of_many_rows(gpu, mx_bits):
    from nanocompile_amd import kernels
    m, k = 4 * 65536 + 70, 5
    rng = np.random.default_rng(mx_bits)
    x, gamma = rng.standard_normal((m, k)).astype(np.float32), np.ones(k, np.float32)
    t, _, q, qs = kernels.add_rms_norm_quant(x, None, gamma, 1e-6, mx_bits=mx_bits)
    _, n = mx.norm(x, None, gamma, 1e-6)
    want = mx.quantize(n, 8) if mx_bits else R.quantize_token(n)
    assert np.array_equal(q.numpy(), want[0]) and same_bits(qs.numpy(), want[1])


@pytest.mark.parametrize("m,n,k", [(3, 1200017, 40), (16500, 16400, 600)])
def test_products_of_many_tiles(gpu, m, n, k):
    """75,002 tiles of 16 x 16, 66,306 of 64 x 64: whole rows about the borders against the definition."""
    from nanocompile_amd import kernels
    x, (w,) = operands(np.random.default_rng(m), m, n, k, 4)
    y = kernels.matmul_mx(*x, *w).numpy()
    for rows in ([0, m - 1], [m // 2]):
        for columns in (slice(0, 300), slice(n // 2, n // 2 + 300), slice(n - 300, n)):
            want, size = mx.matmul(x[0][rows], x[1][rows], w[0][columns], w[1][columns])
            assert (np.abs(y[rows, columns] - want) <= product_error(size, k, 4)).all()
    assert np.isfinite(y).all()
    x[1][:] = w[1][:] = 127                            # every scale 1, all elements: no output is left unwritten
    x[0][:] = w[0][:] = 0x22                           # ones
    ones = kernels.matmul_mx(*x, *w).numpy()
    assert (ones == x[0].shape[1] * 2).all()


# -- together ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("m", [1, 7, 150])
def test_a_blocks_mlp(gpu, m):
    """A decoder block's MLP as these operators run it: residual and norm, gate and up, quantizer, down with the
    residual; each step against its definition on the step's own inputs, and the whole captured and replayed."""
    from nanocompile_amd import hip, kernels
    from nanocompile_amd.hip import DeviceArray
    rng = np.random.default_rng(m)
    h, inner = 896, 1216
    x, delta = activations(rng, m, h), rng.standard_normal((m, h)).astype(np.float32)
    gamma = (1 + 0.1 * rng.standard_normal(h)).astype(np.float32)
    weights = [kernels.quantize_mx((rng.standard_normal(s) * 0.02).astype(np.float32))
               for s in ((inner, h), (inner, h), (h, inner))]
    host = [tuple(a.numpy() for a in w) for w in weights]
    t, _, q, qs = kernels.add_rms_norm_quant(x, delta, gamma, 1e-6, mx_bits=8)
    mid = kernels.matmul_mx_swiglu(q, qs, *weights[0], *weights[1])
    mq, ms = kernels.quantize_mx(mid, 8)
    y = kernels.matmul_mx(mq, ms, *weights[2], residual=t)
    want_t, n = mx.norm(x, delta, gamma, 1e-6)
    assert same_bits(t.numpy(), want_t)
    assert all(np.array_equal(a.numpy(), b) for a, b in zip((q, qs), mx.quantize(n, 8)))
    want, (g, u, gs, us) = mx.swiglu(q.numpy(), qs.numpy(), *host[0], *host[1])
    dg, du = product_error(gs, h, 8), product_error(us, h, 8)
    assert (np.abs(mid.numpy() - want) <= 1.1 * dg * (np.abs(u) + du) + np.abs(g) * du + 16 * HALF * np.abs(want)
            + 1e-37).all()
    assert all(np.array_equal(a.numpy(), b) for a, b in zip((mq, ms), mx.quantize(mid.numpy(), 8)))
    want, size = mx.matmul(mq.numpy(), ms.numpy(), *host[2], residual=t.numpy())
    assert (np.abs(y.numpy() - want) <= product_error(size, inner, 8)).all()

    # the same four calls captured, the residual stream updated in place, replayed on new inputs
    dx, dd, dg_, out = DeviceArray((m, h), np.float32), DeviceArray.from_host(delta), DeviceArray.from_host(gamma), []
    g1 = hip.Graph.capture(lambda: (
        hip.call("nc_add_rms_norm_quant", [dx, None, q, qs, dx, dd, dg_], [m, h, kernels.float_bits(1e-6), 8]),
        hip.call("nc_matmul_mx_swiglu", [mid, q, qs, *weights[0], *weights[1]], [m, inner, h, 8]),
        hip.call("nc_quantize_mx", [mq, ms, mid], [m, inner, 8]),
        hip.call("nc_matmul_mx", [dx, mq, ms, *weights[2], None, dx], [m, h, inner, 8])))
    for _ in range(3):
        dx.upload(x)
        g1.launch()
        hip.sync()
        out.append(dx.numpy())
        kernels.quantize_mx(x, 4)                         # other work in between
    assert all(same_bits(o, y.numpy()) for o in out)
