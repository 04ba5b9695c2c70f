"""The microscaled operators without a GPU: the oracle's own checks, and every call that is refused."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle import mx

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def test_oracle_elements_by_hand():
    """A block whose largest value is in 4 .. 8 has scale 1: every e2m1 value, its borders, and what is past 6."""
    row = np.zeros((1, 32), np.float32)
    row[0, :15] = [6, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 5.01, 7.9, -0.5, -2.49, -0.0, 4]
    codes, scales = mx.quantize(row, 4)
    assert codes.shape == (1, 64) and scales.tolist() == [[127, 0, 0, 0]]
    want = [6, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6, -0.5, -2, 0, 4]
    assert mx.dequantize(codes, scales, 15)[0].tolist() == want
    assert codes[0, 0] & 15 == 7 and codes[0, 6] >> 4 == 8                   # -0.0 keeps its sign


def test_oracle_codes_are_the_values_in_order():
    for bits, count in ((4, 8), (8, 127)):
        every = np.arange(count, dtype=np.uint8)
        codes = np.zeros((1, 64 * bits // 4), np.uint8)
        codes[0, :count if bits == 8 else count // 2] = every if bits == 8 else every[0::2] | every[1::2] << 4
        values = mx.dequantize(codes, np.full((1, 4), 127, np.uint8), count)[0]
        assert (np.diff(values) > 0).all() and values[0] == 0 and values[-1] == (6 if bits == 4 else 448)
        if bits == 4:
            assert values.tolist() == E2M1


def test_oracle_agrees_with_torch_casts():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((64, 160)) * np.exp(4 * rng.standard_normal((64, 160)))).astype(np.float32)
    codes, scales = mx.quantize(x, 8)
    power = np.exp2(scales.astype(np.float64) - 127)
    t = mx._blocks(x) / power[:, :, None]
    cast = torch.from_numpy(t.clip(-448, 448).astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8)
    assert np.array_equal(cast.numpy().reshape(codes.shape), codes)


@pytest.mark.parametrize("bits", [4, 8])
def test_oracle_special_blocks(bits):
    x = np.zeros((4, 32), np.float32)
    x[1, 3], x[2, 0], x[3, 31] = np.nan, np.inf, 1e-45
    codes, scales = mx.quantize(x, bits)
    assert scales[:, 0].tolist() == [0, 255, 255, 0] and not codes[:3].any()
    assert np.isnan(mx.dequantize(codes, scales, 32)[1:3]).all()
    big = np.full((1, 32), np.finfo(np.float32).max, np.float32)
    assert mx.quantize(big, bits)[1][0, 0] == 254 - (2 if bits == 4 else 8)


# -- refusals: checked before anything reaches a GPU ----------------------------------------

P = 1 << 20          # stands for an aligned device address; no call below gets as far as reading it


@pytest.fixture(scope="module")
def call():
    from nanocompile_amd import build, hip
    if not build.LIBRARY.exists():
        build.build()
    hip.load()

    def go(name, pointers, sizes):
        p = (ctypes.c_void_p * 16)(*pointers)
        s = (ctypes.c_int64 * 16)(*sizes)
        return hip.kernel(name)(p, s), hip.last_error()
    return go


CALLS = {
    "nc_quantize_mx": ([P, P, P], [2, 64, 4]),
    "nc_dequantize_mx": ([P, P, P], [2, 64, 4]),
    "nc_add_rms_norm_quant": ([P, P, P, P, P, P, P], [2, 64, 0, 8]),
    "nc_matmul_mx": ([P, P, P, P, P, P, P], [2, 64, 64, 8]),
    "nc_matmul_mx_swiglu": ([P, P, P, P, P, P, P], [2, 64, 64, 8]),
}
NEEDED = {"nc_quantize_mx": (0, 1, 2), "nc_dequantize_mx": (0, 1, 2), "nc_add_rms_norm_quant": (2, 3, 4, 6),
          "nc_matmul_mx": (0, 1, 2, 3, 4), "nc_matmul_mx_swiglu": (0, 1, 2, 3, 4, 5, 6)}
CODES = {"nc_quantize_mx": (0,), "nc_dequantize_mx": (1,), "nc_add_rms_norm_quant": (2,), "nc_matmul_mx": (1, 3),
         "nc_matmul_mx_swiglu": (1, 3, 5)}
SCALES = {"nc_quantize_mx": (1,), "nc_dequantize_mx": (2,), "nc_add_rms_norm_quant": (3,), "nc_matmul_mx": (2, 4),
          "nc_matmul_mx_swiglu": (2, 4, 6)}


@pytest.mark.parametrize("name", CALLS)
def test_refusals(call, name):
    pointers, sizes = CALLS[name]

    def refused(text, at=None, pointer=None, size=None):
        p, s = list(pointers), list(sizes)
        if pointer is not None:
            p[at] = pointer or None
        if size is not None:
            s[at] = size
        status, message = call(name, p, s)
        assert status == 2 and name in message and text in message, (at, pointer, size, status, message)

    for at in NEEDED[name]:
        refused("null operand", at, pointer=0)
    for at, _ in enumerate(sizes):
        bits = at == len(sizes) - 1
        if name == "nc_add_rms_norm_quant" and at == 2:
            continue                                       # eps: any float
        for bad in (-1, 1 << 26) if at == 0 else (0, -1, (1 << 24) + 1) if at == 2 and "matmul" in name else (3, 5, 16) if bits else (0, -1, 1 << 26):
            refused("bits" if bits and name != "nc_add_rms_norm_quant" else "format" if bits else "bad shape", at,
                    size=bad)
    for at in CODES[name]:
        refused("alignment", at, pointer=P + 8)
    for at in SCALES[name]:
        refused("alignment", at, pointer=P + 2)
    if name == "nc_add_rms_norm_quant":
        refused("bad shape", 1, size=32769)


@pytest.mark.parametrize("name", CALLS)
def test_no_rows_is_no_work(call, name):
    pointers, sizes = CALLS[name]
    assert call(name, pointers, [0] + sizes[1:])[0] == 0


def test_too_many_outputs_are_refused(call):
    for name in ("nc_matmul_mx", "nc_matmul_mx_swiglu"):
        status, message = call(name, CALLS[name][0], [1 << 20, 1 << 20, 64, 8])
        assert status == 2 and "bad shape" in message


def test_wrappers_refuse_shapes_before_any_copy():
    from nanocompile_amd import kernels as K
    f = np.zeros((2, 64), np.float32)
    gamma = np.ones(64, np.float32)
    with pytest.raises(ValueError, match="4 or 8 bits"):
        K.quantize_mx(f, 5)
    with pytest.raises(K.ShapeError, match="f32"):
        K.quantize_mx(f.astype(np.float64))
    with pytest.raises(K.ShapeError, match="f32"):
        K.quantize_mx(f[0])
    with pytest.raises(ValueError, match="mx_bits"):
        K.add_rms_norm_quant(f, f, gamma, 1e-6, mx_bits=6)

    def codes(rows, steps, bits):
        return np.zeros((rows, steps * 16 * bits), np.uint8), np.zeros((rows, steps * 4), np.uint8)

    x, w = codes(2, 1, 8), codes(3, 1, 4)
    with pytest.raises(K.ShapeError, match="codes"):
        K.dequantize_mx(x[0], w[1], 64)
    with pytest.raises(K.ShapeError, match="codes"):
        K.matmul_mx(x[0][:, :100], x[1], *w)
    with pytest.raises(K.ShapeError, match="codes"):
        K.matmul_mx_swiglu(x[0][0], x[1], *w, *w)
