"""What the microscaled (MX) operators are timed on: calls a user's program makes, over the sizes it makes them at.

MX formats hold a row as blocks of 32 values, each block a power of two (one byte, its exponent plus 127;
255 is NaN) times 4-bit (e2m1) or 8-bit (e4m3) floating point elements. Rows are padded to a multiple of 128
values with zeros; two 4-bit elements share a byte, the lower index in the low bits. The operators: a quantizer,
its inverse, the residual's addition with rms_norm and an 8-bit (or 4-bit) output, the projection of quantized
activations by 4-bit weights, and SwiGLU's pair of projections.

A case is one pass on operands already on the GPU. With ``own`` false it runs as elementary torch operations.
Sizes are the model's (hidden 896, intermediate 4,864, 14 query heads over 2 KV heads of 64) and generic ones.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6
H, I, QKV = 896, 4864, 1152
BLOCK, PAD = 32, 128
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # The smallest call: one token's gate projection, where latency and the launch count.
        {"name": "linear 1", "kind": "linear", "rows": 1, "n": I, "k": H, "bits": 8, "bias": True, "residual": False},
        # Eight sequences decoded together at a wide layer: the weights' bytes count.
        {"name": "linear 8 wide", "kind": "linear", "rows": 8, "n": 8192, "k": 8192, "bits": 8, "bias": False,
         "residual": False},
        # A prompt's down projection with its residual.
        {"name": "linear 512", "kind": "linear", "rows": 512, "n": H, "k": I, "bits": 8, "bias": False,
         "residual": True},
        # A batch of prompts at a wide layer, activations in 4 bits too: operations count.
        {"name": "linear 4096 wide", "kind": "linear", "rows": 4096, "n": 8192, "k": 8192, "bits": 4, "bias": True,
         "residual": False},
        # One token's gate and up with SwiGLU.
        {"name": "swiglu 1", "kind": "swiglu", "rows": 1, "n": I, "k": H, "bits": 8},
        # Gate and up with SwiGLU over a ragged prompt.
        {"name": "swiglu 1000", "kind": "swiglu", "rows": 1000, "n": I, "k": H, "bits": 8},
        # One token's residual and norm before the int8 projections, the residual stream updated.
        {"name": "norm 1 int8", "kind": "norm", "rows": 1, "k": H, "format": 0, "delta": True},
        # A batch of prompts' residual and norm before the MX projections.
        {"name": "norm 4096 mx8", "kind": "norm", "rows": 4096, "k": 4096, "format": 8, "delta": True},
        # A prompt's SwiGLU output before the down projection.
        {"name": "quantize 1000 mx8", "kind": "quantize", "rows": 1000, "k": I, "bits": 8},
        # A weight of an odd width to 4 bits and the values it then stands for, as its error is looked at.
        {"name": "quantize odd mx4", "kind": "quantize", "rows": 2731, "k": 1003, "bits": 4},
        # A prompt's 8-bit activations back to float32.
        {"name": "dequantize 100 mx8", "kind": "dequantize", "rows": 100, "k": H, "bits": 8},
        # A wide layer's weight back to float32.
        {"name": "dequantize 8192 mx4", "kind": "dequantize", "rows": 8192, "k": 8192, "bits": 4},
    ]


def _log(rng, low, high):
    """A whole number, its logarithm spread evenly over low .. high."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "swiglu", "swiglu", "norm", "norm", "quantize", "dequantize"])
    if kind in ("linear", "swiglu"):
        # the model's projections half of the time, else any width, odd ones among them
        model = [(QKV, H), (H, H), (I, H), (H, I)] if kind == "linear" else [(I, H)]
        n, k = rng.choice(model) if rng.random() < 0.5 else (_log(rng, 16, 8192), _log(rng, 32, 8192))
        case = {"kind": kind, "rows": _log(rng, 1, max(1, min(4096, (1 << 37) // (n * k)))), "n": n, "k": k,
                "bits": rng.choice([4, 8])}
        if kind == "linear":
            case.update(bias=rng.random() < 0.5, residual=rng.random() < 0.5)
        return case
    k = H if rng.random() < 0.3 else _log(rng, 32, 8192)
    rows = _log(rng, 1, min(8192, (1 << 25) // k))
    if kind == "norm":
        return {"kind": kind, "rows": rows, "k": k, "format": rng.choice([0, 4, 8]), "delta": rng.random() < 0.7}
    return {"kind": kind, "rows": rows, "k": k, "bits": rng.choice([4, 8])}


# -- inputs ---------------------------------------------------------------------------


def _padded(k):
    return -(-k // PAD) * PAD


class _Made:
    """Seeded arrays on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed * 2 + 1)

    def normal(self, *shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=self.g)

    def activations(self, rows, k):
        """Normal with one element in a hundred twenty times larger, as a residual stream has."""
        x = self.normal(rows, k)
        big = torch.empty((rows, k), device="cuda").uniform_(generator=self.g) < 0.01
        return torch.where(big, 20 * x, x)

    def held(self, x, bits):
        """Codes and scales of ``x`` as they lie in memory: uint8 [rows, padded k * bits / 8], [rows, padded k / 32]."""
        codes, scales = _quantize(x, bits)
        if bits == 4:
            codes = codes[:, 0::2] | codes[:, 1::2] << 4
        return codes.contiguous(), scales


def _operands(case, seed):
    made, kind = _Made(seed), case["kind"]
    m, k = case["rows"], case["k"]
    if kind == "quantize":
        return {"x": made.activations(m, k)}
    if kind == "dequantize":
        codes, scales = made.held(made.normal(m, k, std=0.02), case["bits"])
        return {"codes": codes, "scales": scales}
    if kind == "norm":
        return {"x": made.activations(m, k), "delta": made.normal(m, k) if case["delta"] else None,
                "gamma": 1 + made.normal(k, std=0.1)}
    n = case["n"]
    got = dict(zip(("xq", "xs"), made.held(made.activations(m, k), case["bits"])))
    for name in ("w",) if kind == "linear" else ("g", "u"):
        got[name + "q"], got[name + "s"] = made.held(made.normal(n, k, std=0.02), 4)
    if kind == "linear":
        got["bias"] = made.normal(n) if case["bias"] else None
        got["residual"] = made.normal(m, n) if case["residual"] else None
    return got


def prepare(case, seed):
    """The operands, and the buffers that a user's program writes its results to."""
    x = _operands(case, seed)
    m, k, kind = case["rows"], case["k"], case["kind"]

    def new(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda")

    bits = case.get("bits", case.get("format"))
    if kind in ("linear", "swiglu"):
        x["y"] = new(m, case["n"])
    elif kind == "dequantize":
        x["values"] = new(m, k)
    elif bits:
        x["codes"] = new(m, _padded(k) * bits // 8, dtype=torch.uint8)
        x["scales"] = new(m, _padded(k) // BLOCK, dtype=torch.uint8)
        x["values"] = new(m, k) if bits == 4 else None
    else:
        x["codes"], x["scales"] = new(m, k, dtype=torch.int8), new(m)
    x["sum"] = new(m, k) if kind == "norm" and case["delta"] else None
    return {"case": case, **x}


# -- the plain forms --------------------------------------------------------------------


def _quantize(x, bits):
    """(element codes uint8 [rows, padded], scales uint8 [rows, padded / 32]) of float32 rows."""
    m, k = x.shape
    b = torch.zeros((m, _padded(k)), device=x.device)
    b[:, :k] = x
    b = b.view(m, -1, BLOCK)
    largest = b.abs().amax(2)
    # the block's power of two puts its largest value into the elements' top binade (4 .. 8, 256 .. 512)
    exponent = (largest.view(torch.int32) >> 23) - (2 if bits == 4 else 8)
    scales = exponent.clamp(min=0)
    inverse = ((254 - scales) << 23).view(torch.float32)
    t = b * inverse[:, :, None]
    if bits == 4:
        a = t.abs()
        # nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6; a tie goes to the even code
        code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)).byte()
        code = code + torch.signbit(t).byte() * 8
    else:
        code = t.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return code.view(m, -1), scales.to(torch.uint8)


def _values(codes, scales, bits, k):
    """Float32 values of codes and scales as they lie in memory."""
    m = codes.shape[0]
    if bits == 4:
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
        v = table[torch.stack((codes & 15, codes >> 4), 2).view(m, -1).int()]
    else:
        v = codes.view(torch.float8_e4m3fn).float()
    power = torch.exp2(scales.double() - 127).float()
    return (v.view(m, -1, BLOCK) * power[:, :, None]).view(m, -1)[:, :k]


def _silu(g):
    return g / (1 + torch.exp(-g))


def _quantized(x, bits):
    """What a pass returns of a quantized ``x``: its values in 4 bits, elements and scales in 8."""
    codes, scales = _quantize(x, bits)
    if bits == 8:
        return [codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)]
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=x.device)
    power = torch.exp2(scales.double() - 127).float()
    return [(table[codes.int()].view(x.shape[0], -1, BLOCK) * power[:, :, None]).view(x.shape[0], -1)[:, :x.shape[1]]]


def _plain(s):
    case = s["case"]
    kind, k = case["kind"], case["k"]
    if kind == "quantize":
        return _quantized(s["x"], case["bits"])
    if kind == "dequantize":
        return [_values(s["codes"], s["scales"], case["bits"], k)]
    if kind == "norm":
        x = s["x"] if s["delta"] is None else s["x"] + s["delta"]
        # in 64 bits, so that no value next to a rounding border depends on the order of the sum
        square = x.double().square().sum(1, keepdim=True) / k
        n = x * (1 / torch.sqrt(square + float(np.float32(EPS)))).float() * s["gamma"]
        kept = [] if s["delta"] is None else [x]
        if case["format"]:
            return kept + _quantized(n, case["format"])
        largest = n.abs().amax(1, keepdim=True)
        scale = (largest.double() / 127).float()
        scale = torch.where(scale <= 0, torch.ones_like(scale), scale)
        r = (n.double() / scale.double()).float()
        r = torch.sign(r) * torch.floor(r.abs().double() + 0.5).float()          # ties away from zero
        return kept + [r.clamp(-127, 127).to(torch.int8), scale[:, 0]]
    x = _values(s["xq"], s["xs"], case["bits"], k)
    if kind == "swiglu":
        return [_silu(x @ _values(s["gq"], s["gs"], 4, k).T) * (x @ _values(s["uq"], s["us"], 4, k).T)]
    y = x @ _values(s["wq"], s["ws"], 4, k).T
    if s["bias"] is not None:
        y = y + s["bias"]
    return [y if s["residual"] is None else s["residual"] + y]


# -- a pass -------------------------------------------------------------------------------


def _at(t):
    return None if t is None else t.data_ptr()


def _own(s):
    from nanocompile_amd import hip
    case = s["case"]
    kind, m, k = case["kind"], case["rows"], case["k"]
    if kind == "linear":
        hip.call("nc_matmul_mx", [_at(s["y"]), _at(s["xq"]), _at(s["xs"]), _at(s["wq"]), _at(s["ws"]), _at(s["bias"]),
                                  _at(s["residual"])], [m, case["n"], k, case["bits"]])
        return [s["y"]]
    if kind == "swiglu":
        hip.call("nc_matmul_mx_swiglu", [_at(s["y"]), _at(s["xq"]), _at(s["xs"]), _at(s["gq"]), _at(s["gs"]),
                                         _at(s["uq"]), _at(s["us"])], [m, case["n"], k, case["bits"]])
        return [s["y"]]
    if kind == "dequantize":
        hip.call("nc_dequantize_mx", [_at(s["values"]), _at(s["codes"]), _at(s["scales"])], [m, k, case["bits"]])
        return [s["values"]]
    kept = []
    if kind == "quantize":
        bits = case["bits"]
        hip.call("nc_quantize_mx", [_at(s["codes"]), _at(s["scales"]), _at(s["x"])], [m, k, bits])
    else:
        bits = case["format"]
        hip.call("nc_add_rms_norm_quant", [_at(s["sum"]), None, _at(s["codes"]), _at(s["scales"]), _at(s["x"]),
                                           _at(s["delta"]), _at(s["gamma"])],
                 [m, k, int(np.float32(EPS).view(np.uint32)), bits])
        kept = [] if s["sum"] is None else [s["sum"]]
    if bits == 0:
        return kept + [s["codes"], s["scales"]]
    if bits == 8:
        return kept + [s["codes"].view(torch.float8_e4m3fn), s["scales"].view(torch.float8_e8m0fnu)]
    hip.call("nc_dequantize_mx", [_at(s["values"]), _at(s["codes"]), _at(s["scales"])], [m, k, bits])
    return kept + [s["values"]]


def run(state):
    return _own(state) if own else _plain(state)


# -- what a pass cannot do without, and what it should give ---------------------------------


def work(case):
    m, k, kind = case["rows"], case["k"], case["kind"]

    def held(rows, bits):
        return rows * _padded(k) * bits // 8 + rows * _padded(k) // BLOCK

    if kind in ("linear", "swiglu"):
        n, pair = case["n"], 2 if kind == "swiglu" else 1
        extra = 4 * n * case.get("bias", False) + 4 * m * n * case.get("residual", False)
        return {"bytes": held(m, case["bits"]) + pair * held(n, 4) + extra + 4 * m * n, "flops": 2 * pair * m * n * k}
    if kind == "dequantize":
        return {"bytes": held(m, case["bits"]) + 4 * m * k, "flops": m * k}
    if kind == "quantize":
        return {"bytes": 4 * m * k + (held(m, 8) if case["bits"] == 8 else 4 * m * k), "flops": 2 * m * k}
    out = {0: m * k + 4 * m, 8: held(m, 8), 4: 4 * m * k}[case["format"]]
    return {"bytes": 4 * m * k * (3 if case["delta"] else 1) + 4 * k + out, "flops": 6 * m * k}


def _element(t, bits):
    """The nearest element value to each of ``t`` (float64), by its binade's step; ties to even, largest kept."""
    least, mantissa, top = (0, 1, 6.0) if bits == 4 else (-6, 3, 448.0)
    e = torch.frexp(t.abs())[1].double() - 1
    step = torch.exp2(torch.clamp(e, min=least) - mantissa)
    return torch.round(t / step).mul(step).clamp(-top, top)


def _held_exact(n, bits):
    """Elements [rows, padded] and powers of two [rows, blocks] of float64 rows."""
    m, k = n.shape
    b = torch.nn.functional.pad(n, (0, _padded(k) - k)).view(m, -1, BLOCK)
    e = torch.frexp(b.abs().amax(2))[1].double() - 1 - (2 if bits == 4 else 8)
    power = torch.exp2(torch.where(b.abs().amax(2) == 0, torch.full_like(e, -127), e.clamp(min=-127)))
    return _element(b / power[:, :, None], bits), power


def _quantized_exact(n, bits):
    element, power = _held_exact(n, bits)
    if bits == 8:
        return [element.view(n.shape[0], -1), power]
    return [(element * power[:, :, None]).view(n.shape[0], -1)[:, :n.shape[1]]]


def _decoded(codes, scales, bits, k):
    """Float64 values from the bits of each element: sign, exponent, mantissa."""
    c = codes.int()
    if bits == 4:
        c = torch.stack((c & 15, c >> 4), 2).view(c.shape[0], -1)
    low, bias = (1, 1) if bits == 4 else (3, 7)
    e, f = (c >> low) & (3 if bits == 4 else 15), (c & ((1 << low) - 1)).double() / (1 << low)
    v = torch.where(e > 0, (1 + f) * torch.exp2(e.double() - bias), f * 2.0 ** (1 - bias))
    v = torch.where((c >> (bits - 1)) > 0, -v, v)
    return (v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1))[:, :k]


def exact(case, seed):
    x, kind, k = _operands(case, seed), case["kind"], case["k"]
    if kind == "quantize":
        return _quantized_exact(x["x"].double(), case["bits"])
    if kind == "dequantize":
        return [_decoded(x["codes"], x["scales"], case["bits"], k)]
    if kind == "norm":
        a = x["x"].double()
        if x["delta"] is not None:
            a = a + x["delta"].double()
        n = a * torch.rsqrt((a * a).mean(1, keepdim=True) + EPS) * x["gamma"].double()
        kept = [] if x["delta"] is None else [a]
        if case["format"] == 0:
            return kept + [None, n.abs().amax(1) / 127]          # the int8 values are whole numbers
        if case["format"] == 4:
            # a value next to a rounding border moves by a whole step on float32's last bit
            return kept + [None]
        return kept + _quantized_exact(n, 8)
    a = _decoded(x["xq"], x["xs"], case["bits"], k)
    if kind == "swiglu":
        g, u = (a @ _decoded(x[w + "q"], x[w + "s"], 4, k).T for w in "gu")
        return [g * torch.sigmoid(g) * u]
    y = a @ _decoded(x["wq"], x["ws"], 4, k).T
    if x["bias"] is not None:
        y = y + x["bias"].double()
    return [y if x["residual"] is None else x["residual"].double() + y]
