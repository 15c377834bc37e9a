"""Workloads of the microscaled (MX) operators: quantising rows to 4- or 8-bit floating point with a power-of-two scale for
every 32 consecutive values, the product of such rows with 4-bit weights, and the two steps in front of a product that leave
their result in this form: the residual addition with RMSNorm, and SiLU(gate) * up.

Sizes are those of the Qwen3 layers that this repository configures, tests and benchmarks.

The format.  A block of 32 values v has one scale 2^e, held as the byte e + 127, and 32 elements q: e2m1 (largest value 6,
"mxfp4", two codes a byte, the first in the low half) or e4m3 (largest value 448, "mxfp8").  e is the smallest exponent with
which the block's largest magnitude, rounded to the nearest element, is not past the largest element, and at least -127; the
elements are v / 2^e rounded to nearest, ties to even.  A block that holds an infinity or a NaN has the byte 255 and stands
for NaN."""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
BLOCK = 32
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
CODE_BYTES = {"mxfp4": 0.5, "mxfp8": 1.0}
MOST_PRODUCT = 8192 * 4096 * 12288
MOST_WEIGHT = 25600 * 5120
F64 = torch.float64


def _quantize(name, rows, k, dtype, fmt):
    return {"name": name, "kind": "quantize", "rows": rows, "k": k, "dtype": dtype, "format": fmt}


def _linear(name, rows, k, n, dtype, fmt="mxfp8", bias=False):
    return {"name": name, "kind": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "format": fmt, "bias": bias}


def _product(name, rows, k, n, dtype, fmt, bias=False):
    return {"name": name, "kind": "product", "rows": rows, "k": k, "n": n, "dtype": dtype, "format": fmt, "bias": bias}


def _norm(name, rows, k, dtype, fmt="mxfp8"):
    return {"name": name, "kind": "norm", "rows": rows, "k": k, "dtype": dtype, "format": fmt}


def _silu(name, rows, k, dtype, fmt="mxfp8"):
    return {"name": name, "kind": "silu", "rows": rows, "k": k, "dtype": dtype, "format": fmt}


def listed():
    return [
        # a few tokens' activations on their way into a product, and back: launch and host latency
        _quantize("quantize_3x2560_f16_mxfp8", 3, 2560, "f16", "mxfp8"),
        # one weight of a large checkpoint to 4 bits, and its values for a caller that wants them dense
        _quantize("quantize_25600x5120_bf16_mxfp4", 25600, 5120, "bf16", "mxfp4"),
        # one sequence decoding: an MLP projection of a small model, activations as they are
        _linear("linear_1x2560x9728_bf16", 1, 2560, 9728, "bf16"),
        # sixteen sequences decoding through an MLP projection of the largest model
        _linear("linear_16x5120x25600_f16", 16, 5120, 25600, "f16"),
        # a batch of prompts through an MLP projection, activations as they are
        _linear("linear_8192x4096x12288_bf16", 8192, 4096, 12288, "bf16"),
        # an odd number of sequences decoding through the largest model's other MLP projection, activations from the step before
        _product("product_41x25600x5120_bf16_mxfp8", 41, 25600, 5120, "bf16", "mxfp8"),
        # a short ragged prompt, an odd output width, a bias
        _product("product_333x2816x9727_f16_mxfp8_bias", 333, 2816, 9727, "f16", "mxfp8", True),
        # a batch of prompts with activations of 4 bits
        _product("product_8192x4096x12288_bf16_mxfp4", 8192, 4096, 12288, "bf16", "mxfp4"),
        # between two blocks of one decoding sequence
        _norm("norm_1x4096_bf16_mxfp8", 1, 4096, "bf16"),
        # the same for a batch of prompts of the largest model
        _norm("norm_8192x5120_bf16_mxfp8", 8192, 5120, "bf16"),
        # an MLP's activation for seven sequences that decode
        _silu("silu_7x9728_f16_mxfp8", 7, 9728, "f16"),
        # the same for a batch of prompts, to 4 bits
        _silu("silu_8192x12288_bf16_mxfp4", 8192, 12288, "bf16", "mxfp4"),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "product", "norm", "silu"])
    fmt = rng.choice(["mxfp4", "mxfp8"])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "quantize":
        k = BLOCK * _between(rng, 1, 800)
        return {"kind": kind, "rows": _between(rng, 1, MOST_WEIGHT // k), "k": k, "dtype": rng.choice(["f16", "bf16", "f32"])
                if k * 25600 <= MOST_WEIGHT // 2 else dtype, "format": fmt}
    if kind in ("norm", "silu"):
        return {"kind": kind, "rows": _between(rng, 1, 8192), "k": BLOCK * _between(rng, 2, 160 if kind == "norm" else 384),
                "dtype": dtype, "format": fmt}
    k = BLOCK * _between(rng, 2, 800)
    n = _between(rng, 16, min(25600, MOST_WEIGHT // k))
    rows = _between(rng, 1, max(1, min(8192, MOST_PRODUCT // (k * n))))
    return {"kind": kind, "rows": rows, "k": k, "n": n, "dtype": dtype, "format": fmt, "bias": rng.random() < 0.3}


# ---- the operators in their plain form ----------------------------------------------------------------------------------
def _power(byte):
    """2^(byte - 127) for the bytes of a scale: its bits are those of the 32-bit float's exponent."""
    bits = byte.to(torch.int32) << 23
    bits = torch.where(byte == 0, 0x00400000, bits)
    return torch.where(byte == 255, 0x7FC00000, bits).view(torch.float32)


def _plain_quantize(x, fmt):
    blocks = x.float().unflatten(-1, (-1, BLOCK))
    largest = blocks.abs().amax(-1)
    four = fmt == "mxfp4"
    # the exponent of 1.75 * 2^n and above (e2m1) or of more than 1.8125 * 2^n (e4m3) is n + 1: rounded, it would be
    byte = ((largest.view(torch.int32) + (0x200000 if four else 0x17FFFF)) >> 23) - (2 if four else 8)
    bad = ~torch.isfinite(blocks).all(-1)
    byte = torch.where(bad, 255, byte.clamp_min(0))
    inverse = ((254 - byte).clamp_min(1) << 23).view(torch.float32)
    scaled = torch.where(bad.unsqueeze(-1), 0.0, blocks * inverse.unsqueeze(-1)).flatten(-2)
    if not four:
        return scaled.to(torch.float8_e4m3fn).view(torch.uint8), byte.to(torch.uint8)
    m = scaled.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)
            + (torch.signbit(scaled).to(torch.uint8) << 3))
    pairs = code.unflatten(-1, (-1, 2))
    return pairs[..., 0] | (pairs[..., 1] << 4), byte.to(torch.uint8)


def _plain_values(codes, scales):
    if codes.shape[-1] == BLOCK * scales.shape[-1]:
        element = codes.view(torch.float8_e4m3fn).float()
    else:
        code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
        m = (code & 7).float()
        m = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, 2 * m - 8))
        element = torch.where(code >= 8, -m, m)
    return (element.unflatten(-1, (-1, BLOCK)) * _power(scales).unsqueeze(-1)).flatten(-2)


def _plain_product(values, state):
    y = values @ _plain_values(state["weight"], state["weight_scales"]).t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["dtype"])


# ---- what a program has in hand before the call -------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, rows, k, dtype):
    """Normal values whose channels have spreads of their own, a few of them large, as hidden states have."""
    spread = torch.exp(0.5 * torch.randn(k, device="cuda", generator=g))
    return (torch.randn(rows, k, device="cuda", generator=g) * spread).to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    kind, rows, k, dtype = case["kind"], case["rows"], case["k"], DTYPES[case["dtype"]]
    state = {"kind": kind, "format": case["format"], "dtype": dtype}
    if kind == "norm":
        state["x"] = _activations(g, rows, k, dtype)
        state["delta"] = torch.randn(rows, k, device="cuda", generator=g).to(dtype)
        state["weight"] = (1 + 0.1 * torch.randn(k, device="cuda", generator=g)).to(dtype)
        return state
    if kind == "silu":
        state["gate"] = (2 * torch.randn(rows, k, device="cuda", generator=g)).to(dtype)
        state["up"] = _activations(g, rows, k, dtype)
        return state
    state["x"] = _activations(g, rows, k, dtype)
    if kind == "quantize":
        return state
    n = case["n"]
    weight = torch.randn(n, k, device="cuda", generator=g) * k ** -0.5
    state["weight"], state["weight_scales"] = _plain_quantize(weight, "mxfp4")
    state["bias"] = torch.randn(n, device="cuda", generator=g).to(dtype) if case["bias"] else None
    if kind == "product":
        state["codes"], state["scales"] = _plain_quantize(state.pop("x"), case["format"])
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(s):
    kind, fmt, dtype = s["kind"], s["format"], s["dtype"]
    if kind == "quantize":
        codes, scales = _plain_quantize(s["x"], fmt)
        return {"values": _plain_values(codes, scales).to(dtype)}
    if kind == "linear":
        return _plain_product(_plain_values(*_plain_quantize(s["x"], fmt)), s)
    if kind == "product":
        return _plain_product(_plain_values(s["codes"], s["scales"]), s)
    if kind == "norm":
        total = (s["x"].float() + s["delta"].float()).to(dtype)
        t = total.float()
        y = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
        return {"total": total, "values": _plain_values(*_plain_quantize(y, fmt)).to(dtype)}
    gate, up = s["gate"].float(), s["up"].float()
    return {"values": _plain_values(*_plain_quantize(gate / (1 + torch.exp(-gate)) * up, fmt)).to(dtype)}


def _run_own(s):
    import nanoquantization_amd as nq

    kind, fmt, dtype = s["kind"], s["format"], s["dtype"]
    if kind == "quantize":
        codes, scales = nq.mx_quantize(s["x"], fmt)
        return {"values": nq.mx_dequantize(codes, scales, dtype)}
    if kind == "linear":
        return nq.mx_linear(s["x"], s["weight"], s["weight_scales"], s["bias"], activations=fmt)
    if kind == "product":
        return nq.mx_linear_quantized(s["codes"], s["scales"], s["weight"], s["weight_scales"], s["bias"], dtype)
    if kind == "norm":
        codes, scales, total = nq.mx_add_rmsnorm(s["x"], s["delta"], s["weight"], EPS, fmt)
        return {"total": total, "values": nq.mx_dequantize(codes, scales, dtype)}
    codes, scales = nq.mx_silu_mul(s["gate"], s["up"], fmt)
    return {"values": nq.mx_dequantize(codes, scales, dtype)}


def work(case):
    rows, k, b = case["rows"], case["k"], BYTES[case["dtype"]]
    packed = CODE_BYTES[case["format"]] + 1 / BLOCK
    kind = case["kind"]
    if kind == "quantize":                        # values in, codes and scales out, values out
        return {"bytes": rows * k * (2 * b + packed), "flops": 2 * rows * k}
    if kind == "norm":                            # both addends in; their sum, codes and scales, values out
        return {"bytes": rows * k * (4 * b + packed) + k * b, "flops": 6 * rows * k}
    if kind == "silu":
        return {"bytes": rows * k * (3 * b + packed), "flops": 6 * rows * k}
    n = case["n"]
    x = rows * k * (b if kind == "linear" else packed)
    return {"bytes": x + n * k * (0.5 + 1 / BLOCK) + rows * n * b + (n * b if case["bias"] else 0), "flops": 2 * rows * k * n}


# ---- from the definition, in 64 bits ------------------------------------------------------------------------------------
def _exact_rounded(x, fmt):
    """The values that x's blocks stand for once quantised."""
    mantissa, least, most, top = (1, 0, 6.0, 2) if fmt == "mxfp4" else (3, -6, 448.0, 8)

    def element(v):
        exponent = (torch.frexp(v)[1] - 1).clamp_min(least)
        step = torch.ldexp(torch.ones_like(v), exponent - mantissa)
        return torch.round(v / step) * step

    v = x.to(F64).unflatten(-1, (-1, BLOCK))
    largest = v.abs().amax(-1, keepdim=True)
    e = torch.frexp(largest)[1] - 1 - top
    e = torch.where(element(torch.ldexp(largest, -e)) > most, e + 1, e)
    e = torch.where(largest == 0, -127, e).clamp_min(-127)
    return torch.ldexp(element(torch.ldexp(v, -e)), e).flatten(-2)


def _exact_stored(codes, scales):
    c = codes.to(torch.int64)
    if codes.shape[-1] == BLOCK * scales.shape[-1]:
        bits, bias = 3, 7
    else:
        c = torch.stack([c % 16, c // 16], -1).flatten(-2)
        bits, bias = 1, 1
    sign = c >> (7 if bits == 3 else 3)
    exponent = (c >> bits) & (15 if bits == 3 else 3)
    fraction = (c & ((1 << bits) - 1)).to(F64) / (1 << bits)
    value = torch.where(exponent == 0, torch.ldexp(fraction, torch.full_like(exponent, 1 - bias)),
                        torch.ldexp(1 + fraction, exponent - bias))
    value = torch.where(sign == 1, -value, value).unflatten(-1, (-1, BLOCK))
    return torch.ldexp(value, (scales.to(torch.int64) - 127).unsqueeze(-1)).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    kind, fmt = case["kind"], case["format"]
    if kind == "quantize":
        return {"values": _exact_rounded(s["x"], fmt)}
    if kind in ("linear", "product"):
        x = _exact_rounded(s["x"], fmt) if kind == "linear" else _exact_stored(s["codes"], s["scales"])
        y = torch.matmul(x, _exact_stored(s["weight"], s["weight_scales"]).t())
        return y if s["bias"] is None else y + s["bias"].to(F64)
    if kind == "norm":
        # the sum is stored in the inputs' type, and the norm is that of the stored sum
        total = s["x"].to(F64) + s["delta"].to(F64)
        t = total.to(s["dtype"]).to(F64)
        y = t / torch.sqrt((t * t).sum(-1, keepdim=True) / case["k"] + EPS) * s["weight"].to(F64)
        return {"total": total, "values": _exact_rounded(y, fmt)}
    gate = s["gate"].to(F64)
    return {"values": _exact_rounded(gate * torch.sigmoid(gate) * s["up"].to(F64), fmt)}
