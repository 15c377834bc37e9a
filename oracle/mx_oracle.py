"""Microscaled formats from their definition, in 64 bits on the CPU: nearest values by search in the table of elements.
Test infrastructure only."""
from __future__ import annotations

import torch

BLOCK = 32


def elements(fmt: str) -> torch.Tensor:
    """The magnitudes of the elements by code without sign: e2m1 codes 0 .. 7, e4m3 codes 0 .. 126."""
    bits, bias, count = (1, 1, 8) if fmt == "mxfp4" else (3, 7, 127)
    out = []
    for code in range(count):
        e, m = code >> bits, (code & ((1 << bits) - 1)) / (1 << bits)
        out.append(m * 2.0 ** (1 - bias) if e == 0 else (1 + m) * 2.0 ** (e - bias))
    return torch.tensor(out, dtype=torch.float64)


def _nearest(v: torch.Tensor, fmt: str) -> torch.Tensor:
    """Code without sign of the element nearest to v >= 0, the even code of two."""
    table = elements(fmt)
    step = table[-1] - table[-2]
    table = torch.cat([table, (table[-1] + step).reshape(1)])       # the next one, were there one: what rounds to it is past the largest
    upper = torch.searchsorted(table, v.contiguous()).clamp(1, len(table) - 1)
    low, high = v - table[upper - 1], table[upper] - v
    code = torch.where((low < high) | ((low == high) & ((upper - 1) % 2 == 0)), upper - 1, upper)
    return torch.where(v >= table[-1], len(table) - 1, code)


def scale_exponents(largest: torch.Tensor, fmt: str) -> torch.Tensor:
    """e of a block by its largest magnitude (finite)."""
    most = len(elements(fmt)) - 1
    a = largest.to(torch.float64)
    e = torch.frexp(torch.where(a == 0, torch.ones_like(a), a))[1].to(torch.int64) - 1 - (2 if fmt == "mxfp4" else 8)
    e = torch.where(_nearest(torch.ldexp(a, -e), fmt) > most, e + 1, e)
    return torch.where(a == 0, -127, e).clamp_min(-127)


def quantize(x: torch.Tensor, fmt: str):
    """(codes, scales) uint8."""
    v = x.detach().cpu().to(torch.float64).unflatten(-1, (-1, BLOCK))
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad.unsqueeze(-1), 0.0, v)
    e = scale_exponents(v.abs().amax(-1), fmt)
    code = _nearest(torch.ldexp(v.abs(), -e.unsqueeze(-1)), fmt)
    sign = torch.signbit(v) & ~bad.unsqueeze(-1)
    code = (code | (sign.to(torch.int64) << (3 if fmt == "mxfp4" else 7))).flatten(-2).to(torch.uint8)
    if fmt == "mxfp4":
        pairs = code.unflatten(-1, (-1, 2))
        code = pairs[..., 0] | (pairs[..., 1] << 4)
    return code, torch.where(bad, 255, e + 127).to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes and scales stand for, float64."""
    codes, scales = codes.detach().cpu(), scales.detach().cpu()
    four = codes.shape[-1] == 16 * scales.shape[-1]
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int64) if four else codes.to(torch.int64)
    table = elements("mxfp4" if four else "mxfp8")
    if not four:
        table = torch.cat([table, torch.full((1,), float("nan"), dtype=torch.float64)])
    v = table[c & (7 if four else 127)]
    v = torch.where(c >> (3 if four else 7) == 1, -v, v).unflatten(-1, (-1, BLOCK))
    power = torch.ldexp(torch.ones((), dtype=torch.float64), scales.to(torch.int64) - 127)
    return (v * torch.where(scales == 255, float("nan"), power).unsqueeze(-1)).flatten(-2)


def half_steps(y: torch.Tensor, e: torch.Tensor, fmt: str) -> torch.Tensor:
    """Half the distance of the elements around y, at blocks of scale 2^e."""
    mantissa, least = (1, 0) if fmt == "mxfp4" else (3, -6)
    s = torch.ldexp(y.abs().unflatten(-1, (-1, BLOCK)), -e.unsqueeze(-1))
    at = (torch.frexp(s)[1].to(torch.int64) - 1).clamp_min(least)
    at = torch.where(s == 0, least, at)
    return torch.ldexp(torch.ones_like(s), at - mantissa - 1 + e.unsqueeze(-1)).flatten(-2)
