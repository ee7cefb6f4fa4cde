"""Block-scaled codes by their definition, in 64 bits on the CPU: the number of
each code from its bits, the nearest number by comparing with all of them."""
import math

import torch

BLOCK = 32
CODES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8, "fp4": torch.uint8}
LARGEST = {"fp8": 448.0, "int8": 127.0, "fp4": 6.0}


def numbers(fmt):
    """The number of every code (256, or 16)."""
    if fmt == "int8":
        return torch.tensor([c - 256 if c > 127 else c for c in range(256)], dtype=torch.float64)
    lead, powers, bias = (3, 4, 7) if fmt == "fp8" else (1, 2, 1)
    out = []
    for c in range(1 << (1 + powers + lead)):
        m, p = c & ((1 << lead) - 1), (c >> lead) & ((1 << powers) - 1)
        v = math.ldexp(1 + m / (1 << lead), p - bias) if p else math.ldexp(m / (1 << lead), 1 - bias)
        if fmt == "fp8" and p == 15 and m == 7:
            v = math.nan
        out.append(-v if c >> (powers + lead) else v)
    return torch.tensor(out, dtype=torch.float64)


def code_bits(codes, fmt):
    """Codes of a pool as integers, one per dim."""
    if fmt == "fp4":
        return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    return codes.view(torch.uint8).long()


def pool_codes(bits, fmt):
    """The reverse."""
    if fmt == "fp4":
        return (bits[..., 0::2] + 16 * bits[..., 1::2]).to(torch.uint8)
    return bits.to(torch.uint8).view(CODES[fmt])


def decode(codes, exponents, fmt):
    """Values in 64 bits."""
    e = exponents.double()
    scale = torch.ldexp(torch.ones_like(e), exponents.int() - 127)
    scale = torch.where(exponents == 255, math.nan, scale)
    return numbers(fmt)[code_bits(codes, fmt)] * torch.repeat_interleave(scale, BLOCK, -1)


def exponent_of(top, fmt):
    """The smallest k with top <= M 2^k (k at least -117), of 64-bit values."""
    k = torch.full(top.shape, -117, dtype=torch.int32)
    while True:
        small = top > LARGEST[fmt] * torch.ldexp(torch.ones_like(top), k)
        if not small.any():
            return k
        k += small.int()


def encode(x, fmt, dtype):
    """(codes, exponents) of 64-bit values [..., dim], as a pool under a model of
    ``dtype`` holds them."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1)
    bad = ~torch.isfinite(top)
    k = exponent_of(torch.where(bad, 0.0, top), fmt)
    largest = torch.finfo(dtype).max
    # no block reads back as an infinity
    limit = {torch.float16: 16, torch.bfloat16: 128}[dtype] - {"fp8": 8, "int8": 6, "fp4": 2}[fmt]
    k = k.clamp(max=limit)
    table = numbers(fmt)
    table = torch.where(torch.isnan(table), math.inf, table)
    if fmt == "int8":
        table[128] = math.inf   # -128 is not made
    y = (blocks / torch.ldexp(torch.ones_like(top), k)[..., None]).flatten(-2)
    cap = torch.repeat_interleave(torch.where(k == limit, {"fp8": 240.0, "int8": 63.0, "fp4": 3.0}[fmt], math.inf),
                                  BLOCK, -1)
    y = torch.minimum(torch.maximum(y, -cap), cap)
    y = torch.where(torch.repeat_interleave(bad, BLOCK, -1), 0.0, y)
    best = torch.empty(y.shape, dtype=torch.long)
    flat, out = y.reshape(-1), best.view(-1)
    for at in range(0, flat.numel(), 1 << 14):
        d = (flat[at:at + (1 << 14), None] - table).abs()
        near = d == d.amin(-1, keepdim=True)
        even = near & (torch.arange(len(table)) % 2 == 0)
        pick = torch.where(even.any(-1, keepdim=True), even, near)
        # +0 and -0 are as near: the sign decides
        sign = torch.signbit(flat[at:at + (1 << 14)])[:, None] == torch.signbit(table)
        both = pick & sign
        out[at:at + (1 << 14)] = torch.where(both.any(-1, keepdim=True), both, pick).int().argmax(-1)
    assert not torch.isinf(decode(pool_codes(best, fmt), torch.where(bad, 255, k + 127).to(torch.uint8), fmt)
                           .abs().clamp(max=2 * largest)).any()
    return pool_codes(best, fmt), torch.where(bad, 255, k + 127).to(torch.uint8)


def rounded(values, dtype):
    """64-bit values as a kernel hands them on: rounded once to ``dtype``.  (Via
    fp32 they would be rounded twice; codes times a power of two have at most 8
    significant bits, so fp32 holds them exactly.)"""
    return values.float().to(dtype)
