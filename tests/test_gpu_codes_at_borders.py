"""Codes of rotated keys next to their borders, and of numbers next to the type's
largest, against the definition in 64 bits."""
import math

import pytest
import torch

import blocks
from conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
FORMATS = ["fp8", "int8", "fp4"]


@pytest.fixture(scope="module")
def ops():
    from adaptiveimi_amd import ops

    return ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_codes_of_keys_near_a_quarter_turn(ops, fmt, interleaved):
    """Keys (1, 0) turned by nearly a quarter: the cosine is the small difference
    of two large angles, and a block of such is scaled up.  Its error: 2 pi (position
    * f) 2^-53 of the fp64 product and of its reduction, twice, which is under
    2^-51 times the angle, and 2^-21 relative for the fp32 functions (4 units in
    the last place) and the sum that follows.  Every code that no error of that size
    changes is the definition's.  (The fraction of a turn rounded to fp32 is off by
    2^-26, 9e-8 of angle: 25 to 240 of the 96000 codes.)"""
    n, D, page = 1500, 128, 16
    # 64 neighbouring fp32 numbers next to a quarter turn per position, odd positions
    bits = torch.tensor(math.pi / 2).view(torch.int32) + torch.arange(-D // 4, D // 4, dtype=torch.int32)
    freq = bits.view(torch.float32)
    pos = 2 * torch.arange(n) + 1
    key = torch.zeros((n, 1, D), dtype=BF)
    first = slice(0, D, 2) if interleaved else slice(0, D // 2)
    key[:, :, first] = 1.0
    # a sequence per position: its last row is the token's, on a page of its own
    table = torch.arange(n, dtype=torch.int32)[:, None].expand(n, int(pos[-1]) // page + 1).contiguous()
    pools = [ops.QuantizedPages.zeros(n, 1, page, D, fmt, DEV) for _ in range(2)]
    batch = ops.PagedBatch(table.to(DEV), (pos + 1).to(torch.int32).to(DEV),
                           torch.arange(n + 1, dtype=torch.int32, device=DEV), 1)
    q = torch.zeros((n, 1, D), dtype=BF, device=DEV)
    ops.qk_norm_rope(q, key.to(DEV), inv_freq=freq.to(DEV), interleaved=interleaved, value=key.to(DEV), batch=batch,
                     key_pages=pools[0], value_pages=pools[1])
    t = pos.double()[:, None] * freq.double()
    y = torch.empty((n, D), dtype=torch.float64)
    rest = slice(1, D, 2) if interleaved else slice(D // 2, D)
    y[:, first], y[:, rest] = t.cos(), t.sin()
    err = torch.empty_like(y)
    err[:, first] = err[:, rest] = t * 2.0 ** -51
    err += y.abs() * 2.0 ** -21
    low, want, high = (blocks.encode(z, fmt, BF) for z in (y - err, y, y + err))
    sure = torch.repeat_interleave(low[1] == high[1], 32, -1)
    sure &= blocks.code_bits(low[0], fmt) == blocks.code_bits(high[0], fmt)
    assert sure.double().mean() > 0.99
    at = torch.arange(n), 0, pos % page
    codes, exps = pools[0].codes.cpu()[at], pools[0].exponents.cpu()[at]
    wrong = (blocks.decode(codes, exps, fmt) != blocks.decode(*want, fmt)) & sure
    assert int(wrong.sum()) == 0, f"{int(wrong.sum())} codes"


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_finite_numbers_read_back_finite(ops, fmt, dtype):
    """Blocks of numbers up to the type's largest, each with every top from there
    down through four powers of two, read back in that type."""
    D, page = 128, 16
    big = torch.finfo(dtype).max
    top = torch.tensor([big], dtype=dtype).view(torch.int16).item()
    near = torch.arange(top, top - 4 * (128 if dtype is BF else 1024), -1 if dtype is BF else -7, dtype=torch.int32)
    tops = near.to(torch.int16).view(dtype)
    n = len(tops) // 4 * 4
    g = torch.Generator().manual_seed(0)
    x = (torch.rand((n, 32), generator=g) * 2 - 1) * tops[:n, None].float()
    x[:, 5] = tops[:n].float() * torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
    x = x.to(dtype).view(n // 4, 1, D)
    N = n // 4
    P = -(-N // page)
    table = torch.arange(P, dtype=torch.int32, device=DEV)[None]
    batch = ops.PagedBatch(table, i32([N]), i32([0, N]), N)
    pools = [ops.QuantizedPages.zeros(P, 1, page, D, fmt, DEV) for _ in range(2)]
    ops.qk_norm_rope(x.to(DEV), x.to(DEV), value=(-x).to(DEV), batch=batch, key_pages=pools[0], value_pages=pools[1])
    keys, values = ops.read_pages(*pools, batch, rows=N, dtype=dtype)
    assert bool(torch.isfinite(keys).all()) and bool(torch.isfinite(values).all())
    # and the encoder that the other tests compare with
    codes, exps = blocks.encode(x.double(), fmt, dtype)
    assert bool(torch.isfinite(blocks.rounded(blocks.decode(codes, exps, fmt), dtype)).all())
    # off by half a step of the number at most, or by what the held-back codes leave:
    # 240, 63 and 3 of 256, 64 and 4
    left = {"fp8": 240 / 256, "int8": 63 / 64, "fp4": 3 / 4}[fmt]
    largest = keys[0, 0].view(-1, 32).abs().amax(-1).double().cpu()
    want = x.view(-1, 32).abs().amax(-1).double()
    assert bool((largest >= left * want * (1 - 2.0 ** -7)).all())
