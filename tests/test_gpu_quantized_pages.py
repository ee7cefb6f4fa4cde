"""Pools in 8 and 4 bits: what qk_norm_rope stores, what read_pages and
paged_attention make of it, against the definition in 64 bits on the CPU."""
import math

import pytest
import torch

import blocks
from conftest import gpu_available
from test_gpu_paged_attention import batch_of, check, expected, make

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


def same(a, b):
    """Equal bits, any NaN equal to any."""
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


# ------------------------------------------------------------------ reading --

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_every_code_reads_as_its_number(ops, fmt, dtype, D):
    """All codes with all exponents, subnormals, infinities and NaN among them."""
    n = len(blocks.numbers(fmt))
    bits = torch.arange(n).repeat(256)                         # code fastest
    e = torch.arange(256).repeat_interleave(n)
    per = D // 32                                              # a block holds 32 codes of one exponent
    bits, e = bits.view(-1, D), e.view(-1, per, 32)[:, :, 0].contiguous() if n >= 32 else None
    if e is None:   # 16 codes: each twice in a block
        bits = torch.arange(16).repeat(256 * 2).view(-1, D)
        e = torch.arange(256).view(-1, per)
    rows, page = bits.shape[0], 16
    codes = blocks.pool_codes(bits, fmt).view(rows // page, 1, page, -1)
    exps = e.to(torch.uint8).view(rows // page, 1, page, per)
    pool = ops.QuantizedPages(codes.to(DEV), exps.to(DEV))
    table = torch.arange(rows // page, dtype=torch.int32, device=DEV)[None]
    batch = ops.PagedBatch(table, i32([rows]), i32([0, 1]), 1)
    keys, values = ops.read_pages(pool, pool, batch, rows=rows, dtype=dtype)
    want = blocks.rounded(blocks.decode(codes, exps, fmt), dtype).view(1, 1, rows, D)
    assert same(keys.cpu(), want) and same(values.cpu(), want)


def fill(fmt, pages, H, page, D, layout, seed):
    """A pool of random codes, NaN among the exponents of nothing that counts."""
    g = torch.Generator().manual_seed(seed)
    bits = torch.randint(0, 16 if fmt == "fp4" else 256, (pages, H, page, D), generator=g)
    if fmt == "fp8":
        bits[(bits & 127) == 127] = 5
    codes = blocks.pool_codes(bits, fmt)
    exps = torch.randint(118, 132, (pages, H, page, D // 32), generator=g).to(torch.uint8)
    if layout == "tokens":
        put = lambda t: t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
        return codes, exps, put(codes.view(torch.uint8)).view(codes.dtype), put(exps)
    return codes, exps, codes.to(DEV), exps.to(DEV)


@pytest.mark.parametrize("fmt", FORMATS + [None])
@pytest.mark.parametrize("D,dtype,page,H,layout", [(128, BF, 16, 2, "heads"), (64, HF, 8, 3, "tokens"),
                                                   (128, HF, 1, 1, "heads"), (64, BF, 128, 1, "tokens")])
def test_read_pages(ops, fmt, D, dtype, page, H, layout):
    lens, first = [0, 1, 77, 300, 129], [0, 0, 70, -5, 2 ** 31 - 1]
    rows = 133
    held = [-(-n // page) for n in lens]
    P = sum(held) + 3
    ids = torch.randperm(P, generator=torch.Generator().manual_seed(3)).tolist()
    table = torch.full((5, max(held) + 1), 2 ** 31 - 1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(held):
        table[s, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    if fmt:
        pools = [fill(fmt, P, H, page, D, layout, s) for s in (1, 2)]
        host = [blocks.rounded(blocks.decode(c, e, fmt), dtype) for c, e, _, _ in pools]
        pools = [ops.QuantizedPages(c, e) for _, _, c, e in pools]
    else:
        host = [torch.randn((P, H, page, D), generator=torch.Generator().manual_seed(s)).to(dtype) for s in (1, 2)]
        pools = [t.to(DEV) if layout == "heads" else t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in host]
    batch = ops.PagedBatch(table.to(DEV), i32(lens), i32([0] * 6), 1)
    for f in (None, first):
        # rows of a token together, with room between them
        store = [torch.full((5, rows + 2, H, D + 8), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
        out = tuple(t[:, :rows, :, :D].transpose(1, 2) for t in store)
        got = ops.read_pages(*pools, batch, first=None if f is None else i32(f), out=out)
        assert got[0] is out[0]
        for t, h, full in zip(out, host, store):
            want = torch.full((5, H, rows, D), 7.0, dtype=dtype)
            for s, n in enumerate(lens):
                for i in range(rows):
                    j = (0 if f is None else f[s]) + i
                    if 0 <= j < n:
                        want[s, :, i] = h[table[s, j // page], :, j % page]
            assert torch.equal(t.cpu(), want)
            assert bool((full[:, rows:] == 7).all()) and bool((full[..., D:] == 7).all())


def test_read_pages_sizes(ops):
    """Rows by default, contiguous rows without a table, nothing to read."""
    codes, exps, c, e = fill("int8", 3, 2, 40, 64, "heads", 5)
    pool = ops.QuantizedPages(c, e)
    batch = ops.PagedBatch(None, i32([40, 3]), i32([0, 0, 0]), 1)
    want = blocks.rounded(blocks.decode(codes, exps, "int8"), BF)
    keys, values = ops.read_pages(pool, pool, batch)
    assert keys.shape == (2, 2, 40, 64)
    assert torch.equal(keys[0].cpu(), want[0]) and torch.equal(values[1, :, :3].cpu(), want[1, :, :3])
    assert ops.read_pages(pool, pool, ops.PagedBatch(None, i32([40, 3]), i32([0, 0, 0]), 1, max_len=17))[0].shape[2] == 17
    assert ops.read_pages(pool, pool, batch, rows=0)[0].shape == (2, 2, 0, 64)
    none = ops.PagedBatch(None, i32([]), i32([0]), 1)
    assert ops.read_pages(pool, pool, none, rows=5)[0].shape == (0, 2, 5, 64)
    # lengths past the rows, page ids outside the pool: forced into them
    wild = ops.PagedBatch(i32([[2 ** 31 - 1, -7]]), i32([1000]), i32([0, 0]), 1)
    k16, _, c16, e16 = fill("int8", 3, 1, 32, 64, "heads", 6)
    pool = ops.QuantizedPages(c16, e16)
    keys, _ = ops.read_pages(pool, pool, wild, rows=200)
    want = blocks.rounded(blocks.decode(k16, e16.cpu(), "int8"), BF)
    assert torch.equal(keys[0, 0, :32].cpu(), want[2, 0]) and torch.equal(keys[0, 0, 32:64].cpu(), want[0, 0])


# ------------------------------------------------------------------ storing --

def edge_rows(n, D, dtype, seed=0):
    """Rows of many magnitudes: blocks of zeros, at the borders of a power, at the
    type's largest and smallest values, with infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, D), generator=g)
    x = (x * torch.exp(2.5 * torch.randn((n, D // 32), generator=g)).repeat_interleave(32, -1)).to(dtype).float()
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    special = [torch.zeros(32), torch.full((32,), -0.0), torch.full((32,), big), torch.full((32,), tiny),
               torch.full((32,), tiny / 4), torch.arange(32) * 448 / 31.0, torch.arange(32) * 127 / 31.0,
               torch.arange(32) * 6 / 31.0, -torch.arange(32) * 0.9921875, torch.tensor([448.0, 449.0] * 16),
               torch.tensor([1.0] * 31 + [math.inf]), torch.tensor([math.nan] + [2.0] * 31),
               torch.tensor([-math.inf] + [0.0] * 31), torch.tensor([big, tiny] * 16),
               torch.arange(32) * 0.25, torch.arange(32) * 0.5 + 0.5, torch.tensor([big * 0.75, -big * 0.5] * 16)]
    flat = x.view(-1, 32)
    for i, s in enumerate(special):
        flat[(5 * i + 1) % len(flat)] = s
    return x.to(dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,page,layout", [(128, 16, "heads"), (64, 4, "tokens")])
def test_stored_codes(ops, fmt, dtype, D, page, layout):
    """Neither norm nor rotation: the codes and exponents are the definition's,
    bit by bit; nothing else of the pools is written."""
    H, Hq, lens, news, pad = 3, 2, [37, 5, 90], [37, 1, 50], 2
    N = sum(news) + pad
    key = torch.stack([edge_rows(N, D, dtype, s) for s in range(H)], 1)
    value = torch.stack([edge_rows(N, D, dtype, 10 + s) for s in range(H)], 1)
    q = torch.randn((N, Hq, D)).to(dtype)
    held = [-(-n // page) for n in lens]
    P = sum(held) + 2
    ids = torch.randperm(P, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.full((3, max(held)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(held):
        table[s, :n] = ids[at:at + n]
        at += n
    start = [0, 37, 38, 88]
    kc, ke, kcd, ked = fill(fmt, P, H, page, D, layout, 1)
    vc, ve, vcd, ved = fill(fmt, P, H, page, D, layout, 2)
    batch = ops.PagedBatch(table.to(DEV), i32(lens), i32(start), max(news))
    q_out, none = ops.qk_norm_rope(q.to(DEV), key.to(DEV), value=value.to(DEV), batch=batch,
                                   key_pages=ops.QuantizedPages(kcd, ked), value_pages=ops.QuantizedPages(vcd, ved))
    assert none is None and torch.equal(q_out[:88].cpu(), q[:88])
    for x, c, e, cd, ed in ((key, kc, ke, kcd, ked), (value, vc, ve, vcd, ved)):
        codes, exps = blocks.encode(x.double(), fmt, dtype)
        c, codes = c.view(torch.uint8), codes.view(torch.uint8)
        for s in range(3):
            for i in range(news[s]):
                j = lens[s] - news[s] + i
                c[table[s, j // page], :, j % page] = codes[start[s] + i]
                e[table[s, j // page], :, j % page] = exps[start[s] + i]
        assert torch.equal(ed.cpu(), e)
        assert torch.equal(cd.cpu().view(torch.uint8), c)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype,D,rotary,interleaved,w32", [(BF, 128, 128, False, False), (HF, 64, 32, True, True),
                                                            (HF, 128, 64, False, True), (BF, 64, 64, True, False)])
def test_stored_keys_are_rounded_once(ops, fmt, dtype, D, rotary, interleaved, w32):
    """Norm, rotation, codes: off by at most half a step of the code next to the
    exact result, plus the fp32 result's own error.

    fp32: the sum of D squares (D 2^-24 relative, half of it in the root), root,
    division and two products (4 2^-24), sine and cosine of an angle whose
    fraction of a turn is rounded to fp32 (2^-24 of half a turn and the
    functions' own error, 2^-21 in all), two products and a sum (3 2^-24): at most
    (D / 2 + 20) 2^-24 of the pair's length.  Half a step: int8 2^k / 2; fp8
    2^-4 |y|, or 2^-10 2^k below 2^-6; fp4 half of the distance of its numbers,
    at most 1/4, 1/2 or 1 times 2^k for |y| up to 2, 4 or 6 of it; k from
    the largest of a block, which may be off by the same error."""
    H, Hq, lens, n = 2, 4, [900], 129
    g = torch.Generator().manual_seed(0)
    key = (2 * torch.randn((n, H, D), generator=g)).to(dtype)
    q = torch.randn((n, Hq, D), generator=g).to(dtype)
    w = (1 + 0.2 * torch.randn((D,), generator=g)).to(torch.float32 if w32 else dtype)
    freq = (500000.0 ** (-torch.arange(rotary // 2).double() * 2 / rotary)).float()
    page, P = 16, 57
    table = torch.randperm(P, generator=g).to(torch.int32)[None]
    pools = [ops.QuantizedPages.zeros(P, H, page, D, fmt, DEV) for _ in range(2)]
    batch = ops.PagedBatch(table.to(DEV), i32(lens), i32([0, n]), n)
    eps = 1e-6
    ops.qk_norm_rope(q.to(DEV), key.to(DEV), inv_freq=freq.to(DEV), query_weight=w.to(DEV), key_weight=w.to(DEV),
                     eps=eps, interleaved=interleaved, value=key.to(DEV), batch=batch, key_pages=pools[0],
                     value_pages=pools[1])
    y = key.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    t = (torch.arange(lens[0] - n, lens[0]).double()[:, None] * freq.double())[:, None]
    a = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    b = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    u, v = y[..., a].clone(), y[..., b].clone()
    size = y.abs().clone()
    size[..., a] = size[..., b] = torch.sqrt(u * u + v * v)
    y[..., a], y[..., b] = u * t.cos() - v * t.sin(), v * t.cos() + u * t.sin()
    err = (D / 2 + 20) * 2.0 ** -24 * size
    top = (y.abs() + err).unflatten(-1, (-1, 32)).amax(-1)
    k = torch.repeat_interleave(torch.ldexp(torch.ones_like(top), blocks.exponent_of(top, fmt)), 32, -1)
    z = (y.abs() + err) / k
    half = {"int8": torch.full_like(z, 0.5), "fp8": torch.maximum(z * 2.0 ** -4, torch.full_like(z, 2.0 ** -10)),
            "fp4": torch.where(z > 4, 1.0, torch.where(z > 2, 0.5, 0.25)).double()}[fmt]
    j = torch.arange(lens[0] - n, lens[0])
    at = table[0, j // page].long(), j % page
    got = blocks.decode(pools[0].codes.cpu()[at[0], :, at[1]], pools[0].exponents.cpu()[at[0], :, at[1]], fmt)
    off = (got - y).abs() - half * k - err
    assert off.max() <= 0, off.max()


# ---------------------------------------------------------------- attention --

def quantize(ops, x, fmt, junk=True):
    """The pools of make()'s tensors as codes, and its rows as what they stand
    for; everything that no sequence owns is NaN."""
    dtype = x["dtype"]
    def one(t):
        c, e = blocks.encode(torch.nan_to_num(t.cpu().double(), nan=0.0), fmt, dtype)
        bad = torch.isnan(t.cpu()).any(-1)
        if junk:
            e[bad] = 255
            if fmt == "fp8":
                c.view(torch.uint8)[bad] = 127
        if t.stride(2) > t.stride(1):   # token-major
            put = lambda y: y.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
            return ops.QuantizedPages(put(c.view(torch.uint8)).view(c.dtype), put(e))
        return ops.QuantizedPages(c.to(DEV), e.to(DEV))
    value = lambda r: blocks.rounded(blocks.decode(*blocks.encode(r.double(), fmt, dtype), fmt), dtype)
    x = dict(x)
    x["rows"] = [(value(k), value(v)) for k, v in x["rows"]]
    x["k"], x["v"] = one(x["k"]), one(x["v"])
    return x


CASES = [
    # lens, news, H, G, D, page, dtype, window, sinks, layout
    ([1], [1], 1, 1, 128, 8, BF, 0, 0, "heads"),
    ([519], [1], 2, 4, 128, 8, BF, 0, 0, "heads"),
    ([2500, 3, 129, 1, 4000], [1] * 5, 2, 8, 128, 16, BF, 0, 0, "tokens"),
    ([700, 64, 1290], [1, 1, 1], 1, 16, 64, 32, HF, 0, 0, "heads"),
    ([900, 33], [3, 2], 2, 8, 128, 16, HF, 0, 0, "heads"),            # two blocks of rows
    ([900, 1500], [5, 4], 1, 5, 64, 8, BF, 300, 5, "tokens"),
    ([300], [300], 1, 4, 128, 16, BF, 0, 0, "heads"),                 # tiles
    ([1030, 70, 5, 260], [200, 70, 1, 3], 2, 7, 128, 4, BF, 0, 0, "tokens"),
    ([500, 90], [333, 41], 1, 3, 64, 64, HF, 100, 9, "heads"),
    ([700], [130], 1, 4, 128, 2, HF, 64, 3, "heads"),                 # rows of a thread on several pages
    ([50, 0, 3], [60, 0, 5], 1, 4, 64, 16, BF, 0, 0, "heads"),        # more new tokens than rows
    ([777, 200], [3, 120], 1, 4, 128, 0, BF, 0, 0, "heads"),          # no table
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("i", range(len(CASES)))
def test_attention(ops, fmt, i):
    lens, news, H, G, D, page, dtype, window, sinks, layout = CASES[i]
    x = quantize(ops, make(lens, news, H, G, D, page, dtype, layout, seed=i, pad=2), fmt)
    out = torch.full((sum(news) + 2, H * G, D), 3.0, dtype=dtype, device=DEV)
    _, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), window=window, sinks=sinks, out=out,
                                 return_lse=True)
    check(x, out, lse, window, sinks)
    assert bool((out[-2:] == 3).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_long(ops, fmt):
    """Several ranges per sequence and head, and their join."""
    x = quantize(ops, make([9000, 4100], [1, 2], 1, 4, 128, 16, BF, seed=5), fmt)
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), return_lse=True)
    check(x, out, lse)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("news", [[6], [90]])
def test_blocks_of_nan_reach_the_tokens_that_see_them(ops, fmt, news):
    """A NaN block of V in the row of the last token but two: the tokens before it
    get what they get without it, those from there on NaN in its 32 dims."""
    x = make([400], news, 1, 4, 128, 16, BF, seed=2)
    x = quantize(ops, x, fmt)
    clean, _ = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), return_lse=True)
    j = 397
    page = int(x["table"][0, j // 16])
    x["v"].exponents[page, 0, j % 16, 1] = 255
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), return_lse=True)
    sees = news[0] - 3
    assert torch.equal(out[:sees], clean[:sees])
    assert bool(torch.isnan(out[sees:, :, 32:64]).all())
    assert torch.equal(out[sees:, :, :32], clean[sees:, :, :32])
    assert torch.equal(out[sees:, :, 64:], clean[sees:, :, 64:]) and not bool(torch.isnan(lse).any())
    x["k"].exponents[page, 0, j % 16, 0] = 255
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), return_lse=True)
    assert torch.equal(out[:sees], clean[:sees]) and bool(torch.isnan(out[sees:]).all())
    assert bool(torch.isnan(lse[sees:]).all()) and not bool(torch.isnan(lse[:sees]).any())


def test_far_pages(ops):
    """Offsets of codes and exponents past 32 bits."""
    P, page, H, D = 35000, 64, 8, 128
    codes = torch.zeros((P, H, page, D), dtype=torch.int8, device=DEV)        # 2.3 GB
    exps = torch.full((P, H, page, D // 32), 127, dtype=torch.uint8, device=DEV)
    assert codes.numel() > 2 ** 31
    pool = ops.QuantizedPages(codes, exps)
    table = i32([[P - 1, P - 2]])
    n = 70
    g = torch.Generator().manual_seed(0)
    key, value = (torch.randn((n, H, D), generator=g).to(BF).to(DEV) for _ in range(2))
    q = torch.randn((n, H, D), generator=g).to(BF).to(DEV)
    far = ops.PagedBatch(table, i32([n]), i32([0, n]), n)
    ops.qk_norm_rope(q, key, value=value, batch=far, key_pages=pool, value_pages=pool)
    near = ops.QuantizedPages(codes[-2:].flip(0).contiguous(), exps[-2:].flip(0).contiguous())
    close = ops.PagedBatch(i32([[0, 1]]), i32([n]), i32([0, n]), n)
    assert bool((near.codes[0] != 0).any())
    for a, b in zip(ops.read_pages(pool, pool, far, rows=n), ops.read_pages(near, near, close, rows=n)):
        assert torch.equal(a, b)
    assert torch.equal(ops.paged_attention(q, pool, pool, far), ops.paged_attention(q, near, near, close))
    one = [ops.PagedBatch(t, i32([n]), i32([0, 1]), 1) for t in (table, i32([[0, 1]]))]
    assert torch.equal(ops.paged_attention(q[:1], pool, pool, one[0]), ops.paged_attention(q[:1], near, near, one[1]))


def test_page_operations_move_codes_and_exponents(ops):
    P, H, page, D = 12, 2, 8, 64
    pools = []
    for fmt in FORMATS:
        _, _, c, e = fill(fmt, P, H, page, D, "heads", 4)
        pools.append(ops.QuantizedPages(c, e))
    before = [(p.codes.clone(), p.exponents.clone()) for p in pools]
    table = ops.PageTable.empty(2, 4, P, page, DEV)
    table.lens.copy_(i32([13, 13]))
    table.pages[:, :2] = i32([[9, 4], [9, 4]])
    table.refs[9] = table.refs[4] = 2
    assert ops.extend_pages(table, i32([1, 0]), pools).all()          # page 4 is copied for sequence 0
    new = int(table.pages[0, 1])
    assert new == 0
    for p, (c, e) in zip(pools, before):
        assert torch.equal(p.codes[0].view(torch.uint8), c[4].view(torch.uint8)) and torch.equal(p.exponents[0], e[4])
    assert int(ops.compact_pages(table, pools)) == 3                  # 0, 4, 9 -> 0, 1, 2
    for p, (c, e) in zip(pools, before):
        a, b = (int(v) for v in table.pages[1, :2])
        assert torch.equal(p.codes[a].view(torch.uint8), c[9].view(torch.uint8)) and torch.equal(p.exponents[a], e[9])
        assert torch.equal(p.codes[b].view(torch.uint8), c[4].view(torch.uint8)) and torch.equal(p.exponents[b], e[4])


def test_captured_steps_and_streams(ops):
    """Store, attend and read in one graph, replayed with other tokens and lengths;
    the same eager on another stream."""
    H, G, D, page, P = 2, 4, 128, 16, 40
    pools = [ops.QuantizedPages.zeros(P, H, page, D, "fp8", DEV) for _ in range(2)]
    table = torch.arange(P, dtype=torch.int32, device=DEV).view(2, 20)
    lens, start = i32([100, 7]), i32([0, 1, 2])
    batch = ops.PagedBatch(table, lens, start, 1)
    q, k, v = (torch.randn((2, h, D), device=DEV).to(BF) for h in (H * G, H, H))
    out = torch.zeros_like(q)
    back = tuple(torch.zeros((2, H, 320, D), dtype=BF, device=DEV) for _ in range(2))

    def step(pools, out, back):
        ops.qk_norm_rope(q, k, value=v, batch=batch, key_pages=pools[0], value_pages=pools[1], query_out=out)
        ops.paged_attention(out, *pools, batch, out=out)
        ops.read_pages(*pools, batch, out=back)

    eager = [ops.QuantizedPages(p.codes.clone(), p.exponents.clone()) for p in pools]
    e_out, e_back = torch.zeros_like(out), tuple(torch.zeros_like(t) for t in back)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([ops.QuantizedPages(p.codes.clone(), p.exponents.clone()) for p in pools], torch.zeros_like(out),
             tuple(torch.zeros_like(t) for t in back))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pools, out, back)
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device=DEV))
        lens.copy_(i32([101 + i, 8 + 90 * i]))
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(eager, e_out, e_back)
        side.synchronize()
        assert torch.equal(out, e_out) and torch.equal(back[0], e_back[0]) and torch.equal(back[1], e_back[1])


def test_layer_of_arguments_refuses(ops):
    """The Python layer's checks of pools, outputs and rows."""
    P, H, page, D = 6, 2, 8, 64
    pool = ops.QuantizedPages.zeros(P, H, page, D, "fp8", DEV)
    batch = ops.PagedBatch(i32([[0, 1, 2]]), i32([20]), i32([0, 1]), 1)
    q = torch.zeros((1, 4, D), dtype=BF, device=DEV)
    key = torch.zeros((1, H, D), dtype=BF, device=DEV)
    plain = torch.zeros((P, H, page, D), dtype=BF, device=DEV)
    wide = ops.QuantizedPages.zeros(P, H, page, 128, "fp8", DEV)
    whole = ops.QuantizedPages.zeros(P, H, page, D, "int8", DEV)
    flat = ops.QuantizedPages(pool.codes, pool.exponents[:1].expand(P, H, page, 2))
    for k, v in ((pool, plain), (plain, pool), (pool, whole), (wide, wide)):
        with pytest.raises((TypeError, ValueError)):
            ops.paged_attention(q, k, v, batch)
        with pytest.raises((TypeError, ValueError)):
            ops.qk_norm_rope(q, key, value=key, batch=batch, key_pages=k, value_pages=v)
    assert ops.paged_attention(q, flat, flat, batch).shape == q.shape      # read, not written
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, key, value=key, batch=batch, key_pages=flat, value_pages=flat)
    with pytest.raises((TypeError, ValueError)):
        ops.read_pages(pool, plain, batch)
    out = [torch.zeros((1, H, 20, D), dtype=BF, device=DEV) for _ in range(2)]
    assert ops.read_pages(pool, pool, batch, out=tuple(out))[0] is out[0]
    for kw in (dict(rows=-1), dict(dtype=torch.float32), dict(out=tuple(out), rows=19), dict(first=i32([0, 0])),
               dict(first=torch.zeros(1, dtype=torch.int64, device=DEV)), dict(out=(out[0], out[1].half())),
               dict(out=(out[0], out[1].transpose(2, 3).contiguous().transpose(2, 3))),
               dict(out=(out[0][:, :1].expand(1, H, 20, D), out[1][:, :1].expand(1, H, 20, D)))):
        with pytest.raises((TypeError, ValueError)):
            ops.read_pages(pool, pool, batch, **kw)
    with pytest.raises(TypeError):
        ops.read_pages(plain, plain, batch, dtype=HF)       # 16-bit rows are read as they are


def test_sixteen_bit_type_of_the_rows_read(ops):
    """One pool read as bf16 and as fp16."""
    codes, exps, c, e = fill("fp8", 4, 1, 16, 128, "heads", 3)
    pool = ops.QuantizedPages(c, e)
    batch = ops.PagedBatch(i32([[2, 0]]), i32([32]), i32([0, 0]), 1)
    want = blocks.decode(codes, exps, "fp8")
    for dtype in (BF, HF):
        keys, _ = ops.read_pages(pool, pool, batch, rows=32, dtype=dtype)
        assert keys.dtype is dtype
        assert torch.equal(keys[0, 0].cpu(), torch.cat([blocks.rounded(want[i, 0], dtype) for i in (2, 0)]))
