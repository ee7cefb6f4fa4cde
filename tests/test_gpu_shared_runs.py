"""Runs of share_prefixes next to sequences that share little with them, and the
attention of shared batches where one side outweighs the other, against the
definition in 64 bits on the CPU."""
import pytest
import torch

from conftest import gpu_available
from test_gpu_paged_attention import check
from test_gpu_quantized_pages import quantize
from test_gpu_shared_prefixes import attend, forked, ones

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from adaptiveimi_amd import ops

    return ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def table_of(families, header, page, width):
    """families: (sequences, leading pages that they share); all tables begin with
    the same `header` pages, every other page is held once."""
    g = torch.Generator().manual_seed(7)
    fresh = iter(torch.randperm(1 << 20, generator=g).tolist())
    take = lambda n: [next(fresh) for _ in range(n)]
    head, rows = take(header), []
    for size, common in families:
        same = head + take(max(common - header, 0))
        rows += [same + take(width - len(same)) for _ in range(size)]
    return torch.tensor(rows, dtype=torch.int32)


@pytest.mark.parametrize("page,header", [(16, 1), (16, 3), (4, 15), (1, 63), (2, 7)])
def test_a_short_header_parts_runs(ops, page, header):
    """Two families of long common prompts, and between and behind them a sequence
    that has only the header of all (fewer than 64 rows) in common with them: each
    family keeps its own rows."""
    long, short = 1040 // page, 640 // page
    families = [(32, long), (1, header), (3, short), (1, header), (1, header)]
    width = 1200 // page
    table = table_of(families, header, page, width)
    S = len(table)
    batch = ops.PagedBatch(table.to(DEV), i32([width * page] * S), i32(list(range(S + 1))), 1)
    got = ops.share_prefixes(batch, page)
    rows = lambda pages: pages * page // 8 * 8
    assert got.shared.tolist() == [rows(long)] * 32 + [0] + [rows(short)] * 3 + [0, 0]
    assert got.members.tolist() == [32] + [0] * 32 + [3] + [0] * 4
    assert got.leaders.tolist() == [0] * 32 + [32] + [33] * 3 + [36, 37]
    assert got.saved.tolist() == [31 * rows(long) + 2 * rows(short)]


@pytest.mark.parametrize("page,header", [(16, 4), (32, 2), (4, 16), (1, 64)])
def test_a_header_of_64_rows_joins_runs(ops, page, header):
    """From 64 rows on a run holds all that begin alike, and shares what all have."""
    families = [(4, 640 // page), (2, 320 // page), (1, header)]
    table = table_of(families, header, page, 700 // page)
    batch = ops.PagedBatch(table.to(DEV), i32([700 // page * page] * 7), i32(list(range(8))), 1)
    got = ops.share_prefixes(batch, page)
    assert got.shared.tolist() == [64] * 7 and got.members.tolist() == [7] + [0] * 6
    got = ops.share_prefixes(batch, page, labels=i32([0, 0, 0, 0, 1, 1, 2]))
    assert got.members.tolist() == [4, 0, 0, 0, 2, 0, 0]
    assert got.shared.tolist() == [640 // page * page] * 4 + [320 // page * page] * 2 + [0]


def test_attention_of_parted_runs(ops):
    """Tables that part after one page of 16 rows: the families on either side are
    attended together, each token over its own sequence's rows."""
    x = forked([(512, ones(5, 60, 9)), (16, ones(40)), (320, ones(1, 30))], 2, 4, 128, 16, BF)
    first = int(x["table"][0, 0])
    held = x["table"][:, 0].clone()
    for s in range(6):   # all begin with the first page of sequence 0, and its rows
        x["table"][s, 0] = first
        for i in (0, 1):
            x["rows"][s][i][:, :16] = x["rows"][0][i][:, :16]
    assert len(set(held.tolist())) == 3
    batch, (out, lse) = attend(ops, x)
    assert batch.members.tolist() == [3, 0, 0, 0, 2, 0] and batch.shared.tolist() == [512] * 3 + [0] + [320] * 2
    check(x, out, lse)


def put_row(x, s, j, which, row):
    """Row j of sequence s (head 0) in the pool (16 bits) and in what it is compared with."""
    x["kv"[which]][int(x["table"][s, j // x["page"]]), 0, j % x["page"]] = row.to(DEV)
    x["rows"][s][which][0, j] = row


@pytest.mark.parametrize("where", ["common", "own", "both"])
@pytest.mark.parametrize("size", [64.0, 1024.0])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_one_side_outweighs_the_other(ops, where, size, dtype):
    """A common row, a row of a sequence's own, or one of each, whose scores (exact:
    +-1 times +-size) are so far above all others that their weights are 0 in fp32:
    724 and 11585 times log2(e), the latter past what a weight's exponent may lose
    to rounding.  Few rows and tiles; the output is the row's value, or the mean."""
    prompts = (200, 320)
    x = forked([(200, ones(30, 30, 9)), (320, [(60, 50), (40, 40), (1, 1)])], 1, 2, 128, 8, dtype, seed=3)
    u = torch.where(torch.randn(128, generator=torch.Generator().manual_seed(1)) > 0, 1.0, -1.0).to(dtype)
    x["q"].copy_(u.to(DEV).expand_as(x["q"]))
    x["q64"] = u.double().expand(x["q64"].shape)
    for s in range(6):
        prompt = prompts[s // 3]
        if where != "own":
            put_row(x, s, 17, 0, u * size)
        if where != "common":
            put_row(x, s, prompt, 0, u * size)    # every token of the sequence sees it
    batch, (out, lse) = attend(ops, x)
    assert batch.shared.tolist() == [200] * 3 + [320] * 3
    check(x, out, lse)
    for s in range(6):
        prompt = prompts[s // 3]
        v = x["rows"][s][1][0].double()
        want = {"common": v[17], "own": v[prompt], "both": (v[17] + v[prompt]) / 2}[where]
        got = out[x["start_host"][s]:x["start_host"][s + 1]].double().cpu()
        # a weight is rounded to the type before it multiplies V and not in the sum that
        # divides (half a step), the output is rounded (half a step), sums in fp32
        value = (v[17].abs() + v[prompt].abs()) / (2 if where == "both" else 1)
        assert ((got - want).abs() <= (torch.finfo(dtype).eps + 2.0 ** -20) * value + 2.0 ** -24).all()


@pytest.mark.parametrize("fmt", [None, "fp8", "int8", "fp4"])
@pytest.mark.parametrize("where", ["common", "few", "tile"])
@pytest.mark.parametrize("own", [60, 3000])
def test_nan_in_shared_batches(ops, fmt, where, own):
    """A NaN (codes: a block of 32 dims) of V in a common row, in a row that a few
    new tokens of one sequence see, and in one that a part of a chunk sees: those get
    NaN in its dims and the bits of the call without it elsewhere, as all others do;
    whole results (60 own rows) and partials (3000)."""
    x = forked([(500, [(20, 3), (own, 50), (40, 1)]), (320, ones(30, 8))], 1, 4, 128, 16, BF, seed=4)
    if fmt:
        x = quantize(ops, x, fmt)
    _, (clean, lse0) = attend(ops, x)
    s, j, hit = {"common": (1, 323, slice(0, 54)), "few": (0, 518, slice(1, 3)),
                 "tile": (1, 500 + own - 10, slice(3 + 40, 3 + 50))}[where]
    page = int(x["table"][s, j // 16])
    if fmt:
        x["v"].exponents[page, 0, j % 16, 1] = 255
        dims = slice(32, 64)
    else:
        x["v"][page, 0, j % 16, 40] = float("nan")
        dims = slice(40, 41)
    batch, (out, lse) = attend(ops, x)
    assert batch.members.tolist() == [3, 0, 0, 2, 0]
    bad = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    bad[hit, :, dims] = True
    assert bool(torch.isnan(out[bad]).all()) and torch.equal(out[~bad], clean[~bad]) and torch.equal(lse, lse0)


@pytest.mark.parametrize("fmt", [None, "fp8"])
def test_out_may_be_the_queries(ops, fmt):
    """Runs whose first sequence has no new token, sequences on their own between
    them, few rows and a chunk: the queries' own memory takes the output."""
    groups = [(320, [(9, 0), (30, 2), (600, 60)]), (0, [(77, 1)]), (200, [(5, 0), (8, 0), (40, 3)]), (0, ones(900)),
              (128, [(90, 80), (3, 0), (1, 1)])]
    x = forked(groups, 2, 4, 128, 8, BF, seed=6, pad=2)
    if fmt:
        x = quantize(ops, x, fmt)
    batch, (out, lse) = attend(ops, x)
    assert batch.members.tolist() == [3, 0, 0, 0, 3, 0, 0, 0, 3, 0, 0]
    check(x, out, lse)
    q = x["q"].clone()
    _, (again, lse2) = attend(ops, dict(x, q=q), out=q)
    assert again is q and torch.equal(q[:-2], out[:-2]) and torch.equal(q[-2:], x["q"][-2:]) and torch.equal(lse2[:-2], lse[:-2])


def test_exponents_of_another_memory_order(ops):
    """Codes by head and exponents by token, and both in one buffer, row by row."""
    x = quantize(ops, forked([(200, ones(30, 8)), (0, [(300, 40)])], 2, 4, 128, 16, HF, seed=8), "int8")
    _, (want, lse) = attend(ops, x)
    check(x, want, lse)

    def by_token(pool):
        e = pool.exponents.transpose(1, 2).contiguous().transpose(1, 2)
        return ops.QuantizedPages(pool.codes, e)

    def one_buffer(pool):
        P, H, page, D = pool.codes.shape
        buf = torch.zeros((P, H, page, D + 16), dtype=torch.uint8, device=DEV)
        buf[..., :D], buf[..., D:D + D // 32] = pool.codes.view(torch.uint8), pool.exponents
        return ops.QuantizedPages(buf.view(torch.int8)[..., :D], buf[..., D:D + D // 32])

    for form in (by_token, one_buffer):
        y = dict(x, k=form(x["k"]), v=form(x["v"]))
        _, (out, _) = attend(ops, y)
        assert torch.equal(out, want)
        for a, b in zip(ops.read_pages(y["k"], y["v"], ops.PagedBatch(x["table"], x["lens"], x["start"], 40), rows=230),
                        ops.read_pages(x["k"], x["v"], ops.PagedBatch(x["table"], x["lens"], x["start"], 40), rows=230)):
            assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2]) and torch.equal(a[1, :, :208], b[1, :, :208])


@pytest.mark.parametrize("dtype,D,page", [(BF, 128, 16), (HF, 64, 8)])
def test_chunks_behind_long_common_rows(ops, dtype, D, page):
    """Chunks of up to 600 rows (tokens times heads), of runs and on their own, beside
    single tokens: common and own rows in several ranges each."""
    groups = [(3008, [(70, 40), (300, 1), (1500, 150), (90, 17)]), (0, ones(500)), (0, [(2700, 100)]),
              (1504, [(40, 16), (50, 30)])]
    x = forked(groups, 2, 4, D, page, dtype, seed=11, pad=1)
    out = torch.full(x["q"].shape, 3.0, dtype=dtype, device=DEV)
    batch, (_, lse) = attend(ops, x, out=out)
    assert batch.members.tolist() == [4, 0, 0, 0, 0, 0, 2, 0]
    check(x, out, lse)
    assert bool((out[-1] == 3).all())
