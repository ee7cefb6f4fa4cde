"""Runs of share_prefixes next to sequences that share little with them."""
import pytest
import torch

from conftest import gpu_available
from test_gpu_paged_attention import check
from test_gpu_shared_prefixes import attend, forked, ones

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = "cuda:0"
BF = torch.bfloat16


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
