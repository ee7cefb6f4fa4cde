"""How many rows read_pages gives, and where it may write them."""
import pytest
import torch

from conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from adaptiveimi_amd import ops

    return ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rows_pool(P, H, page, D):
    g = torch.Generator().manual_seed(2)
    return [torch.randn((P, H, page, D), generator=g).to(BF).to(DEV) for _ in range(2)]


def test_rows_by_default(ops):
    """max_len says how many rows a read gives, up to what the table holds; rows says
    otherwise.  Attention sees all rows whatever it says."""
    pools = rows_pool(8, 2, 16, 64)
    table = i32([[0, 1, 2, 3], [4, 5, 6, 7]])
    lens = [64, 40]
    make = lambda max_len: ops.PagedBatch(table, i32(lens), i32([0, 1, 2]), 1, max_len)
    whole = [t[table.long()].permute(0, 2, 1, 3, 4).reshape(2, 2, 64, 64) for t in pools]
    for max_len, rows, gives in ((None, None, 64), (64, None, 64), (70, None, 64), (2 ** 40, None, 64), (50, None, 50),
                                 (50, 64, 64), (10, 64, 64), (50, 66, 66)):
        for t, want in zip(ops.read_pages(*pools, make(max_len), rows=rows), whole):
            assert t.shape == (2, 2, gives, 64), max_len
            for s, n in enumerate(lens):
                assert torch.equal(t[s, :, :min(n, gives)], want[s, :, :min(n, gives)])
    q = torch.randn((2, 4, 64), device=DEV).to(BF)
    full = ops.paged_attention(q, *pools, make(None))
    assert torch.equal(ops.paged_attention(q, *pools, make(10)), full)


def test_outputs_that_are_one_tensor(ops):
    """Keys and values read into the same memory: refused; into one buffer side by
    side: not."""
    pools = rows_pool(4, 2, 16, 64)
    batch = ops.PagedBatch(i32([[0, 1, 2, 3]]), i32([20]), i32([0, 1]), 1)
    out = torch.zeros((1, 2, 64, 64), dtype=BF, device=DEV)
    with pytest.raises(ValueError):
        ops.read_pages(*pools, batch, out=(out, out))
    both = torch.zeros((1, 2, 64, 2, 64), dtype=BF, device=DEV)      # keys and values of a row together
    got = ops.read_pages(*pools, batch, out=(both[..., 0, :], both[..., 1, :]))
    want = ops.read_pages(*pools, batch)
    for a, b in zip(got, want):
        assert torch.equal(a[:, :, :20], b[:, :, :20])
