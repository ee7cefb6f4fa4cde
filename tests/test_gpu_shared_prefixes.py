"""share_prefixes against its definition, and attention that attends common rows
once, against the definition in 64 bits on the CPU (tolerances as in
test_gpu_paged_attention: joins of partial sums are fp32 there too)."""
import pytest
import torch

from conftest import gpu_available
from test_gpu_paged_attention import check
from test_gpu_quantized_pages import quantize

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
LEAST = 64   # rows


@pytest.fixture(scope="module")
def ops():
    from adaptiveimi_amd import ops

    return ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- the runs --

def runs(table, lens, start, page, labels=None):
    """(shared, members, leaders) by the definition."""
    S, cap = len(lens), table.shape[1] * page
    old = [max(min(max(n, 0), cap) - max(start[s + 1] - start[s], 0), 0) // page for s, n in enumerate(lens)]
    shared, members, leaders = [0] * S, [0] * S, list(range(S))
    s = 0
    while s < S:
        def joins(t):
            return (t < S and min(old[t - 1], old[t]) > 0 and table[t, 0] == table[t - 1, 0]
                    and (labels is None or labels[t] == labels[t - 1]))
        end = s + 1
        while joins(end):
            end += 1
        most = min(old[s:end])
        same = (table[s:end, :most] == table[s, :most]).all(0)
        pages = most if bool(same.all()) else int((~same).int().argmax())
        rows = pages * page // 8 * 8
        if end - s > 1 and rows >= LEAST:
            shared[s:end] = [rows] * (end - s)
            members[s] = end - s
            leaders[s:end] = [s] * (end - s)
        s = end
    return shared, members, leaders


def families(sizes, commons, page, width, seed=0, loners=1):
    """A table whose neighbouring sequences have `common` leading pages alike."""
    g = torch.Generator().manual_seed(seed)
    rows, fresh = [], iter(torch.randperm(1 << 20, generator=g).tolist())
    take = lambda n: [next(fresh) for _ in range(n)]
    for size, common in zip(sizes, commons):
        head = take(common)
        rows += [head + take(width - common) for _ in range(size)]
        rows += [take(width) for _ in range(loners)]
    return torch.tensor(rows, dtype=torch.int32)


@pytest.mark.parametrize("page,width", [(1, 300), (2, 90), (4, 40), (8, 20), (16, 40), (128, 1500)])
def test_runs(ops, page, width):
    sizes = [2, 70, 1, 200, 5, 3]
    commons = [width, width // 2, width, max(1, width // 3), 1, 0]
    table = families(sizes, commons, page, width, seed=page)
    S = len(table)
    g = torch.Generator().manual_seed(1)
    lens = (width * page - torch.randint(0, max(1, width * page // 4), (S,), generator=g)).tolist()
    lens[3], lens[90], lens[200] = 0, 5, 2 ** 31 - 1
    news = torch.randint(0, 4, (S,), generator=g).tolist()
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    labels = torch.randint(0, 2, (S,), generator=g).sort().values.tolist()
    dev = table.to(DEV)
    for lab in (None, labels):
        batch = ops.PagedBatch(dev, i32(lens), i32(start), 4)
        got = ops.share_prefixes(batch, page, labels=None if lab is None else i32(lab))
        want = runs(table, lens, start, page, lab)
        assert got.shared.tolist() == want[0] and got.members.tolist() == want[1]
        assert got.leaders.tolist() == want[2]
        assert got.saved.tolist() == [sum(max(m - 1, 0) * r for r, m in zip(*want[:2]))]
        assert batch.shared is None and got.lens is batch.lens


def test_runs_of_few(ops):
    for S in (1, 2, 64, 65, 129):
        table = i32([[5, 6, 7, 8, 9]]).repeat(S, 1)
        batch = ops.PagedBatch(table, i32([70] * S), i32(list(range(S + 1))), 1)
        got = ops.share_prefixes(batch, 16)
        rows = 64 if S > 1 else 0
        assert got.shared.tolist() == [rows] * S and got.members.tolist() == [S if rows else 0] + [0] * (S - 1)
    none = ops.share_prefixes(ops.PagedBatch(i32([]).view(0, 3), i32([]), i32([0]), 1), 16)
    q = torch.randn((2, 4, 64), device=DEV).to(BF)
    pool = torch.randn((3, 2, 16, 64), device=DEV).to(BF)
    assert ops.paged_attention(q, pool, pool, none).shape == q.shape


# ----------------------------------------------------------- the attention --

def forked(groups, H, G, D, page, dtype, layout="heads", seed=0, pad=0):
    """groups: (prompt rows, [(own rows, new tokens), ...]), the new tokens the
    last of the own rows.  Sequences of a group hold the same full pages of its
    prompt."""
    g = torch.Generator().manual_seed(seed)
    lens, news, rows, table_rows = [], [], [], []
    pages, fresh = [], 0
    def new_page():
        nonlocal fresh
        fresh += 1
        return fresh - 1
    for prompt, members in groups:
        pk, pv = (torch.randn((H, prompt, D), generator=g).to(dtype) for _ in range(2))
        same = [new_page() for _ in range(prompt // page)]
        for own, new in members:
            n = prompt + own
            k, v = (torch.cat([t, torch.randn((H, own, D), generator=g).to(dtype)], 1) for t in (pk, pv))
            held = same + [new_page() for _ in range(-(-n // page) - len(same))]
            lens.append(n), news.append(new), rows.append((k, v)), table_rows.append(held)
    P = fresh + 2
    ids = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lens), max(map(len, table_rows)) + 1), 2 ** 31 - 1, dtype=torch.int32)
    k, v = (torch.full((P, H, page, D), float("nan"), dtype=dtype) for _ in range(2))
    for s, held in enumerate(table_rows):
        for j, p in enumerate(held):
            table[s, j] = ids[p]
            part = slice(j * page, min(lens[s], (j + 1) * page))
            k[ids[p], :, :part.stop - part.start] = rows[s][0][:, part]
            v[ids[p], :, :part.stop - part.start] = rows[s][1][:, part]
    if layout == "tokens":
        k, v = (t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in (k, v))
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    q = torch.randn((start[-1] + pad, H * G, D), generator=g).to(dtype)
    return dict(q=q.to(DEV), k=k.to(DEV), v=v.to(DEV), table=table.to(DEV), lens=i32(lens), start=i32(start), rows=rows,
                q64=q.double(), lens_host=lens, start_host=start, H=H, G=G, D=D, dtype=dtype, page=page,
                most=max(news))


def attend(ops, x, labels=None, max_query=None, max_len=None, **kw):
    batch = ops.PagedBatch(x["table"], x["lens"], x["start"], max_query or x["most"], max_len)
    batch = ops.share_prefixes(batch, x["page"], labels, least_bytes=1)
    return batch, ops.paged_attention(x["q"], x["k"], x["v"], batch, return_lse=True, **kw)


ones = lambda *own: [(n, 1) for n in own]
FORMS = {
    # groups, H, G, D, page, dtype, layout
    "pair": ([(200, ones(5, 60))], 2, 4, 128, 8, BF, "heads"),
    "many": ([(700, ones(*range(1, 71)))], 1, 8, 128, 16, BF, "tokens"),                 # 560 rows: three tiles
    "groups": ([(130, ones(3, 9, 40)), (1000, ones(1, 300)), (5, ones(20)), (90, ones(7, 8, 9, 300, 2))], 2, 7, 64, 8,
               HF, "heads"),
    "long": ([(9000, ones(1, 17, 500))], 1, 4, 128, 16, BF, "heads"),                    # common rows cut into ranges
    "long_own": ([(300, ones(4000, 2, 2500))], 1, 4, 128, 32, BF, "tokens"),             # own rows joined
    "drafts": ([(400, [(9, 5), (30, 3), (6, 6)]), (64, [(2, 2), (2, 1)])], 2, 8, 128, 16, HF, "heads"),
    "chunks": ([(333, [(100, 100), (1, 1), (290, 200)]), (80, [(33, 1), (40, 40)])], 1, 4, 128, 16, BF, "heads"),
    "pages_of_one": ([(67, ones(3, 4))], 1, 4, 64, 1, BF, "heads"),
    "no_own_row_but_new": ([(256, ones(1, 1, 1, 1))], 1, 16, 128, 16, HF, "heads"),
    "wide": ([(150, ones(6, 7))], 1, 40, 64, 16, BF, "heads"),                           # more heads than the few-row kernel's
    "idle": ([(640, [(5, 1), (8, 0), (9, 2)])], 1, 4, 128, 16, BF, "heads"),             # no new token in between
}


@pytest.mark.parametrize("name", FORMS)
@pytest.mark.parametrize("fmt", [None, "fp8", "int8", "fp4"])
def test_shared_attention(ops, name, fmt):
    groups, *shape = FORMS[name]
    x = forked(groups, *shape, seed=len(name), pad=3)
    if fmt:
        x = quantize(ops, x, fmt)
    out = torch.full(x["q"].shape, 3.0, dtype=x["dtype"], device=DEV)
    batch, (_, lse) = attend(ops, x, out=out)
    assert int(batch.members.max()) > 1
    check(x, out, lse)
    assert bool((out[-3:] == 3).all())


@pytest.mark.parametrize("max_len", [None, 100])
def test_own_rows_in_one_workgroup(ops, max_len):
    """Short own rows with a hint that keeps whole sequences in a workgroup."""
    x = forked([(90, ones(1, 2, 3)), (300, ones(9, 8))], 2, 4, 128, 8, BF)
    _, (out, lse) = attend(ops, x, max_len=max_len)
    check(x, out, lse)


def test_windows_see_their_rows(ops):
    """With a window the common rows are hidden in part: attended by each."""
    x = forked([(300, ones(5, 60, 7))], 2, 4, 128, 16, BF)
    for window, sinks in ((64, 5), (290, 0), (10 ** 6, 3)):
        _, (out, lse) = attend(ops, x, window=window, sinks=sinks)
        check(x, out, lse, window, sinks)


def test_little_to_save(ops):
    """Below what sharing has to save, on the device's and on the host's count: the
    bits of the call without."""
    x = forked([(640, ones(30, 5, 90)), (640, ones(400))], 2, 4, 128, 16, BF)
    plain = ops.PagedBatch(x["table"], x["lens"], x["start"], 1)
    want = ops.paged_attention(x["q"], x["k"], x["v"], plain, return_lse=True)
    row = 2 * 2 * 128 * 2
    for least, same in ((2 * 640 * row, False), (2 * 640 * row + row, True), (10 ** 18, True), (None, True)):
        batch = ops.share_prefixes(plain, 16, least_bytes=least)
        assert batch.saved.tolist() == [2 * 640]
        out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch, return_lse=True)
        assert torch.equal(lse, want[1]) == same and (torch.equal(out, want[0]) or not same)
        check(x, out, lse)


def test_nothing_shared_changes_nothing(ops):
    """Sequences on their own: the bits of the call without."""
    x = forked([(0, ones(900)), (0, ones(30)), (0, [(70, 5)])], 2, 4, 128, 16, BF)
    batch, (out, lse) = attend(ops, x)
    assert not bool(batch.members.any())
    plain = ops.PagedBatch(x["table"], x["lens"], x["start"], x["most"])
    a, b = ops.paged_attention(x["q"], x["k"], x["v"], plain, return_lse=True)
    assert torch.equal(a, out) and torch.equal(b, lse)


def test_labels_and_repeats(ops):
    """Labels part neighbours; the same call gives the same bits."""
    x = forked([(512, ones(4, 40, 9, 300, 5, 6))], 1, 4, 128, 16, BF)
    batch, (out, lse) = attend(ops, x, labels=i32([1, 1, 0, 0, 0, 4]))
    assert batch.members.tolist() == [2, 0, 3, 0, 0, 0] and batch.shared.tolist() == [512] * 5 + [0]
    check(x, out, lse)
    _, again = attend(ops, x, labels=i32([1, 1, 0, 0, 0, 4]))
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_scores_far_from_zero(ops):
    """Common rows that outweigh a sequence's own, and the reverse, by more than
    fp32's range of exponentials."""
    for scale in (1.0, 1e4):
        x = forked([(200, ones(30, 30))], 1, 4, 128, 8, BF, seed=3)
        _, (out, lse) = attend(ops, x, scale=scale)
        plain = ops.PagedBatch(x["table"], x["lens"], x["start"], 1)
        a, b = ops.paged_attention(x["q"], x["k"], x["v"], plain, scale=scale, return_lse=True)
        assert bool(torch.isfinite(out).all())
        check(x, out, lse, scale=scale) if scale == 1.0 else None
        # one row takes all of the weight: its value, to bf16's rounding (the scores' order is the same fp32 sum)
        assert torch.allclose(out.float(), a.float(), rtol=2 ** -7, atol=2 ** -7) and torch.allclose(lse, b, rtol=1e-6)


@pytest.mark.parametrize("where", ["common", "own"])
def test_nan_rows_reach_those_that_see_them(ops, where):
    groups = [(500, [(20, 3), (20, 3), (40, 1)]), (320, ones(30, 8))]
    x = forked(groups, 1, 4, 128, 16, BF)
    _, (clean, _) = attend(ops, x)
    if where == "common":     # a row of the first group's prompt: all of its tokens
        x["v"][int(x["table"][1, 20]), 0, 3, 7] = float("inf")
        hit = slice(0, 7)
    else:                     # the last token but one of sequence 1: its last two
        j = 518
        x["v"][int(x["table"][1, j // 16]), 0, j % 16, 7] = float("inf")
        hit = slice(4, 6)
    _, (out, _) = attend(ops, x)
    bad = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    bad[hit, :, 7] = True
    assert bool((out[bad] == float("inf")).all()) and torch.equal(out[~bad], clean[~bad])


def test_captured_steps(ops):
    """share_prefixes and two layers in one graph, replayed as lengths and tables
    change; two graphs replayed in turn."""
    x = forked([(320, ones(5, 60, 20)), (96, ones(40, 30))], 2, 4, 128, 16, BF)
    y = forked([(128, ones(5, 6))], 2, 4, 128, 16, BF, seed=9)

    def step(x, out):
        batch = ops.share_prefixes(ops.PagedBatch(x["table"], x["lens"], x["start"], 1), x["page"], least_bytes=1)
        ops.paged_attention(x["q"], x["k"], x["v"], batch, out=out[0])
        ops.paged_attention(out[0], x["k"], x["v"], batch, out=out[1])

    outs, graphs = [], []
    for z in (x, y):
        out = [torch.zeros_like(z["q"]) for _ in range(2)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(z, out)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(z, out)
        outs.append(out), graphs.append(graph)
    for i in range(4):
        x["lens"].sub_(3 * i)
        if i == 2:   # the runs part
            x["table"][1, 2] = x["table"][3, 0]
        x["q"].copy_(torch.randn(x["q"].shape, device=DEV))
        for z, out, graph in zip((x, y), outs, graphs):
            graph.replay()
        torch.cuda.synchronize()
        for z, out in zip((x, y), outs):
            want = [torch.zeros_like(z["q"]) for _ in range(2)]
            step(z, want)
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_a_server_with_beams(ops):
    """Prompt, fork, several steps of beams in an 8-bit cache: what the shared
    attention gives is what each sequence's rows, read back, give in 64 bits."""
    import math

    H, G, D, page, P, S, M = 2, 4, 128, 16, 60, 4, 14
    table = ops.PageTable.empty(S, M, P, page, DEV)
    other = ops.PageTable.empty(S, M, P, page, DEV)
    pools = [ops.QuantizedPages.zeros(P, H, page, D, "fp8", DEV) for _ in range(2)]
    inv_freq = 10000.0 ** (-torch.arange(64, device=DEV).float() / 64)
    g = torch.Generator().manual_seed(0)

    def step(table, counts):
        assert ops.extend_pages(table, i32(counts), pools).all()
        start = [0]
        for c in counts:
            start.append(start[-1] + c)
        q, k, v = (torch.randn((start[-1], h, D), generator=g).to(BF).to(DEV) for h in (H * G, H, H))
        batch = ops.share_prefixes(table.batch(i32(start), max(counts)), least_bytes=1)
        q, _ = ops.qk_norm_rope(q, k, inv_freq=inv_freq, value=v, batch=batch, key_pages=pools[0], value_pages=pools[1])
        out, lse = ops.paged_attention(q, *pools, batch, return_lse=True)
        keys, values = ops.read_pages(*pools, batch)
        lens = table.lens.tolist()
        x = dict(q64=q.double().cpu(), rows=[(keys[s, :, :n].cpu(), values[s, :, :n].cpu()) for s, n in enumerate(lens)],
                 lens_host=lens, start_host=start, H=H, G=G, D=D, dtype=BF)
        check(x, out, lse)
        return batch

    assert not bool(step(table, [150, 0, 0, 0]).members.any())
    ops.fork_pages(table, i32([0, 0, 0, 0]), out=other)
    batch = step(other, [1, 1, 1, 1])
    assert batch.members.tolist() == [4, 0, 0, 0] and batch.shared.tolist() == [144] * 4
    for parents in ([0, 0, 2, 3], [1, 1, 1, 3], [3, 2, 2, 0]):
        table, other = other, table
        ops.fork_pages(table, i32(parents), out=other)
        step(other, [1, 2, 1, 1])
    table, other = other, table
    ops.fork_pages(table, i32([0, -1, 2, 3]), out=other)      # one has ended: it parts the others
    batch = step(other, [1, 0, 3, 1])
    assert batch.members.tolist() == [0, 0, 2, 0]
    assert math.isfinite(float(batch.shared.sum()))


@pytest.mark.parametrize("chunk", [1, 60])
def test_many_sequences(ops, chunk):
    """More tiles than a workgroup plans for itself, of common and of own rows."""
    groups = [(72, ones(*[1 + i % 9 for i in range(259)])), (64, ones(*[1 + i % 5 for i in range(258)]) + [(60, chunk)])]
    x = forked(groups, 1, 2, 64, 8, BF)
    batch, (out, lse) = attend(ops, x)
    assert sorted(batch.members.tolist())[-2:] == [259, 259]
    check(x, out, lse)


def test_a_batch_is_shared_again(ops):
    """The result of share_prefixes is a batch like others; the given one stays."""
    x = forked([(200, ones(5, 60, 9))], 2, 4, 128, 8, BF)
    plain = ops.PagedBatch(x["table"], x["lens"], x["start"], 1)
    once = ops.share_prefixes(plain, 8, least_bytes=1)
    twice = ops.share_prefixes(once, labels=i32([0, 0, 1]), least_bytes=1)
    assert plain.shared is None and once.members.tolist() == [3, 0, 0] and twice.members.tolist() == [2, 0, 0]
    for batch in (plain, once, twice):
        out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch, return_lse=True)
        check(x, out, lse)
    with pytest.raises(ValueError):
        ops.paged_attention(x["q"], x["k"][:, :, :4], x["v"][:, :, :4], once)   # pages of another size
    for kw in (dict(page_size=None), dict(page_size=8, labels=i32([0])), dict(page_size=8, least_bytes=0)):
        with pytest.raises(ValueError):
            ops.share_prefixes(plain, **kw)
    with pytest.raises(ValueError):
        ops.share_prefixes(once, 16)
    with pytest.raises(ValueError):
        ops.share_prefixes(ops.PagedBatch(None, x["lens"], x["start"], 1), 8)


def test_a_sequence_handed_to_retrieval(ops):
    """Rows of an 8-bit paged cache, read back, build the same index as the same rows
    in a tensor of their own."""
    H, D, page, n = 2, 128, 16, 700
    x = forked([(0, ones(n))], H, 4, D, page, BF, seed=5)
    x = quantize(ops, x, "int8")
    batch = ops.PagedBatch(x["table"], x["lens"], x["start"], 1)
    keys, values = ops.read_pages(x["k"], x["v"], batch, rows=n)
    own_k, own_v = (t.to(DEV).contiguous() for t in x["rows"][0])
    assert torch.equal(keys[0], own_k) and torch.equal(values[0], own_v)
    got = []
    for k, v in ((keys[0], values[0]), (own_k, own_v)):
        cent, labels, _ = ops.kmeans(k, (8, 8), 5)
        got.append(ops.build_index(k, v, cent, labels, (8, 8)))
    assert all(torch.equal(got[0][name], got[1][name]) for name in ("cell_count", "perm", "list_keys", "list_values"))
