"""ops.paged_attention against the definition in 64 bits on the CPU.

Tolerance.  With w the exact weights and A = sum w |v|, the kernel differs from
the exact output by: its weights rounded to the tensor type before the product
(half a step, eps / 2, relative to each weight: eps / 2 * A; in fp16 a weight
under 2^-14 keeps an absolute 2^-25 instead, against a sum of at least 1), the
scores' fp32 sums (at most (D + 2) 2^-24 sum |q k| scale each, which scales a
weight by as much, numerator and sum: twice), exp2 and its argument (2^-21 for
scores up to 8), the sums over n rows (n 2^-24 twice), and the output's own
rounding (eps / 2 relative)."""
import math

import pytest
import torch

from conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = "cuda:0"


def make(lens, news, H, G, D, page, dtype, layout="heads", seed=0, packed=False, pad=0, junk=float("nan"), slack=3):
    """Tensors on the device and their 64-bit copies.  Everything that no
    sequence owns (unused pages, slots behind a last row, table entries behind
    a last page) is junk."""
    g = torch.Generator().manual_seed(seed)
    S, N = len(lens), sum(news) + pad
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    width = Hw = H * G
    if packed:
        Hw = width + 2 * H
    q = torch.randn((N, Hw, D), generator=g).to(dtype)
    rows = [(torch.randn((H, n, D), generator=g).to(dtype), torch.randn((H, n, D), generator=g).to(dtype))
            for n in lens]
    if page:
        held = [-(-n // page) for n in lens]
        P = sum(held) + slack
        ids = torch.randperm(P, generator=g).tolist()
        table = torch.full((S, max(held + [0]) + 2), 2 ** 31 - 1, dtype=torch.int32)
        k = torch.full((P, H, page, D), junk, dtype=dtype)
        v = torch.full((P, H, page, D), junk, dtype=dtype)
        at = 0
        for s, n in enumerate(lens):
            for j in range(held[s]):
                p = ids[at]
                at += 1
                table[s, j] = p
                part = slice(j * page, min(n, (j + 1) * page))
                k[p, :, :part.stop - part.start] = rows[s][0][:, part]
                v[p, :, :part.stop - part.start] = rows[s][1][:, part]
        table = table.to(DEV)
    else:
        table = None
        k = torch.full((S, H, max(lens + [1]) + slack, D), junk, dtype=dtype)
        v = k.clone()
        for s, n in enumerate(lens):
            k[s, :, :n], v[s, :, :n] = rows[s]
    if layout == "tokens":
        k, v = (t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in (k, v))
    else:
        k, v = k.to(DEV), v.to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    return dict(q=q.to(DEV)[:, :width], k=k, v=v, table=table, lens=i32(lens), start=i32(start), rows=rows,
                q64=q[:, :width].double(), lens_host=lens, start_host=start, H=H, G=G, D=D, dtype=dtype)


def batch_of(ops, x, **kw):
    news = [b - a for a, b in zip(x["start_host"], x["start_host"][1:])]
    return ops.PagedBatch(x["table"], x["lens"], x["start"], max_query=max(news + [1]), **kw)


def expected(x, window=0, sinks=0, scale=None):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits; rows of no
    sequence are None in the mask."""
    H, G, D = x["H"], x["G"], x["D"]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    eps = torch.finfo(x["dtype"]).eps
    N = x["q64"].shape[0]
    out = torch.zeros((N, H * G, D), dtype=torch.float64)
    lse = torch.full((N, H * G), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    mine = torch.zeros(N, dtype=torch.bool)
    for s, n in enumerate(x["lens_host"]):
        a, b = x["start_host"][s], x["start_host"][s + 1]
        mine[a:b] = True
        k, v = x["rows"][s][0].double(), x["rows"][s][1].double()
        for t in range(a, b):
            p = n - (b - a) + t - a
            seen = [j for j in range(0, p + 1) if window == 0 or j > p - window or j < sinks]
            if not seen:
                continue
            for h in range(H):
                ks, vs = k[h, seen], v[h, seen]
                q = x["q64"][t, h * G:(h + 1) * G]
                sc = scale * q @ ks.T
                w = torch.softmax(sc, -1)
                o = w @ vs
                A = w @ vs.abs()
                ds = (D + 2) * 2.0 ** -24 * scale * (q.abs() @ ks.abs().T).amax(-1, keepdim=True) + 2.0 ** -21
                m = len(seen)
                err = (eps / 2 + 2 * ds + 2 * m * 2.0 ** -24) * A + eps / 2 * o.abs() + 1e-6
                if x["dtype"] == torch.float16:
                    err = err + 2.0 ** -25 * vs.abs().sum(0) + 2.0 ** -25
                hs = slice(h * G, (h + 1) * G)
                out[t, hs], tol[t, hs] = o, err
                lse[t, hs] = torch.logsumexp(sc, -1)
                ltol[t, hs] = (2 * ds[:, 0] + m * 2.0 ** -24) + 2.0 ** -22 * lse[t, hs].abs() + 1e-6
    return out, lse, tol, ltol, mine


def check(x, got, got_lse, window=0, sinks=0, scale=None):
    out, lse, tol, ltol, mine = expected(x, window, sinks, scale)
    got, got_lse = got.double().cpu(), got_lse.double().cpu()
    err = (got - out).abs()[mine]
    assert torch.all(err <= tol[mine]), f"out: {err.max()} (worst excess {(err - tol[mine]).max()})"
    empty = torch.isinf(lse) & mine[:, None]
    assert torch.all(got_lse[empty] == -math.inf) and torch.all(got[empty] == 0)
    live = ~torch.isinf(lse) & mine[:, None]
    lerr = (got_lse - lse).abs()[live]
    assert torch.all(lerr <= ltol[live]), f"lse: {lerr.max()}"


@pytest.fixture(scope="module")
def ops():
    from adaptiveimi_amd import ops

    return ops


BF, HF = torch.bfloat16, torch.float16
CASES = [
    # lens, news, H, G, D, page, dtype, window, sinks, layout
    ([1], [1], 1, 1, 128, 8, BF, 0, 0, "heads"),
    ([519], [1], 2, 4, 128, 8, BF, 0, 0, "heads"),
    ([2500], [1], 2, 4, 128, 16, BF, 0, 0, "heads"),           # several workgroups, joined
    ([2500, 3, 129, 1, 4000], [1] * 5, 2, 8, 128, 16, BF, 0, 0, "tokens"),
    ([700, 64, 1290], [1, 1, 1], 1, 16, 64, 32, HF, 0, 0, "heads"),
    ([700, 64, 1290], [5, 4, 3], 2, 3, 128, 64, HF, 100, 7, "tokens"),
    ([2000, 300], [5, 5], 2, 4, 64, 32, HF, 150, 32, "heads"),
    ([300, 40, 9], [8, 8, 8], 1, 4, 128, 1, BF, 0, 0, "heads"),
    ([300], [300], 1, 1, 128, 16, BF, 0, 0, "heads"),
    ([300], [300], 2, 4, 64, 16, HF, 0, 0, "tokens"),
    ([450], [130], 1, 7, 128, 16, BF, 0, 0, "heads"),
    ([450], [450], 1, 2, 128, 0, BF, 64, 4, "tokens"),
    ([450], [200], 1, 2, 128, 8, BF, 1, 0, "heads"),            # a token sees itself alone
    ([333], [333], 1, 3, 128, 8, HF, 5, 40, "heads"),           # more sinks than window
    ([200, 1, 333, 77, 64, 500], [1, 1, 150, 77, 2, 1], 2, 5, 128, 16, BF, 0, 0, "heads"),
    ([200, 1, 333, 77, 64, 500], [1, 1, 150, 77, 2, 1], 1, 33, 64, 16, BF, 90, 3, "tokens"),   # more than 32 rows a token
    ([64, 129, 31], [64, 129, 31], 1, 4, 128, 0, HF, 0, 0, "heads"),
    ([600], [100], 1, 4, 128, 8, BF, 301, 100, "heads"),        # sinks and window with a few rows between them
    ([700], [100], 1, 2, 64, 16, HF, 203, 69, "tokens"),        # a gap of more
    ([500], [90], 1, 4, 128, 1, BF, 0, 0, "heads"),             # pages of one row and of two
    ([500], [90], 1, 4, 128, 2, HF, 77, 5, "heads"),
    ([1500], [700], 1, 4, 128, 16, BF, 0, 0, "heads"),
]


@pytest.mark.parametrize("lens,news,H,G,D,page,dtype,window,sinks,layout", CASES)
def test_matches_definition(ops, lens, news, H, G, D, page, dtype, window, sinks, layout):
    x = make(lens, news, H, G, D, page, dtype, layout)
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), window=window, sinks=sinks,
                                   return_lse=True)
    check(x, out, lse, window, sinks)


def same_class(got, want, tol):
    """Equal infinities and NaN, and within tol elsewhere."""
    nan, inf = torch.isnan(want), torch.isinf(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[inf], want[inf])
    fin = ~nan & ~inf
    assert torch.all((got - want).abs()[fin] <= tol[fin])


@pytest.mark.parametrize("lens,news,H,G,D,page,dtype,window,sinks", [
    ([120], [120], 1, 4, 128, 16, BF, 0, 0),
    ([300], [300], 2, 2, 64, 16, HF, 0, 0),
    ([500], [300], 1, 5, 128, 8, BF, 70, 9),       # rows that leave a tile's window
    ([400, 90], [6, 5], 2, 4, 128, 16, HF, 0, 0),  # few rows
    ([400, 90], [3, 5], 1, 4, 64, 16, BF, 30, 2),
])
def test_infinities_and_nan_reach_only_what_sees_them(ops, lens, news, H, G, D, page, dtype, window, sinks):
    """Rows of V that hold infinities or NaN, the last rows among them, change
    the outputs of the tokens that see them and no other's."""
    x = make(lens, news, H, G, D, page, dtype)
    g = torch.Generator().manual_seed(7)
    for s, n in enumerate(lens):
        first = max(n - news[s], 0)
        for j in [n - 1, n - 2] + torch.randint(max(first - 3, 0), n, (6,), generator=g).tolist() + [0]:
            d = int(torch.randint(0, D, (1,), generator=g))
            h = int(torch.randint(0, H, (1,), generator=g))
            val = [math.inf, -math.inf, math.nan][int(torch.randint(0, 3, (1,), generator=g))]
            x["rows"][s][1][h, j, d] = val
            if j != 0 or window:   # a first row that every token sees makes for few finite outputs
                x["v"][int(x["table"][s, j // page]), h, j % page, d] = val
            else:
                x["rows"][s][1][h, j, d] = x["v"][int(x["table"][s, 0]), h, 0, d].cpu()
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), window=window, sinks=sinks,
                                   return_lse=True)
    want, want_lse, tol, ltol, mine = expected(x, window, sinks)
    assert torch.isfinite(want).any() and not torch.isfinite(want).all()
    same_class(out.double().cpu(), want, torch.nan_to_num(tol, nan=0.0, posinf=0.0))
    assert torch.all((lse.double().cpu() - want_lse).abs() <= ltol)


def test_nan_keys_reach_only_what_sees_them(ops):
    """A NaN key makes NaN of the tokens that see it; earlier ones, and those
    whose window has left it, stay as they are."""
    for news, window in ((150, 0), (150, 40), (5, 0), (5, 3)):
        x = make([200], [news], 2, 3, 128, 16, BF)
        clean = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), window=window)
        j = 200 - news + news // 2
        x["k"][int(x["table"][0, j // 16]), 1, j % 16, 5] = math.nan
        out = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), window=window)
        p = torch.arange(200 - news, 200)
        hit = (p >= j) & ((p < j + window) if window else True)
        assert torch.isnan(out[hit.to(DEV)][:, 3:]).all()
        keep = torch.ones((news, 6), dtype=torch.bool)
        keep[hit, 3:] = False
        assert torch.equal(out[keep.to(DEV)], clean[keep.to(DEV)])


def test_empty_sequences_and_rows(ops):
    """Sequences of no rows, of no new tokens, more new tokens than rows; rows
    of no sequence keep what the given outputs hold."""
    lens, news = [0, 7, 50, 3, 0, 200], [0, 0, 2, 5, 3, 150]
    for G in (1, 4):
        x = make(lens, news, 2, G, 128, 8, BF, pad=11)
        out = torch.full((sum(news) + 11, 2 * G, 128), 5.0, dtype=BF, device=DEV)
        lse = torch.full((sum(news) + 11, 2 * G), 6.0, device=DEV)
        a, b = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), out=out, lse=lse)
        assert a is out and b is lse
        check(x, out, lse)
        assert torch.all(out[sum(news):] == 5.0) and torch.all(lse[sum(news):] == 6.0)
    # nothing to do at all
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    out = ops.paged_attention(x["q"][:0], x["k"], x["v"], batch_of(ops, x))
    assert out.shape == (0, 8, 128)
    none = ops.PagedBatch(None, i32([]), i32([0]), max_query=1)
    assert ops.paged_attention(x["q"], x["k"], x["v"], none).shape == x["q"].shape


@pytest.mark.parametrize("news", [[1, 1, 1], [40, 3, 130]])
def test_strides(ops, news):
    """Queries inside a projection's rows, outputs inside a wider tensor, heads
    and tokens in either order."""
    lens = [300, 64, 500]
    x = make(lens, news, 2, 4, 64, 16, HF, layout="tokens", packed=True)
    assert not x["q"].is_contiguous()
    N = x["q"].shape[0]
    wide = torch.full((N, 3, 8, 64), 2.0, dtype=HF, device=DEV)
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), out=wide[:, 1], return_lse=True)
    check(x, out, lse)
    assert torch.all(wide[:, 0] == 2.0) and torch.all(wide[:, 2] == 2.0)
    by_head = torch.empty((8, N, 64), dtype=HF, device=DEV).transpose(0, 1)
    q2 = x["q"].transpose(0, 1).contiguous().transpose(0, 1)
    again = ops.paged_attention(q2, x["k"], x["v"], batch_of(ops, x), out=by_head)
    assert torch.equal(again, out)


def test_lies_about_lengths_stay_in_bounds(ops):
    """Lengths past the table, starts past the tensor and pages outside the
    pool are forced into range: the call returns, and what is well described
    is right."""
    x = make([100, 90], [1, 1], 1, 4, 128, 16, BF, junk=0.0)
    good = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    table = x["table"].clone()
    table[1] = -7
    b = ops.PagedBatch(table, i32([100, 10 ** 9]), i32([0, 1, 2 ** 30]), max_query=1)
    out = ops.paged_attention(x["q"], x["k"], x["v"], b)
    assert torch.equal(out[0], good[0])
    b = ops.PagedBatch(table, i32([100, -5]), i32([0, 1, -3]), max_query=1)
    out = ops.paged_attention(x["q"], x["k"], x["v"], b)
    assert torch.equal(out[0], good[0])


@pytest.mark.parametrize("S,n,news", [(1, 30000, 1), (1, 30000, 6), (70, 900, 1), (3, 9000, 33), (200, 40, 1)])
def test_splits_agree_with_one_call_per_sequence(ops, S, n, news):
    """Many sequences in one call, cut into ranges and joined, against each
    sequence alone with a hint that keeps it whole where that path exists."""
    g = torch.Generator().manual_seed(3)
    lens = [max(news, int(n * (0.3 + 0.7 * float(torch.rand((), generator=g))))) for _ in range(S)]
    x = make(lens, [news] * S, 1, 4, 64, 32, HF, seed=4)
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), return_lse=True)
    for s in range(0, S, max(1, S // 5)):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        b = ops.PagedBatch(x["table"][s:s + 1], i32([lens[s]]), i32([0, news]), max_query=news, max_len=1)
        one, one_lse = ops.paged_attention(x["q"][s * news:(s + 1) * news], x["k"], x["v"], b, return_lse=True)
        got, got_lse = out[s * news:(s + 1) * news], lse[s * news:(s + 1) * news]
        # each within eps of the same value (weights and output rounded), so within two of each other
        scale = one.double().abs().amax()
        assert (got.double() - one.double()).abs().max() <= 2 * 2.0 ** -10 * (scale + 1)
        assert (got_lse - one_lse).abs().max() <= 1e-4
    again = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x))
    assert torch.equal(again, out)   # the same call gives the same bits


def test_large_pages_offsets_past_32_bits(ops):
    """A pool of more than 2^32 bytes: pages far apart."""
    page, H, D = 128, 8, 128
    P = (5 << 30) // (page * H * D * 2)
    k = torch.zeros((P, H, page, D), dtype=BF, device=DEV)
    v = torch.zeros_like(k)
    x = make([500], [1], H, 4, D, page, BF, seed=8)
    far = [P - 1, 3, P - 7, P // 2]
    for j, p in enumerate(far):
        src = int(x["table"][0, j])
        k[p], v[p] = x["k"][src].nan_to_num(0.0), x["v"][src].nan_to_num(0.0)
    table = torch.tensor([far], dtype=torch.int32, device=DEV)
    for news in (1, 100):
        y = make([500], [news], H, 4, D, page, BF, seed=8)
        y["rows"] = x["rows"]
        b = ops.PagedBatch(table, y["lens"], y["start"], max_query=news)
        out, lse = ops.paged_attention(y["q"], k, v, b, return_lse=True)
        check(y, out, lse)


@pytest.mark.parametrize("lens,news", [([600, 40, 1], [1, 1, 1]), ([700, 90], [200, 5])])
def test_captured_replays_and_streams(ops, lens, news):
    """One captured call replayed as the batch changes, then the same call on
    two streams at once: every result equals the eager one."""
    x = make(lens, news, 2, 4, 128, 16, BF, junk=0.0)
    cap = x["table"].shape[1] * 16
    b = ops.PagedBatch(x["table"], x["lens"], x["start"], max_query=max(news))
    eager = lambda: ops.paged_attention(x["q"], x["k"], x["v"], b, return_lse=True)
    eager()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out, lse = eager()
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):   # a second capture on the stream
        eager()
    for step in range(4):
        x["q"].normal_()
        x["lens"].copy_(torch.tensor([max(1, n - 7 * step) for n in lens], dtype=torch.int32))
        graph.replay()
        want, want_lse = eager()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse), step
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(eager())
    graph.replay()
    torch.cuda.synchronize()
    for r, l in results:
        assert torch.equal(r, want) and torch.equal(l, want_lse)
    assert torch.equal(out, want)


def test_refusals(ops):
    x = make([40, 9], [2, 1], 2, 2, 64, 8, BF)
    b = batch_of(ops, x)
    call = lambda **kw: ops.paged_attention(**{**dict(query=x["q"], key_pages=x["k"], value_pages=x["v"], batch=b), **kw})
    with pytest.raises(TypeError):
        call(query=x["q"].float())
    with pytest.raises(TypeError):
        call(key_pages=x["k"].half())
    with pytest.raises(ValueError):
        call(query=x["q"][:, :3])
    with pytest.raises(ValueError):
        call(value_pages=x["v"][:, :, :4])
    with pytest.raises(ValueError):
        call(out=torch.empty_like(x["q"])[:1].expand(x["q"].shape))
    with pytest.raises(ValueError):
        call(lse=torch.empty((3, 4), device=DEV).double())
    with pytest.raises(ValueError):
        call(query=x["q"].cpu())
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    with pytest.raises(TypeError):
        ops.PagedBatch(x["table"], x["lens"].long(), x["start"], 2)
    with pytest.raises(ValueError):
        ops.PagedBatch(x["table"], x["lens"], x["start"][:2], 2)
    with pytest.raises(ValueError):
        ops.PagedBatch(x["table"][:1], x["lens"], x["start"], 2)
    with pytest.raises(ValueError):
        ops.PagedBatch(x["table"].T.contiguous().T, x["lens"], x["start"], 2)
    with pytest.raises(ValueError, match="contiguous rows"):
        ops.paged_attention(x["q"], x["k"][:1], x["v"][:1], ops.PagedBatch(None, x["lens"], x["start"], 2))
    from adaptiveimi_amd._lib import IMIError

    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(window=-1), dict(sinks=-2)):
        with pytest.raises(IMIError):
            call(**kw)
    with pytest.raises(IMIError, match="power of two"):
        call(key_pages=x["k"][:, :, :6], value_pages=x["v"][:, :, :6])
    with pytest.raises(IMIError, match="max_query"):
        call(batch=ops.PagedBatch(x["table"], x["lens"], x["start"], 0))


@pytest.mark.parametrize("G,news,max_query", [(4, [1, 2, 1], 1), (1, [3, 9, 2], 3), (8, [4, 2, 3], 3)])
def test_more_new_tokens_than_max_query(ops, G, news, max_query):
    """Sequences within max_query are right; rows of the others may be left,
    and nothing else is written."""
    lens = [3000, 2000, 900]
    x = make(lens, news, 2, G, 128, 16, BF, junk=0.0)
    b = ops.PagedBatch(x["table"], x["lens"], x["start"], max_query=max_query)
    N = sum(news)
    wide = torch.full((N + 2, 2 * G, 128), 7.0, dtype=BF, device=DEV)
    out = ops.paged_attention(x["q"], x["k"], x["v"], b, out=wide[1:-1])
    want, _, tol, _, _ = expected(x)
    for s, n in enumerate(news):
        rows = slice(x["start_host"][s], x["start_host"][s + 1])
        if n <= max_query:
            assert torch.all((out[rows].double().cpu() - want[rows]).abs() <= tol[rows])
        else:
            got = out[rows].double().cpu()
            assert torch.all((got == 7.0) | ((got - want[rows]).abs() <= tol[rows]))
    assert torch.all(wide[0] == 7.0) and torch.all(wide[-1] == 7.0)


def test_window_of_every_row_is_none(ops):
    for lens, news in (([900, 70], [1, 1]), ([900, 70], [300, 70])):
        x = make(lens, news, 1, 4, 64, 16, HF)
        cap = x["table"].shape[1] * 16
        want = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x))
        for window in (900, cap - 1, cap, 2 ** 31 - 1):
            got = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), window=window, sinks=2 ** 31 - 1)
            assert (got.double() - want.double()).abs().max() <= 2 * 2.0 ** -10 * (want.double().abs().max() + 1)


def test_more_heads_than_a_launch_has_workgroups(ops):
    """Half a million short sequences: their units are shared out."""
    S, H = (1 << 16) + 1, 64
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randn((3, H, 16, 64), generator=g, device=DEV).to(HF) for _ in range(2))
    q = torch.randn((S, H, 64), generator=g, device=DEV).to(HF)
    ids = torch.arange(S, device=DEV)
    lens, page = ids % 17, ids % 3
    b = ops.PagedBatch(page.int()[:, None].contiguous(), lens.int(), torch.arange(S + 1, device=DEV).int(), 1)
    out = ops.paged_attention(q, k, v, b)
    for n in (0, 1, 9, 16):
        for p in range(3):
            rows = ids[(lens == n) & (page == p)][:200]
            if n == 0:
                assert torch.all(out[rows] == 0)
                continue
            for h in (0, 63):
                qs, ks, vs = q[rows, h].double().cpu(), k[p, h, :n].double().cpu(), v[p, h, :n].double().cpu()
                w = torch.softmax(qs @ ks.T / 8, -1)
                err = (out[rows, h].double().cpu() - w @ vs).abs()
                # weights and output rounded: half a step each, and the scores' fp32 sums
                assert torch.all(err <= (2.0 ** -11 + 2.0 ** -17) * (w @ vs.abs()) + 2.0 ** -11 * (w @ vs).abs() + 1e-5)


def test_a_batch_serves_pools_of_its_own_sizes(ops):
    x = make([40], [1], 1, 1, 64, 8, HF)
    b = batch_of(ops, x)
    one = b.bind(5, 8, 1)
    two = b.bind(9, 16, 3)
    assert (one.n_pages, one.page_size, one.n_tokens) == (5, 8, 1)
    assert (two.n_pages, two.page_size, two.n_tokens) == (9, 16, 3)


def test_numbers_past_32_bits(ops):
    """Windows, sinks and bounds are not taken modulo 2^32."""
    x = make([90, 40], [1, 30], 1, 2, 64, 8, HF)
    want = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x))
    b = ops.PagedBatch(x["table"], x["lens"], x["start"], 2 ** 32 + 1, max_len=2 ** 32 + 1)
    assert torch.equal(ops.paged_attention(x["q"], x["k"], x["v"], b, window=2 ** 32 + 5, sinks=2 ** 33), want)
    assert torch.equal(ops.paged_attention(x["q"], x["k"], x["v"], b, window=10, sinks=2 ** 32 + 1),
                       ops.paged_attention(x["q"], x["k"], x["v"], b, window=10, sinks=90))
    with pytest.raises(ValueError, match="no columns"):
        ops.PagedBatch(x["table"][:, :0], x["lens"], x["start"], 1)


def test_out_may_be_the_queries(ops):
    for lens, news in (([700, 30], [1, 1]), ([3000, 300], [150, 300])):
        x = make(lens, news, 2, 4, 128, 16, BF)
        want = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x))
        q = x["q"].clone()
        assert ops.paged_attention(q, x["k"], x["v"], batch_of(ops, x), out=q) is q
        assert torch.equal(q, want)


@pytest.mark.parametrize("S,long", [(600, 0), (1100, 700)])
def test_many_sequences_of_many_rows(ops, S, long):
    """More tiles than a workgroup plans for itself, more sequences than a
    workgroup has threads; one sequence of many tiles among them."""
    g = torch.Generator().manual_seed(S)
    news = torch.randint(0, 11, (S,), generator=g).tolist()
    lens = [n + int(torch.randint(0, 14, (), generator=g)) for n in news]
    if long:
        news[S // 2], lens[S // 2] = long, long + 300
    x = make(lens, news, 1, 4, 64, 8, BF, seed=2)
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), return_lse=True)
    check(x, out, lse)


@pytest.mark.parametrize("n,news,H", [(700, 1, 1), (700, 5, 1), (6000, 3, 4), (600, 70, 1), (6000, 70, 2)])
@pytest.mark.parametrize("first", [1.6, 2.2, 2.5])
def test_many_small_weights_in_half_precision(ops, n, news, H, first):
    """One row without a value outweighs every other by 2^18, 2^25 or 2^29;
    what the others hold is the output.  A weight far under fp16's range keeps
    an absolute 2^-36 of the largest, not the 2^-25 that expected() allows."""
    G, D = 4, 64
    x = make([n], [news], H, G, D, 0, HF, slack=0)
    g = torch.Generator().manual_seed(12)
    k, v = x["rows"][0]
    k.copy_(0.05 * torch.randn(k.shape, generator=g))
    v.copy_(64.0 + 32.0 * torch.randn(v.shape, generator=g))
    q = (1.0 + 0.05 * torch.randn((news, H * G, D), generator=g)).to(HF)
    k[:, 0], v[:, 0] = first, 0.0      # scores 64 first / 8 above the others'
    x["k"][0], x["v"][0] = k.to(DEV), v.to(DEV)
    x["q"], x["q64"] = q.to(DEV), q.double()
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), return_lse=True)
    want, want_lse, tol, ltol, _ = expected(x)
    last = [n - news + i for i in range(news)]
    seen = torch.stack([v[:, :p + 1].double().abs().sum(1) for p in last]).repeat_interleave(G, 1)
    tol = tol - (2.0 ** -25 - 2.0 ** -36) * seen
    assert tol.min() > 0 and (want.abs() > 8 * tol).any()
    err = (out.double().cpu() - want).abs()
    assert torch.all(err <= tol), f"{err.max()} (worst excess {(err - tol).max()})"
    assert torch.all((lse.double().cpu() - want_lse).abs() <= ltol)


@pytest.mark.parametrize("n,news,D,dtype,window", [
    (300, 1, 128, BF, 0), (5000, 1, 64, HF, 0), (5000, 5, 128, BF, 0), (40, 45, 64, BF, 0), (3, 6, 128, HF, 0),
    (900, 70, 128, BF, 0), (900, 150, 64, HF, 50), (70, 90, 64, BF, 0),
])
def test_scores_of_minus_infinity(ops, n, news, D, dtype, window):
    """Softmax over scores that are all -infinity is 0 / 0: NaN, not the zeros of a
    token that sees nothing."""
    G = 4
    x = make([n], [news], 2, G, D, 0, dtype, slack=0)
    k = x["k"].clone()
    k[..., 0] = -1.0
    q = x["q"].clone()
    hit = torch.zeros((news, 2 * G), dtype=torch.bool, device=DEV)
    hit[::3, ::2] = True
    q[..., 0] = torch.where(hit, math.inf, q[..., 0])
    out, lse = ops.paged_attention(q, k, x["v"], batch_of(ops, x), window=window, return_lse=True)
    none = (torch.arange(news, device=DEV) < news - n)[:, None].expand_as(hit)
    assert torch.all(out[none] == 0) and torch.all(lse[none] == -math.inf)
    assert torch.isnan(out[hit & ~none]).all() and torch.all(lse[hit & ~none] == -math.inf)
    assert torch.isfinite(out[~hit]).all()


@pytest.mark.parametrize("n,news,window", [(300, 1, 0), (5000, 1, 0), (5000, 5, 0), (600, 5, 90), (900, 70, 0), (900, 150, 50)])
@pytest.mark.parametrize("dtype,size", [(HF, -2.0 ** 13), (HF, 2.0 ** 13), (BF, -2.0 ** 13), (BF, 2.0 ** 13), (BF, -2.0 ** 60),
                                        (BF, 2.0 ** 60), (HF, None), (BF, None)])
def test_scores_far_from_zero(ops, n, news, window, dtype, size):
    """Scores of size^2 plus a few units, or rows padded with the type's lowest
    value.  Every product and sum of them is exact in fp32, so what is left of the
    tolerance is the weights' rounding and the output's, and for exponents of up
    to 24 log2(e) their fp32 rounding (three of 2^-24 relative: 2^-17), the sums'
    (n 2^-24, twice) and exp2's."""
    H, G, D = 2, 4, 64
    x = make([n], [news], H, G, D, 0, dtype, slack=0, seed=3)
    g = torch.Generator().manual_seed(6)
    k, v = x["rows"][0]
    k.zero_()
    q = torch.zeros((news, H * G, D), dtype=dtype)
    q[..., 40] = 1.0
    k[..., 40] = 8.0 * torch.randint(0, 4, (H, n), generator=g)
    if size is None:     # seven of every ten blocks of 50 rows; not the last
        q[..., 0] = 255.0 if dtype == HF else 1.0
        block = torch.arange(n) // 50
        k[:, (block % 10 < 7) & (block < n // 50 - 1), 0] = torch.finfo(dtype).min
    else:
        q[..., 0] = abs(size)
        k[..., 0] = size
    if size is not None and abs(size) > 2 ** 20:
        k[..., 40] = 0.0     # (no sum of these is exact)
    x["k"][0], x["v"][0] = k.to(DEV), v.to(DEV)
    x["q"], x["q64"] = q.to(DEV), q.double()
    out, lse = ops.paged_attention(x["q"], x["k"], x["v"], batch_of(ops, x), scale=1.0, window=window, return_lse=True)
    want, want_lse, _, _, _ = expected(x, window, 0, 1.0)
    eps = torch.finfo(dtype).eps
    A = torch.zeros_like(want)
    for i in range(news):
        p = n - news + i
        first = max(0, p - window + 1) if window else 0
        for h in range(H):
            w = torch.softmax(x["q64"][i, h * G:(h + 1) * G] @ k[h, first:p + 1].double().T, -1)
            A[i, h * G:(h + 1) * G] = w @ v[h, first:p + 1].double().abs()
    tol = (eps / 2 + 2.0 ** -17 + 2 * n * 2.0 ** -24 + 2.0 ** -21) * A + eps / 2 * want.abs() + 1e-6
    err = (out.double().cpu() - want).abs()
    assert torch.all(err <= tol), f"{err.max()} (worst excess {(err - tol).max()})"
    lerr = (lse.double().cpu() - want_lse).abs()
    assert torch.all(lerr <= 2.0 ** -22 * want_lse.abs() + 2.0 ** -16 + n * 2.0 ** -23)


def test_numbers_under_32_bits(ops):
    """Nor are negative ones: they are refused as -1 is, and a hint is none."""
    from adaptiveimi_amd._lib import IMIError

    x = make([90, 40], [1, 30], 1, 2, 64, 8, HF)
    b = batch_of(ops, x)
    call = lambda b, **kw: ops.paged_attention(x["q"], x["k"], x["v"], b, **kw)
    for n in (-1, -2 ** 31, -2 ** 32 + 5, -2 ** 33):
        for kw in (dict(window=n), dict(window=9, sinks=n)):
            with pytest.raises(IMIError, match="must be >= 0"):
                call(b, **kw)
        with pytest.raises(IMIError, match="max_query"):
            call(ops.PagedBatch(x["table"], x["lens"], x["start"], n))
        assert torch.equal(call(ops.PagedBatch(x["table"], x["lens"], x["start"], 30, max_len=n)), call(b))
        table = ops.PageTable(x["table"], x["lens"], torch.zeros((9,), dtype=torch.int32, device=DEV), n)
        counts = torch.ones((2,), dtype=torch.int32, device=DEV)
        for f in (lambda: ops.fork_pages(table, counts), lambda: ops.extend_pages(table, counts),
                  lambda: ops.compact_pages(table)):
            with pytest.raises(IMIError, match="page_size"):
                f()


@pytest.mark.parametrize("P,H,page", [(9, 1, 8), (9, 2, 1), (1, 2, 64)])
def test_keys_and_values_of_one_layout(ops, P, H, page):
    """Strides of a dimension with one entry are torch's to choose: a head-major
    key pool and a token-major value pool of one head are the same layout."""
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn((P, H, page, 64), generator=g, device=DEV).to(BF) for _ in range(2))
    other = v.as_strided(v.shape, [s if n > 1 else 8 for s, n in zip(v.stride(), v.shape)])
    assert other.stride() != k.stride()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    b = ops.PagedBatch(i32([list(range(P))]), i32([P * page - 1]), i32([0, 1]), 1)
    q = torch.randn((1, 2, 64), generator=g, device=DEV).to(BF)
    assert torch.equal(ops.paged_attention(q, k, other, b), ops.paged_attention(q, k, v, b))
