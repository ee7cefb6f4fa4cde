"""ops.qk_norm_rope against the definition in 64 bits on the CPU.

Tolerance of an element: the output's rounding (eps / 2 relative to it) plus
the fp32 arithmetic relative to the normed pair's size m = |y_a| + |y_b| (or
|y| where nothing turns): the sum of D squares, division, root and two products
(under (D / 2 + 8) 2^-24), sine and cosine of the reduced angle (4 2^-24, and
2^-22 from the fraction of a turn in fp32 times 2 pi), two products and a sum
(3 2^-24)."""
import math

import pytest
import torch

from conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from adaptiveimi_amd import ops

    return ops


def definition(x, w, eps, pos, inv_freq, interleaved):
    """(value, size of what the rounding errors are relative to), 64 bits."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    m = y.abs().clone()
    z = y.clone()
    if inv_freq is not None:
        r = 2 * len(inv_freq)
        ang = pos.double()[:, None] * inv_freq.double()[None]
        for i in range(r // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
            c, s = torch.cos(ang[:, i])[:, None], torch.sin(ang[:, i])[:, None]
            z[..., a] = y[..., a] * c - y[..., b] * s
            z[..., b] = y[..., b] * c + y[..., a] * s
            m[..., a] = m[..., b] = y[..., a].abs() + y[..., b].abs()
    return z, m


def close(got, want, size, D):
    eps = torch.finfo(got.dtype).eps
    tiny = 2.0 ** -24 if got.dtype == HF else 0.0   # half a step of fp16's subnormals, and to spare
    tol = eps / 2 * want.abs() + ((D / 2 + 15) * 2.0 ** -24 + 2.0 ** -22) * size * (1 + eps) + tiny
    err = (got.double().cpu() - want).abs()
    assert torch.all(err <= tol), f"{err.max()} (excess {(err - tol).max()})"


def inputs(N, Hq, Hk, D, dtype, seed=0, packed=True):
    g = torch.Generator().manual_seed(seed)
    qkv = (2 * torch.randn((N, (Hq + 2 * Hk) * D), generator=g)).to(dtype)
    d = qkv.to(DEV)
    cut = [(0, Hq), (Hq, Hq + Hk), (Hq + Hk, Hq + 2 * Hk)]
    views = lambda t: [t[:, a * D:b * D].unflatten(1, (b - a, D)) for a, b in cut]
    host, dev = views(qkv), views(d)
    if not packed:
        dev = [t.contiguous() for t in dev]
    return host, dev


def weights(D, dtype, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [(1 + 0.3 * torch.randn((D,), generator=g)).to(dtype) for _ in range(2)]


def freqs(r, theta=500000.0):
    return (theta ** (-torch.arange(0, r // 2, dtype=torch.float64) * 2 / r)).float()


@pytest.mark.parametrize("N,Hq,Hk,D,dtype,rotary,interleaved,norm,wtype,pos64", [
    (1, 4, 1, 128, BF, 128, False, True, BF, False),
    (1, 1, 1, 64, HF, 64, False, True, HF, True),
    (37, 6, 2, 64, HF, 32, True, True, torch.float32, False),
    (130, 8, 8, 128, BF, 64, False, True, torch.float32, True),
    (600, 5, 1, 128, BF, 96, False, True, BF, False),
    (600, 32, 8, 128, HF, 128, True, False, None, False),
    (2100, 3, 1, 64, BF, 16, False, True, BF, False),
    (9, 70, 2, 128, BF, 0, False, True, BF, False),
    (5, 2, 2, 128, BF, 128, False, False, None, False),
])
def test_positions(ops, N, Hq, Hk, D, dtype, rotary, interleaved, norm, wtype, pos64):
    (q, k, _), (dq, dk, _) = inputs(N, Hq, Hk, D, dtype)
    qw, kw = weights(D, wtype) if norm else (None, None)
    f = freqs(rotary) if rotary else None
    g = torch.Generator().manual_seed(9)
    pos = torch.randint(0, 1_000_000, (N,), generator=g).to(torch.int64 if pos64 else torch.int32)
    pos[0] = 0
    dev = lambda t: None if t is None else t.to(DEV)
    qo, ko = ops.qk_norm_rope(dq, dk, pos.to(DEV), inv_freq=dev(f), query_weight=dev(qw), key_weight=dev(kw),
                              eps=1e-5, interleaved=interleaved)
    assert qo.shape == (N, Hq, D) and ko.shape == (N, Hk, D)
    close(qo, *definition(q, qw, 1e-5, pos, f, interleaved), D)
    close(ko, *definition(k, kw, 1e-5, pos, f, interleaved), D)
    # in place, in the projection's own rows
    a, b = ops.qk_norm_rope(dq, dk, pos.to(DEV), inv_freq=dev(f), query_weight=dev(qw), key_weight=dev(kw), eps=1e-5,
                            interleaved=interleaved, query_out=dq, key_out=dk)
    assert a is dq and b is dk and torch.equal(dq, qo) and torch.equal(dk, ko)


@pytest.mark.parametrize("lens,news,page,D,dtype,layout,pad", [
    ([1], [1], 16, 128, BF, "heads", 0),
    ([40, 7, 9, 128], [1, 7, 0, 100], 8, 64, HF, "tokens", 5),
    ([100] * 70, [1] * 70, 16, 128, BF, "heads", 3),     # more sequences than a wave has lanes
    ([5, 0, 3], [5, 0, 3], 0, 128, BF, "heads", 2),      # contiguous rows
    ([3, 20], [5, 2], 4, 128, BF, "tokens", 0),          # more new tokens than rows: the first two have none
])
def test_stored_in_pages(ops, lens, news, page, D, dtype, layout, pad):
    Hq, Hk = 6, 2
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    N = start[-1] + pad
    (q, k, v), (dq, dk, dv) = inputs(N, Hq, Hk, D, dtype)
    qw, kw = weights(D, dtype)
    f = freqs(D)
    S = len(lens)
    if page:
        held = [-(-n // page) for n in lens]
        ids = torch.randperm(sum(held) + 4, generator=torch.Generator().manual_seed(1)).tolist()
        table = torch.full((S, max(held) + 1), -1, dtype=torch.int32)
        at = 0
        for s in range(S):
            for j in range(held[s]):
                table[s, j] = ids[at]
                at += 1
        P, rows = len(ids), page
    else:
        table, P, rows = None, S, max(lens)
    shape = (P, Hk, rows, D) if layout == "heads" else (P, rows, Hk, D)
    order = (lambda t: t) if layout == "heads" else (lambda t: t.transpose(1, 2))
    kp, vp = (order(torch.full(shape, 7.0, dtype=dtype, device=DEV)) for _ in range(2))
    qo = torch.full((N, Hq, D), 9.0, dtype=dtype, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    batch = ops.PagedBatch(None if table is None else table.to(DEV), i32(lens), i32(start), max_query=max(news))
    got, none = ops.qk_norm_rope(dq, dk, value=dv, batch=batch, key_pages=kp, value_pages=vp, inv_freq=f.to(DEV),
                                 query_weight=qw.to(DEV), key_weight=kw.to(DEV), query_out=qo)
    assert got is qo and none is None
    assert torch.all(qo[start[-1]:] == 9.0)
    pos = torch.tensor([lens[s] - news[s] + i for s in range(S) for i in range(news[s])])
    n = start[-1]
    zq, mq = definition(q[:n], qw, 1e-6, pos, f, False)
    zk, mk = definition(k[:n], kw, 1e-6, pos, f, False)
    close(qo[:n], zq, mq, D)
    seq = [s for s in range(S) for _ in range(news[s])]
    touched = torch.zeros((P, rows), dtype=torch.bool)
    for t in range(n):
        p = int(pos[t])
        if p < 0:
            continue
        at = (int(table[seq[t], p // page]), p % page) if page else (seq[t], p)
        touched[at] = True
        close(kp[at[0], :, at[1]], zk[t], mk[t], D)
        assert torch.equal(vp[at[0], :, at[1]].cpu(), v[t])
    rest = ~touched.to(DEV)
    assert torch.all(kp.transpose(1, 2)[rest] == 7.0) and torch.all(vp.transpose(1, 2)[rest] == 7.0)


def test_no_page_no_store(ops):
    """Rows whose table entry is no page of the pool are not stored."""
    (_, _, _), (dq, dk, dv) = inputs(40, 2, 1, 128, BF)
    table = torch.tensor([[1, -1, 2 ** 31 - 1, 3, 0]], dtype=torch.int32, device=DEV)
    kp = torch.full((4, 1, 8, 128), 7.0, dtype=BF, device=DEV)
    vp = kp.clone()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    ops.qk_norm_rope(dq, dk, value=dv, batch=ops.PagedBatch(table, i32([40]), i32([0, 40]), 40), key_pages=kp,
                     value_pages=vp)
    assert torch.equal(kp[1, 0], dk[:8, 0]) and torch.equal(kp[3, 0], dk[24:32, 0])
    assert torch.equal(kp[0, 0], dk[32:, 0]) and torch.all(kp[2] == 7.0) and torch.all(vp[2] == 7.0)


def test_far_positions(ops):
    """The largest positions: the fraction of a turn is taken in 64 bits."""
    (q, k, _), (dq, dk, _) = inputs(4, 2, 1, 128, HF)
    pos = torch.tensor([2 ** 31 - 1, -5, 2 ** 20, 1], dtype=torch.int32)
    f = freqs(128)
    qo, ko = ops.qk_norm_rope(dq, dk, pos.to(DEV), inv_freq=f.to(DEV))
    # 2^31 turns of 2^-53 relative: 2^-22 of a turn more than the tolerance counts at the far end
    for got, x in ((qo, q), (ko, k)):
        z, m = definition(x, None, 0.0, pos, f, False)
        close(got, z, m * 2, 128)


def test_captured_and_on_streams(ops):
    """A captured store replayed as positions move, and two streams at once."""
    (_, _, _), (q, k, v) = inputs(6, 4, 2, 128, BF)
    qw, kw = (w.to(DEV) for w in weights(128, BF))
    f = freqs(128).to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    lens, start = i32([30, 9, 50]), i32([0, 1, 5, 6])
    table = torch.randperm(12, device=DEV).int().view(3, 4)
    pools = [torch.zeros((12, 2, 16, 128), dtype=BF, device=DEV) for _ in range(4)]
    batch = ops.PagedBatch(table, lens, start, 4)
    call = lambda out, kp, vp: ops.qk_norm_rope(q, k, inv_freq=f, query_weight=qw, key_weight=kw, query_out=out,
                                                value=v, batch=batch, key_pages=kp, value_pages=vp)
    outs = [torch.zeros_like(q, memory_format=torch.contiguous_format) for _ in range(4)]
    call(outs[0], *pools[:2])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call(outs[1], *pools[2:])
    for step in range(4):
        q.normal_()
        lens.copy_(i32([30 + step, 9 + 2 * step, 50 + step]))
        graph.replay()
        call(outs[0], *pools[:2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(pools[0], pools[2])
        # (the first eager call, before the graph, stored the first step's values too)
        assert torch.equal(pools[1], pools[3])
    pos = torch.arange(6, device=DEV)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.qk_norm_rope(q, k, pos, inv_freq=f, query_weight=qw, key_weight=kw))
    torch.cuda.synchronize()
    assert all(torch.equal(a, got[0][0]) and torch.equal(b, got[0][1]) for a, b in got)


def test_refusals(ops):
    from adaptiveimi_amd._lib import IMIError

    (_, _, _), (q, k, v) = inputs(3, 4, 2, 128, BF, packed=False)
    pos = torch.arange(3, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = i32([[0, 1]])
    pages = torch.zeros((2, 2, 16, 128), dtype=BF, device=DEV)
    batch = ops.PagedBatch(table, i32([3]), i32([0, 3]), 3)
    store = dict(value=v, batch=batch, key_pages=pages, value_pages=pages.clone())
    for kw in (dict(), dict(positions=pos, **store), dict(batch=batch), dict(positions=pos, value=v),
               dict(key_out=k, **store), dict(positions=pos[:2]), dict(positions=pos.cpu()),
               dict(positions=pos, inv_freq=torch.ones(64, dtype=torch.float64, device=DEV)),
               dict(positions=pos, query_weight=torch.ones(64, dtype=BF, device=DEV)),
               dict(positions=pos, query_out=q[:1].expand(q.shape)),
               dict(store, value=v[:2]), dict(store, key_pages=pages[:, :1], value_pages=pages[:, :1]),
               dict(store, key_pages=pages[:1].expand(2, -1, -1, -1), value_pages=pages[:1].expand(2, -1, -1, -1))):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(q, k, **kw)
    for kw in (dict(positions=pos.float()), dict(positions=pos, query_weight=torch.ones(128, dtype=HF, device=DEV)),
               dict(positions=pos, query_weight=torch.ones(128, dtype=BF, device=DEV),
                    key_weight=torch.ones(128, device=DEV)), dict(store, key_pages=pages.half())):
        with pytest.raises(TypeError):
            ops.qk_norm_rope(q, k, **kw)
    with pytest.raises(IMIError, match="rotary"):
        ops.qk_norm_rope(q, k, pos, inv_freq=torch.ones(4, device=DEV))
    with pytest.raises(IMIError, match="eps"):
        ops.qk_norm_rope(q, k, pos, eps=-1.0)
    with pytest.raises(IMIError, match="dim=96"):
        ops.qk_norm_rope(q[..., :96].contiguous(), k[..., :96].contiguous(), pos)
    none = ops.qk_norm_rope(q[:0], k[:0], pos[:0])
    assert none[0].shape == (0, 4, 128) and none[1].shape == (0, 2, 128)
