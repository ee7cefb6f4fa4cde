"""The paged cache's operators together, as a server uses them: page tables
that grow, fork and are compacted, keys and values normed, rotated and stored,
attention over them; chunks of a prompt, decoding, beams."""
import pytest
import torch

from conftest import gpu_available
from test_gpu_paged_attention import expected
from test_gpu_qk_norm_rope import close, definition, freqs, weights

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = "cuda:0"
LAYERS = 2


@pytest.fixture(scope="module")
def ops():
    from adaptiveimi_amd import ops

    return ops


class Server:
    """S slots, LAYERS layers of pools; keeps on the host what every sequence
    stored (the bits), layer by layer."""

    def __init__(self, ops, S, M, P, page, Hq, Hk, D, dtype, window=0, sinks=0, token_major=False):
        self.ops, self.S, self.Hq, self.Hk, self.D, self.dtype = ops, S, Hq, Hk, D, dtype
        self.window, self.sinks, self.page = window, sinks, page
        self.tables = [ops.PageTable.empty(S, M, P, page, DEV) for _ in range(2)]
        shape = (P, page, Hk, D) if token_major else (P, Hk, page, D)
        self.pools = [[torch.full(shape, float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
                      for _ in range(LAYERS)]
        self.heads_first = (lambda t: t.transpose(1, 2)) if token_major else (lambda t: t)
        self.hist = [[None] * S for _ in range(LAYERS)]   # (k, v) [Hk, n, D] on the host
        self.lens = [0] * S
        self.weights = [weights(D, dtype, seed=i) for i in range(LAYERS)]
        self.inv_freq = freqs(D // 2)
        self.gen = torch.Generator().manual_seed(3)

    @property
    def flat_pools(self):
        return [t for layer in self.pools for t in layer]

    def i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def step(self, news, pad=0):
        ops, table = self.ops, self.tables[0]
        assert ops.extend_pages(table, self.i32(news), self.flat_pools).all()
        self.lens = [n + c for n, c in zip(self.lens, news)]
        start = [0]
        for c in news:
            start.append(start[-1] + c)
        N = start[-1] + pad
        batch = table.batch(self.i32(start), max_query=max(news))
        Hq, Hk, D = self.Hq, self.Hk, self.D
        pos = torch.tensor([n - c + i for n, c in zip(self.lens, news) for i in range(c)])
        for layer in range(LAYERS):
            qkv = torch.randn((N, Hq + 2 * Hk, D), generator=self.gen).to(self.dtype)
            q, k, v = qkv.to(DEV).split([Hq, Hk, Hk], dim=1)
            qw, kw = self.weights[layer]
            kp, vp = (self.heads_first(t) for t in self.pools[layer])
            out = torch.full((N, Hq, D), 9.0, dtype=self.dtype, device=DEV)
            q, _ = ops.qk_norm_rope(q, k, inv_freq=self.inv_freq.to(DEV), query_weight=qw.to(DEV),
                                    key_weight=kw.to(DEV), query_out=q, value=v, batch=batch, key_pages=kp,
                                    value_pages=vp)
            out, lse = ops.paged_attention(q, kp, vp, batch, window=self.window, sinks=self.sinks, out=out,
                                           return_lse=True)
            assert torch.all(out[start[-1]:] == 9.0)
            self.check(layer, qkv, q, out, lse, news, start, pos, kp, vp)

    def check(self, layer, qkv, q, out, lse, news, start, pos, kp, vp):
        Hq, Hk, D, n_new = self.Hq, self.Hk, self.D, start[-1]
        qw, kw = self.weights[layer]
        host = qkv[:n_new]
        close(q[:n_new], *definition(host[:, :Hq], qw, 1e-6, pos, self.inv_freq, False), D)
        wk, size = definition(host[:, Hq:Hq + Hk], kw, 1e-6, pos, self.inv_freq, False)
        table = self.tables[0].pages.cpu()
        rows = []
        for s, n in enumerate(self.lens):
            ids = table[s, :-(-n // self.page)].long().to(DEV)
            k, v = (t[ids].transpose(0, 1).flatten(1, 2)[:, :n].cpu() for t in (kp, vp))
            old, new = n - news[s], slice(start[s], start[s + 1])
            if old:   # earlier rows are the bits that were stored, wherever they moved
                assert torch.equal(k[:, :old], self.hist[layer][s][0]) and torch.equal(v[:, :old],
                                                                                       self.hist[layer][s][1])
            if news[s]:
                close(k[:, old:].transpose(0, 1), wk[new], size[new], D)
                assert torch.equal(v[:, old:].transpose(0, 1), host[new, Hq + Hk:])
            self.hist[layer][s] = (k, v)
            rows.append((k, v))
        x = dict(q64=q.double().cpu(), rows=rows, lens_host=self.lens, start_host=start, H=Hk, G=Hq // Hk, D=D,
                 dtype=self.dtype)
        want, want_lse, tol, ltol, mine = expected(x, self.window, self.sinks)
        assert torch.all((out.double().cpu() - want).abs()[mine] <= tol[mine])
        got = lse.double().cpu()[mine]
        assert torch.all((got - want_lse[mine]).abs() <= ltol[mine])

    def fork(self, parents):
        a, b = self.tables
        self.ops.fork_pages(a, self.i32(parents), out=b)
        self.tables = [b, a]
        ok = [0 <= p < self.S for p in parents]
        self.lens = [self.lens[p] if o else 0 for p, o in zip(parents, ok)]
        self.hist = [[layer[p] if o else None for p, o in zip(parents, ok)] for layer in self.hist]

    def compact(self):
        n = self.ops.compact_pages(self.tables[0], self.flat_pools).item()
        refs = self.tables[0].refs
        assert torch.all(refs[:n] > 0) and torch.all(refs[n:] == 0)


@pytest.mark.parametrize("page,Hq,Hk,D,dtype,window,sinks,token_major", [
    (16, 8, 2, 128, torch.bfloat16, 0, 0, False),
    (4, 3, 3, 64, torch.float16, 0, 0, True),
    (32, 8, 1, 64, torch.bfloat16, 100, 5, False),
])
def test_chunks_decode_beams_and_compaction(ops, page, Hq, Hk, D, dtype, window, sinks, token_major):
    s = Server(ops, 4, 512 // page, 2400 // page, page, Hq, Hk, D, dtype, window, sinks, token_major)
    s.step([130, 33, 0, 1], pad=3)         # prompts of any length
    s.step([70, 1, 0, 1])                  # a chunk among decoding sequences
    s.fork([0, 0, 0, 1])                   # beams of the first, the second moved on
    s.step([1, 1, 1, 1])                   # each writes its own copy of the shared page
    s.step([3, 3, 3, 1], pad=1)            # a few tokens are verified
    s.fork([2, 2, -1, 3])                  # one beam wins, one sequence ends
    s.step([1, 1, 5, 1])                   # and a new one begins in its place
    s.compact()
    s.step([1, 1, 1, 1])
    s.fork([-1, 1, -1, -1])
    s.compact()
    s.step([90, 1, 40, 2])


def test_a_batch_of_a_table_knows_its_pages(ops):
    """Pools of another page size, as a token-major pool that is not transposed
    looks like, and of fewer pages than the table's are refused."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = ops.PageTable.empty(2, 4, 12, 16, DEV)
    pool = torch.randn((12, 16, 8, 64), device=DEV).to(torch.bfloat16)      # token-major, pages of 16 rows, 8 heads
    assert ops.extend_pages(table, i32([20, 3]), [pool]).all()
    batch = table.batch(i32([0, 1, 2]), max_query=1)
    q = torch.randn((2, 32, 64), device=DEV).to(torch.bfloat16)
    k = q[:, :8]
    good = pool.transpose(1, 2)
    out = ops.paged_attention(q, good, good, batch)
    for bad, heads in ((pool, 16), (good[:11], 8)):
        with pytest.raises(ValueError, match="pages of 16 rows"):
            ops.paged_attention(q, bad, bad, batch)
        with pytest.raises(ValueError, match="pages of 16 rows"):
            ops.qk_norm_rope(q, q[:, :heads], value=q[:, :heads], batch=batch, key_pages=bad, value_pages=bad)
    more = torch.cat([pool, pool]).transpose(1, 2)      # more pages than the table's are never reached
    assert torch.equal(ops.paged_attention(q, more, more, batch), out)


def take_back(table, rejected):
    """Rows that verification rejected, as the integration notes give it."""
    page, cols = table.page_size, torch.arange(table.pages.shape[1], device=table.device)
    held = lambda lens: ((lens + page - 1) // page)[:, None]
    lens = (table.lens - rejected).clamp_(min=0)
    drop = (cols >= held(lens)) & (cols < held(table.lens))
    table.refs.scatter_add_(0, table.pages.clamp(min=0).flatten().long(), -drop.flatten().int())
    table.lens.copy_(lens)


def counted(table):
    """What refs has to be."""
    refs = [0] * table.refs.shape[0]
    for row, n in zip(table.pages.tolist(), table.lens.tolist()):
        for p in row[:-(-n // table.page_size)]:
            refs[p] += 1
    return refs


@pytest.mark.parametrize("page,dtype", [(4, torch.bfloat16), (16, torch.float16)])
def test_drafted_tokens_taken_back(ops, page, dtype):
    """Drafts verified and taken back across page borders, by sequences that
    share pages too: no page is lost, rows that stayed are the bits that were
    stored, and nobody writes into a page that another sequence holds."""
    s = Server(ops, 4, 256 // page, 900 // page, page, 4, 2, 64, dtype)
    s.step([50, 17, 0, 1])
    s.fork([0, 0, 1, 3])
    for news, rejected in (([5, 5, 5, 5], [5, 3, 0, 4]), ([9, 2, 7, 1], [8, 2, 1, 0]), ([1, 1, 1, 1], [0, 0, 0, 0]),
                           ([6, 6, 6, 6], [20, 6, 11, 9]), ([7, 5, 3, 2], [40, 0, 3, 9])):
        s.step(news)
        take_back(s.tables[0], s.i32(rejected))
        s.lens = [max(n - r, 0) for n, r in zip(s.lens, rejected)]
        s.hist = [[(k[:, :n], v[:, :n]) for (k, v), n in zip(layer, s.lens)] for layer in s.hist]
        assert s.tables[0].lens.tolist() == s.lens
        assert s.tables[0].refs.tolist() == counted(s.tables[0])
        if rejected[0] == 8:
            s.fork([0, 0, 2, 1])   # the last page of each is shared again
    s.compact()
    s.step([3, 2, 1, 9])
    s.fork([-1] * 4)
    assert not s.tables[0].refs.any()


def test_taking_back_in_a_graph(ops):
    """Extension and taking back captured together, replayed; an eager copy of
    the table follows."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    tables = [ops.PageTable.empty(5, 12, 40, 4, DEV) for _ in range(2)]
    counts, rejected = i32([0] * 5), i32([0] * 5)
    step = lambda t: (ops.extend_pages(t, counts), take_back(t, rejected))
    step(tables[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(tables[0])
    for new, back in (([9, 4, 1, 0, 17], [0, 0, 0, 0, 3]), ([5, 5, 5, 5, 5], [5, 4, 3, 2, 1]), ([1] * 5, [9, 0, 9, 0, 20]),
                      ([7, 0, 0, 12, 2], [0] * 5)):
        counts.copy_(i32(new))
        rejected.copy_(i32(back))
        graph.replay()
        step(tables[1])
        torch.cuda.synchronize()
        a, b = tables
        assert torch.equal(a.lens, b.lens) and torch.equal(a.refs, b.refs)
        assert a.refs.tolist() == counted(a) == counted(b)
