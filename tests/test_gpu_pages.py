"""ops.fork_pages, extend_pages and compact_pages against their rules applied
one sequence after another on the CPU; everything has to be equal."""
import pytest
import torch

from conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a HIP device")]

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from adaptiveimi_amd import ops

    return ops


class Model:
    """The rules, in the plainest form; pools are lists of page contents."""

    def __init__(self, S, M, P, page, n_pools=0):
        self.S, self.M, self.P, self.page = S, M, P, page
        self.rows = [[] for _ in range(S)]
        self.lens = [0] * S
        self.pools = [[(i, p) for p in range(P)] for i in range(n_pools)]

    def refs(self):
        r = [0] * self.P
        for row in self.rows:
            for p in row:
                r[p] += 1
        return r

    def fork(self, parents):
        ok = [0 <= p < self.S for p in parents]
        self.rows, self.lens = ([list(self.rows[p]) if o else [] for p, o in zip(parents, ok)],
                                [self.lens[p] if o else 0 for p, o in zip(parents, ok)])

    def extend(self, counts):
        refs = self.refs()
        free = [p for p in range(self.P) if refs[p] == 0]
        granted, used = [], 0
        writes = []
        for s, c in enumerate(counts):
            c = max(c, 0)
            held, after = len(self.rows[s]), -(-(self.lens[s] + c) // self.page)
            if after > self.M:
                granted.append(False)
                continue
            copy = c > 0 and self.lens[s] % self.page != 0 and refs[self.rows[s][-1]] > 1
            need = after - held + copy
            used += need
            ok = need == 0 or used <= len(free)
            granted.append(ok)
            if not ok:
                continue
            new = free[used - need:used]
            if copy:
                writes.append((self.rows[s][-1], new[0]))
                self.rows[s][-1] = new[0]
                new = new[1:]
            self.rows[s] += new
            self.lens[s] += c
        for pool in self.pools:
            old = list(pool)
            for a, b in writes:
                pool[b] = old[a]
        return granted

    def compact(self):
        refs = self.refs()
        n = sum(r > 0 for r in refs)
        to = [p for p in range(n) if refs[p] == 0]
        fro = [p for p in range(n, self.P) if refs[p] > 0]
        where = dict(zip(fro, to))
        self.rows = [[where.get(p, p) for p in row] for row in self.rows]
        for pool in self.pools:
            for a, b in zip(fro, to):
                pool[b] = pool[a]
        return n

    def same(self, table):
        assert table.lens.tolist() == self.lens
        assert table.refs.tolist() == self.refs()
        pages = table.pages.tolist()
        for s in range(self.S):
            assert pages[s][:len(self.rows[s])] == self.rows[s], s


def content(shape, i):
    """Pool i: page p filled with a value of its own."""
    P = shape[0]
    v = (torch.arange(P, dtype=torch.int32) * 64 + i).view(P, *([1] * (len(shape) - 1)))
    return v.expand(shape).contiguous().to(DEV)


def pools_equal(model, pools):
    for i, pool in enumerate(pools):
        want = torch.tensor([p * 64 + j for j, p in model.pools[i]], dtype=torch.int32, device=DEV)
        assert torch.equal(pool, want.view(-1, *([1] * (pool.dim() - 1))).expand_as(pool))


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("S,M,P,page,steps,seed", [
    (1, 4, 3, 1, 6, 0),
    (4, 10, 40, 8, 12, 1),
    (7, 33, 100, 16, 15, 2),
    (33, 20, 300, 4, 12, 3),
    (130, 12, 900, 8, 8, 4),
    (1500, 6, 5000, 2, 5, 5),       # more sequences than a workgroup has threads
    (20, 2000, 36000, 3, 6, 6),     # more pages than one pass takes; a page size that is no power of two
])
def test_random_walk(ops, S, M, P, page, steps, seed):
    """Forks, frees, growth past what the pool or the table holds, compaction,
    in a random order; every state is compared."""
    import random

    rng = random.Random(seed)
    m = Model(S, M, P, page, n_pools=2)
    table = ops.PageTable.empty(S, M, P, page, DEV)
    other = ops.PageTable.empty(S, M, P, page, DEV)
    shapes = [(P, 2, 4), (P, 36)]
    pools = [content(shapes[0], 0), content(shapes[1], 1)]
    assert ops.extend_pages(table, i32([0] * S), pools).tolist() == m.extend([0] * S)
    for _ in range(steps):
        big = max(1, int(1.5 * page * min(M, P / S) / 3))
        counts = [rng.choice([0, 1, 1, -3, rng.randint(1, big), rng.randint(1, 2 * big)]) for _ in range(S)]
        assert ops.extend_pages(table, i32(counts), pools).tolist() == m.extend(counts)
        m.same(table)
        pools_equal(m, pools)
        act = rng.random()
        if act < 0.6:
            parents = [rng.choice([s, s, rng.randrange(S), rng.randrange(S), -1, S + 3]) for s in range(S)]
            out = ops.fork_pages(table, i32(parents), out=other)
            assert out is other
            m.fork(parents)
            held = [len(r) for r in m.rows]
            assert all(set(row[n:]) <= {-1} for row, n in zip(out.pages.tolist(), held))
            table, other = out, table
            m.same(table)
        if act > 0.4:
            assert ops.compact_pages(table, pools).tolist() == [m.compact()]
            m.same(table)
            pools_equal(m, pools)


def test_everything_shared_then_extended(ops):
    """Every sequence holds the same half-filled page: each gets its own copy,
    the old page is free afterwards."""
    m = Model(6, 4, 20, 8, 1)
    table, pools = ops.PageTable.empty(6, 4, 20, 8, DEV), [content((20, 4), 0)]
    for counts, parents in (([12, 0, 0, 0, 0, 0], [0] * 6), ([1] * 6, None)):
        assert ops.extend_pages(table, i32(counts), pools).tolist() == m.extend(counts)
        if parents:
            table = ops.fork_pages(table, i32(parents))
            m.fork(parents)
        m.same(table)
        pools_equal(m, pools)
    assert table.refs.tolist()[1] == 0 and table.refs.tolist()[0] == 6


def test_many_pools_and_layouts(ops):
    """More pools than one launch takes; token-major views, pages a part of a
    larger record, several types."""
    S, P, page = 3, 12, 4
    m = Model(S, 6, P, page, 0)
    table = ops.PageTable.empty(S, 6, P, page, DEV)
    ref, pools = [], []
    g = torch.Generator().manual_seed(0)
    for i in range(70):
        t = torch.randn((P, page, 2, 8), generator=g).to(torch.bfloat16 if i % 2 else torch.float32)
        if i % 3 == 0:
            t = t.transpose(1, 2)
        if i % 5 == 0:
            t = t[:, :1]
            t = t.contiguous() if i % 2 else t if t.stride(1) >= t.stride(0) else torch.cat([t, t], 1).contiguous()[:, :1]
        ref.append(t.clone(memory_format=torch.preserve_format))
        pools.append(torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=DEV).copy_(t))
    assert ops.extend_pages(table, i32([6, 0, 9]), pools).tolist() == m.extend([6, 0, 9])
    table = ops.fork_pages(table, i32([0, 0, 2]))
    m.fork([0, 0, 2])
    before = [list(r) for r in m.rows]
    assert ops.extend_pages(table, i32([1, 1, 1]), pools).tolist() == m.extend([1, 1, 1])
    m.same(table)
    moves = [(b[-1], r[len(b) - 1]) for b, r in zip(before, m.rows) if b and b[-1] != r[len(b) - 1]]
    assert len(moves) == 3 - 1
    for t, p in zip(ref, pools):
        for a, b in moves:
            t[b] = t[a]
        assert torch.equal(p.cpu(), t)


def test_captured_steps(ops):
    """fork, extend and compact in one graph, replayed from changing states;
    the tables' arrays are the graph's inputs and outputs."""
    S, M, P, page = 5, 8, 60, 4
    base = ops.PageTable.empty(S, M, P, page, DEV)
    work = ops.PageTable.empty(S, M, P, page, DEV)
    pools = [content((P, 8), 0)]
    parents, counts = i32([0] * S), i32([0] * S)
    run = lambda: (ops.extend_pages(ops.fork_pages(base, parents, out=work), counts, pools),
                   ops.compact_pages(work, pools))
    run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        granted, n_live = run()
    m = Model(S, M, P, page, 1)
    for p in range(P):
        pools[0][p] = p * 64
    for par, cnt in (([0, 1, 2, 3, 4], [5, 3, 0, 9, 1]), ([0, 0, 3, 3, -1], [1, 1, 2, 30, 4]),
                     ([4, 1, 1, 2, 2], [0, 7, 7, 1, 1])):
        parents.copy_(i32(par))
        counts.copy_(i32(cnt))
        graph.replay()
        m.fork(par)
        assert granted.tolist() == m.extend(cnt)
        assert n_live.tolist() == [m.compact()]
        m.same(work)
        pools_equal(m, pools)
        for a, b in ((base.pages, work.pages), (base.lens, work.lens), (base.refs, work.refs)):
            a.copy_(b)
        torch.cuda.synchronize()


def test_fork_refuses_shared_memory(ops):
    table, other = (ops.PageTable.empty(4, 8, 16, 4, DEV) for _ in range(2))
    for parents in (other.lens, other.refs[3:7], other.pages.view(-1)[9:13]):
        with pytest.raises(ValueError, match="share no memory"):
            ops.fork_pages(table, parents, out=other)
    with pytest.raises(ValueError, match="share no memory"):
        ops.fork_pages(table, i32([0, 1, 2, 3]), out=table)


def test_counts_may_be_the_lengths(ops):
    """Every sequence doubled; the same pool listed twice moves once."""
    m = Model(3, 40, 64, 4, n_pools=1)
    table = ops.PageTable.empty(3, 40, 64, 4, DEV)
    (pool,) = pools = [content((64, 8), 0)]
    for counts in ([5, 9, 2], None, None):
        given = m.lens[:] if counts is None else counts
        ops.extend_pages(table, table.lens if counts is None else i32(counts), [pool, pool])
        m.extend(given)
        m.same(table)
    m.fork([-1, 1, 1])
    table = ops.fork_pages(table, i32([-1, 1, 1]))
    ops.extend_pages(table, i32([1, 1, 1]), [pool, pool])
    m.extend([1, 1, 1])
    assert ops.compact_pages(table, [pool, pool]).item() == m.compact()
    m.same(table)
    pools_equal(m, pools)


def test_shared_last_page_takes_a_page_per_holder(ops):
    """Two beams on one half-filled page with one free page left: the first gets
    its copy, the second is refused and keeps the page for itself."""
    m = Model(2, 4, 2, 8, 1)
    table, pools = ops.PageTable.empty(2, 4, 2, 8, DEV), [content((2, 4), 0)]
    assert ops.extend_pages(table, i32([5, 0]), pools).tolist() == m.extend([5, 0])
    table = ops.fork_pages(table, i32([0, 0]))
    m.fork([0, 0])
    for counts, granted in (([1, 1], [True, False]), ([0, 1], [True, True]), ([2, 2], [True, True])):
        assert ops.extend_pages(table, i32(counts), pools).tolist() == m.extend(counts) == granted
        m.same(table)
        pools_equal(m, pools)
    assert table.refs.tolist() == [1, 1] and table.lens.tolist() == [8, 8]
