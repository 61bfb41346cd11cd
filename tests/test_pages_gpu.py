"""Pages of kept rows (pages_take, pages_free, pages_fork, pages_copy, pages_compact, pages_write) against a restatement on
lists. Everything here is whole numbers and moved bytes: the results are equal."""
import random

import pytest
import torch

import mako_h3 as mh

pytestmark = pytest.mark.gpu


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Model:
    """A table of lists, its counts and pools, as the calls document them."""

    def __init__(self, rng, streams, cols, pages, fill=0.5, share=0.2):
        self.rng, self.pages = rng, pages
        self.table = [[-1] * cols for _ in range(streams)]
        self.refs = [0] * pages
        order = rng.sample(range(pages), pages)
        for line in self.table:
            for e in range(cols):
                if rng.random() < fill:
                    shared = [p for p in range(pages) if self.refs[p]] if rng.random() < share else []
                    if shared:
                        line[e] = rng.choice(shared)
                    elif order:
                        line[e] = order.pop()
                    if line[e] >= 0:
                        self.refs[line[e]] += 1

    def on(self, dev):
        return ints(self.table, dev), ints(self.refs, dev)

    def take(self, first, last):
        none, cols = 0, len(self.table[0])
        free = [p for p, r in enumerate(self.refs) if r == 0]
        for line, a, b in zip(self.table, first, last):
            for e in range(min(max(a, 0), cols), min(b, cols)):
                if line[e] < 0:
                    if free:
                        line[e] = free.pop(0)
                        self.refs[line[e]] = 1
                    else:
                        none += 1
        return none

    def free(self, first, last):
        cols = len(self.table[0])
        for line, a, b in zip(self.table, first, last):
            for e in range(min(max(a, 0), cols), min(b, cols)):
                if 0 <= line[e] < self.pages:
                    self.refs[line[e]] -= 1
                line[e] = -1

    def fork(self, parents, rows, page_rows):
        """Returns (pages copied as (from, to), how many were missing)."""
        free = [p for p, r in enumerate(self.refs) if r == 0]
        fresh, moves, none, cols = [], [], 0, len(self.table[0])
        for s, (p, n) in enumerate(zip(parents, rows)):
            if p == s:
                fresh.append(list(self.table[s]))
                continue
            line = [-1] * cols
            if 0 <= p < len(self.table):
                full = max(n, 0) // page_rows
                line = [x if e < full else -1 for e, x in enumerate(self.table[p])]
                if max(n, 0) % page_rows and full < cols and self.table[p][full] >= 0:
                    if free:
                        line[full] = free.pop(0)
                        moves.append((self.table[p][full], line[full]))
                    else:
                        none += 1
            fresh.append(line)
        self.table = fresh
        self.count()
        return moves, none

    def count(self):
        self.refs = [0] * self.pages
        for line in self.table:
            for p in line:
                if p >= 0:
                    self.refs[p] += 1

    def compact(self):
        used = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(used)
        to = {p: p for p in used if p < n}
        holes = [p for p in range(n) if self.refs[p] == 0]
        moves = list(zip([p for p in used if p >= n], holes))
        to.update(moves)
        self.table = [[to.get(p, -1) for p in line] for line in self.table]
        old, self.refs = self.refs, [0] * self.pages
        for p in used:
            self.refs[to[p]] = old[p]
        return [to.get(p, -1) for p in range(self.pages)], n, moves

    def same(self, table, refs):
        assert table.tolist() == self.table
        assert refs.tolist() == self.refs


SHAPES = [
    # streams, entries, pages
    (1, 1, 1), (1, 1, 2), (3, 5, 16), (5, 40, 100), (2, 3, 7), (64, 17, 900), (7, 2025, 9001), (300, 3, 20000),
    (1100, 4, 3000),
]


@pytest.mark.parametrize("streams,cols,pages", SHAPES)
@pytest.mark.parametrize("seed", [0, 1])
def test_take_and_free(dev, streams, cols, pages, seed):
    rng = random.Random(f"{streams} {cols} {pages} {seed}")
    m = Model(rng, streams, cols, pages, fill=rng.choice([0.0, 0.5, 0.9]), share=0.0 if pages > 200 else 0.3)
    table, refs = m.on(dev)
    for _ in range(3):
        a, b = ([rng.randint(-1, cols + 1) for _ in range(streams)] for _ in range(2))
        missing = mh.pages_take(table, refs, ints(a, dev), ints(b, dev))
        assert int(missing) == m.take(a, b)
        m.same(table, refs)
        a, b = ([rng.randint(-1, cols + 1) for _ in range(streams)] for _ in range(2))
        mh.pages_free(table, refs, ints(a, dev), ints(b, dev))
        m.free(a, b)
        m.same(table, refs)


def test_take_where_no_page_of_the_pool_is(dev):
    """Entries outside the pool are no page, whichever side they lie on; those that find none end as -1."""
    table = ints([[1, 9, -7, 2**31 - 1, -2**31, 4]], dev)
    refs = ints([0, 1, 2, 0], dev)
    assert int(mh.pages_take(table, refs, ints([0], dev), ints([6], dev))) == 3
    assert table.tolist() == [[1, 0, 3, -1, -1, -1]] and refs.tolist() == [1, 1, 2, 1]


def test_take_at_the_int_range(dev):
    """Bounds at the ends of int32, more wants than a workgroup has threads, and a pool that runs out in their midst."""
    m = Model(random.Random(5), 3, 3001, 5000, fill=0.1, share=0.0)
    table, refs = m.on(dev)
    a, b = [-2 ** 31, 0, 2 ** 31 - 1], [2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31]
    assert int(mh.pages_take(table, refs, ints(a, dev), ints(b, dev))) == m.take(a, b) > 0
    m.same(table, refs)
    assert int((refs == 0).sum()) == 0
    mh.pages_free(table, refs, ints(a, dev), ints(b, dev))
    m.free(a, b)
    m.same(table, refs)


def pools_of(g, pages, dev):
    """Pools of several types and page sizes (one chunk, a part of one, several), one with gaps between its pages."""
    wide = torch.randint(0, 256, (pages, 5, 1024), generator=g, device=dev, dtype=torch.uint8)
    return [torch.randn((pages, 2, 16, 128), generator=g, device=dev).to(torch.bfloat16),
            wide[:, 1:3], torch.randn((pages, 4), generator=g, device=dev),
            torch.randint(-99, 99, (pages, 24000), generator=g, device=dev, dtype=torch.int32) if pages < 1000 else
            torch.zeros((pages, 8), dtype=torch.int64, device=dev)], wide


@pytest.mark.parametrize("streams,cols,pages", SHAPES)
@pytest.mark.parametrize("page_rows", [1, 16, 100])
def test_fork(dev, streams, cols, pages, page_rows):
    rng = random.Random(f"{streams} {cols} {pages} {page_rows}")
    m = Model(rng, streams, cols, pages, fill=0.6, share=0.0 if pages > 200 else 0.3)
    table, refs = m.on(dev)
    pools, wide = pools_of(torch.Generator(device=dev).manual_seed(streams), pages, dev)
    want, wide0 = [p.clone() for p in pools], wide.clone()
    parents = [rng.choice([s, rng.randrange(streams), rng.randrange(streams), -1, streams + 3]) for s in range(streams)]
    rows = [rng.choice([rng.randint(0, cols * page_rows), -5, cols * page_rows + 9, 0]) for _ in range(streams)]
    old = table.clone()
    new, missing = mh.pages_fork(pools, table, refs, ints(parents, dev), ints(rows, dev), page_rows)
    moves, none = m.fork(parents, rows, page_rows)
    assert int(missing) == none and torch.equal(table, old)
    m.same(new, refs)
    for src, dst in moves:
        for p in want:
            p[dst] = p[src]
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    assert torch.equal(wide[:, 0], wide0[:, 0]) and torch.equal(wide[:, 3:], wide0[:, 3:])


def test_fork_swaps_and_chains(dev):
    """All rows go by the old table: two that swap, a chain, and several from one whose own row goes on elsewhere."""
    m = Model(random.Random(1), 6, 4, 64, fill=1.0, share=0.0)
    table, refs = m.on(dev)
    pool = torch.arange(64 * 64, device=dev, dtype=torch.int32).view(64, 64).clone()
    want = pool.clone()
    parents, rows = [1, 0, 1, 2, 2, 2], [50, 64, 16, 1, 33, 48]
    new, _ = mh.pages_fork(pool, table, refs, ints(parents, dev), ints(rows, dev), 16)
    moves, _ = m.fork(parents, rows, 16)
    for src, dst in moves:
        want[dst] = want[src]
    m.same(new, refs)
    assert torch.equal(pool, want)


@pytest.mark.parametrize("pages,n", [(1, 1), (2, 1), (30, 9), (500, 200), (40, 60), (20000, 16384)])
def test_copy(dev, pages, n):
    rng = random.Random(f"{pages} {n}")
    pools, wide = pools_of(torch.Generator(device=dev).manual_seed(pages), pages, dev)
    want, wide0 = [p.clone() for p in pools], wide.clone()
    src = [rng.randint(-2, pages + 1) for _ in range(n)]
    dst = [rng.randint(-2, pages + 1) for _ in range(n)]
    mh.pages_copy(pools, ints(src, dev), ints(dst, dev))
    from_, seen, a, b = set(src), set(), [], []
    for s, d in zip(src, dst):
        if 0 <= s < pages and 0 <= d < pages and d not in from_ and d not in seen:
            a.append(s)
            b.append(d)
        seen.add(d)
    a, b = torch.tensor(a, dtype=torch.long, device=dev), torch.tensor(b, dtype=torch.long, device=dev)
    for p in want:
        p[b] = p[a]
    assert all(torch.equal(x, y) for x, y in zip(pools, want))
    assert torch.equal(wide[:, 0], wide0[:, 0]) and torch.equal(wide[:, 3:], wide0[:, 3:])


@pytest.mark.parametrize("streams,cols,pages", SHAPES + [(20, 1000, 30001)])
@pytest.mark.parametrize("fill", [0.0, 0.3, 1.0])
def test_compact(dev, streams, cols, pages, fill):
    rng = random.Random(f"{streams} {cols} {pages} {fill}")
    m = Model(rng, streams, cols, pages, fill=fill, share=0.0 if pages > 200 else 0.3)
    table, refs = m.on(dev)
    pools, wide = pools_of(torch.Generator(device=dev).manual_seed(streams), pages, dev)
    want, wide0 = [p.clone() for p in pools], wide.clone()
    got, used = mh.pages_compact(pools, table, refs)
    to, n, moves = m.compact()
    m.same(table, refs)
    assert got.tolist() == to and int(used) == n
    if moves:
        a, b = (torch.tensor(x, device=dev) for x in zip(*moves))
        for p in want:
            p[b] = p[a]
    assert all(torch.equal(x, y) for x, y in zip(pools, want))
    assert torch.equal(wide[:, 0], wide0[:, 0]) and torch.equal(wide[:, 3:], wide0[:, 3:])
    again, _ = mh.pages_compact(pools, table, refs)    # nothing is left to move
    m.same(table, refs)
    assert again.tolist() == list(range(n)) + [-1] * (pages - n)


def test_no_pages_of_the_pool(dev):
    """Entries outside the pool are no pages: nothing is counted, moved or written for them."""
    bad = [[0, 7, -9, 8], [2 ** 31 - 1, 3, -2 ** 31, 100]]
    refs0 = [1, 0, 0, 1, 0, 0, 0, 1]
    pool = torch.arange(8 * 4, device=dev, dtype=torch.int32).view(8, 4).clone()
    table, refs = ints(bad, dev), ints(refs0, dev)
    new, missing = mh.pages_fork(pool, table, refs, ints([1, 1], dev), ints([40, 0], dev), 10)
    assert new.tolist() == [[-1, 3, -1, -1], bad[1]] and refs.tolist() == [0, 0, 0, 2, 0, 0, 0, 0] and int(missing) == 0
    table, refs = ints(bad, dev), ints(refs0, dev)
    to, used = mh.pages_compact(pool, table, refs)
    # In use: 0, 3 and 7, so three; past the end 3 and 7, in this order into the free 1 and 2.
    assert table.tolist() == [[0, 2, -1, -1], [-1, 1, -1, -1]] and refs.tolist() == [1, 1, 1, 0, 0, 0, 0, 0]
    assert to.tolist() == [0, -1, -1, 1, -1, -1, -1, 2] and int(used) == 3
    assert pool[:3, 0].tolist() == [0, 12, 28]
    table, refs = ints(bad, dev), ints(refs0, dev)
    mh.pages_free(table, refs, ints([1, 0], dev), ints([4, 1], dev))
    assert table.tolist() == [[0, -1, -1, -1], [-1, 3, -2 ** 31, 100]] and refs.tolist() == [1, 0, 0, 1, 0, 0, 0, 0]


@pytest.mark.parametrize("layout", ["heads", "rows"])
@pytest.mark.parametrize("page_layout", ["heads", "rows"])
@pytest.mark.parametrize("heads,page_rows,streams,new", [(1, 16, 1, 1), (2, 64, 3, 70), (8, 32, 20, 3), (7, 5, 4, 33)])
@pytest.mark.parametrize("accepted", [False, True])
def test_write(dev, heads, page_rows, streams, new, layout, page_layout, accepted):
    """Rows into one layer's slice of pages that hold two; rows before the first stream and behind the last, entries without
    a page, places before the first and past the table, and sources that do not exist, are passed over."""
    rng = random.Random(f"{heads} {page_rows} {streams} {new} {layout} {page_layout}")
    g = torch.Generator(device=dev).manual_seed(heads)
    cols, pages = 6, streams * 6 + 3
    m = Model(rng, streams, cols, pages, fill=0.8, share=0.0)
    m.table[0][-1] = pages + 5
    counts = [rng.choice([0, new, rng.randint(0, new)]) for _ in range(streams)]
    off = [2]
    for c in counts:
        off.append(off[-1] + c)
    n = off[-1] + 3
    starts = [rng.randint(-3, cols * page_rows + 2) for _ in range(streams)]
    n_rows = n + 5 if accepted else n
    rows = [rng.randint(-2, n_rows + 2) for _ in range(n)] if accepted else None
    k, v = (torch.randn((heads, n_rows, 128), generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    shape = (pages, 2, 2, heads, page_rows, 128) if page_layout == "heads" else (pages, 2, 2, page_rows, heads * 128)
    pool = torch.randn(shape, generator=g, device=dev).to(torch.bfloat16)
    want = pool.clone()
    for s, line in enumerate(m.table):
        for j in range(off[s], off[s + 1]):
            place, row = starts[s] + j - off[s], rows[j] if accepted else j
            if not (0 <= row < n_rows and 0 <= place < cols * page_rows and 0 <= line[place // page_rows] < pages):
                continue
            for i, x in enumerate((k, v)):
                at = want[line[place // page_rows], 1, i]
                if page_layout == "heads":
                    at[:, place % page_rows] = x[:, row]
                else:
                    at[place % page_rows] = x[:, row].reshape(-1)
    lay = (lambda x: x) if layout == "heads" else lambda x: x.transpose(0, 1).reshape(n_rows, -1)
    mh.pages_write(lay(k), lay(v), pool[:, 1, 0], pool[:, 1, 1], ints(m.table, dev), ints(starts, dev), ints(off, dev),
                   rows=ints(rows, dev) if accepted else None, layout=layout, page_layout=page_layout)
    assert torch.equal(pool, want)


def test_strided_table(dev):
    """A table that is a slice of a wider one: the other columns stay as they are."""
    m = Model(random.Random(2), 5, 7, 60, fill=0.5)
    wide = torch.full((5, 12), 77, dtype=torch.int32, device=dev)
    table, refs = wide[:, 3:10], ints(m.refs, dev)
    table.copy_(ints(m.table, dev))
    a, b = [0, 1, 2, 0, 6], [7, 3, 2, 1, 7]
    mh.pages_take(table, refs, ints(a, dev), ints(b, dev))
    m.take(a, b)
    m.same(table, refs)
    pool = torch.randn((60, 8), device=dev)
    new, _ = mh.pages_fork(pool, table, refs, ints([0, 0, 0, 1, 9], dev), ints([7, 5, 3, 2, 1], dev), 1)
    m.fork([0, 0, 0, 1, 9], [7, 5, 3, 2, 1], 1)
    m.same(new, refs)
    table.copy_(new)
    mh.pages_compact(pool, table, refs)
    m.compact()
    m.same(table, refs)
    assert bool((wide[:, :3] == 77).all()) and bool((wide[:, 10:] == 77).all())


def test_captured(dev):
    """A step's calls in a graph, replayed: each replay goes on from where the last one left the state."""
    m = Model(random.Random(3), 4, 50, 250, fill=0.2, share=0.0)
    table, refs = m.on(dev)
    pool = torch.randn((250, 2, 2, 16, 128), device=dev).to(torch.bfloat16)
    want = pool.clone()
    first, last = [0, 3, 10, 40], [20, 9, 30, 50]
    parents, rows = [0, 0, 2, 3], [0, 100, 0, 0]
    a, b, p, r = ints(first, dev), ints(last, dev), ints(parents, dev), ints(rows, dev)
    src, dst = ints([1, 2, 3], dev), ints([7, 8, 9], dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        mh.pages_take(table, refs, a, b)
        new, _ = mh.pages_fork(pool, table, refs, p, r, 16)
        table.copy_(new)
        mh.pages_copy(pool, src, dst)
        mh.pages_free(table, refs, b, a)
        mh.pages_free(table, refs, a, p)
        mh.pages_compact(pool, table, refs)

    def model():
        m.take(first, last)
        for s, d in m.fork(parents, rows, 16)[0] + [(1, 7), (2, 8), (3, 9)]:
            want[d] = want[s]
        m.free(last, first)
        m.free(first, parents)
        for s, d in m.compact()[2]:
            want[d] = want[s]

    with torch.cuda.stream(side):
        step()
        model()
    torch.cuda.current_stream().wait_stream(side)
    m.same(table, refs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        graph.replay()
        model()
        torch.cuda.synchronize()
        m.same(table, refs)
        assert torch.equal(pool, want)


def test_nothing_to_do(dev):
    """Empty lists and spans, streams that go on from themselves, pages that lie together: everything stays as it is."""
    g = torch.Generator(device=dev).manual_seed(9)
    pool = torch.randn((6, 2, 16, 128), generator=g, device=dev).to(torch.bfloat16)
    pools, want = [pool, pool.clone()], pool.clone()
    table, refs = ints([[0, 2, -1], [1, -1, -1]], dev), ints([1, 1, 1, 0, 0, 0], dev)
    table0, refs0 = table.clone(), refs.clone()
    assert int(mh.pages_take(table, refs, ints([3, 2], dev), ints([1, 2], dev))) == 0
    mh.pages_free(table, refs, ints([2, 9], dev), ints([2, 3], dev))
    mh.pages_copy(pools, ints([], dev), ints([], dev))
    off = ints([0, 0, 0], dev)
    rows = torch.zeros((2, 4, 128), dtype=torch.bfloat16, device=dev)
    mh.pages_write(rows, rows, *pools, table, ints([0, 0], dev), off)
    mh.pages_write(rows, rows, *pools, table, ints([0, 0], dev), off, rows=ints([], dev))
    mh.pages_write(rows[:, :0], rows[:, :0], *pools, table, ints([0, 0], dev), off)
    fresh, missing = mh.pages_fork(pools, table, refs, ints([0, 1], dev), ints([1000, -4], dev), 16)
    moved, used = mh.pages_compact(pools, table, refs)
    assert int(missing) == 0 and int(used) == 3 and moved.tolist() == [0, 1, 2, -1, -1, -1]
    for t in (table, fresh):
        assert torch.equal(t, table0)
    assert torch.equal(refs, refs0) and all(torch.equal(p, want) for p in pools)
