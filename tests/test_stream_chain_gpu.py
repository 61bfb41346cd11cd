"""Streams that generate rows as a program runs them: pages taken and written, drafted trees attended over them, accepted
rows kept, candidates forked, what a window has left behind freed, the rest compacted. Beside it each stream's rows are kept
in one piece, as lists: every step's attention is checked against float64 of those, and its pages hold them to the bit."""
import math
import random

import pytest
import torch

import mako_h3 as mh
from test_attn_dense_gpu import check

pytestmark = pytest.mark.gpu

PAGE, HEADS, KV, SINKS, COLS, PAGES = 16, 8, 2, 20, 64, 300


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Program:
    def __init__(self, dev, streams, window, seed):
        self.dev, self.window, self.rng = dev, window, random.Random(seed)
        self.g = torch.Generator(device=dev).manual_seed(seed)
        self.table = torch.full((streams, COLS), -1, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(PAGES, dtype=torch.int32, device=dev)
        self.pool = torch.full((PAGES, 2, KV, PAGE, 128), float("nan"), dtype=torch.bfloat16, device=dev)
        self.k, self.v = ([torch.empty((KV, 0, 128), dtype=torch.bfloat16, device=dev)] * streams for _ in range(2))

    def lengths(self):
        return [x.shape[1] for x in self.k]

    def rows(self, heads, n):
        return torch.randn((heads, n, 128), generator=self.g, device=self.dev).to(torch.bfloat16)

    def pages(self):
        return self.pool[:, 0], self.pool[:, 1]

    def append(self, k, v, counts, rows=None):
        """k, v: rows of all streams; counts: how many each takes, of them those that `rows` says."""
        had = self.lengths()
        first = [-(-n // PAGE) for n in had]
        last = [-(-(n + c) // PAGE) for n, c in zip(had, counts)]
        assert int(mh.pages_take(self.table, self.refs, ints(first, self.dev), ints(last, self.dev))) == 0
        off = [sum(counts[:i]) for i in range(len(counts) + 1)]
        mh.pages_write(k, v, *self.pages(), self.table, ints(had, self.dev), ints(off, self.dev),
                       rows=None if rows is None else ints(rows, self.dev))
        at = list(range(k.shape[1])) if rows is None else rows
        for s in range(len(counts)):
            mine = at[off[s]:off[s + 1]]
            self.k[s], self.v[s] = (torch.cat([a[s], x[:, mine]], 1) for a, x in ((self.k, k), (self.v, v)))

    def step(self, new, tree):
        """One call for `new` rows of each stream; checked, and its k, v and parents."""
        n = len(self.k)
        q, k, v = self.rows(HEADS, n * new), self.rows(KV, n * new), self.rows(KV, n * new)
        parents = [self.rng.randint(-1, i - 1) if i else -1 for _ in range(n) for i in range(new)] if tree else None
        kept = self.lengths()
        got = mh.flash_attn_pages_128(q, k, v, *self.pages(), self.table, ints(kept, self.dev),
                                      ints([new * s for s in range(n + 1)], self.dev), window=self.window,
                                      parents=ints(parents, self.dev) if tree else None,
                                      sinks=ints([SINKS] * n, self.dev))
        want, mag = torch.zeros(q.shape, dtype=torch.float64, device=self.dev), torch.zeros(q.shape, dtype=torch.float64,
                                                                                          device=self.dev)
        for s in range(n):
            seen = torch.zeros((new, kept[s] + new), dtype=torch.bool)
            for i in range(new):
                line = [i]
                while (up := parents[s * new + line[-1]] if tree else line[-1] - 1) >= 0:
                    line.append(up)
                place = kept[s] + len(line) - 1
                places = list(range(kept[s])) + [-1] * new
                for back, j in enumerate(line):
                    places[kept[s] + j] = place - back
                seen[i] = torch.tensor([p >= 0 and (not self.window or p > place - self.window or p < SINKS)
                                        for p in places])
            mine = slice(s * new, s * new + new)
            for h in range(HEADS):
                kd = torch.cat([self.k[s][h // 4], k[h // 4, mine]]).double()
                vd = torch.cat([self.v[s][h // 4], v[h // 4, mine]]).double()
                x = q[h, mine].double() @ kd.T.contiguous() / math.sqrt(128)
                p = torch.softmax(torch.where(seen.to(self.dev), x, -math.inf), -1)
                want[h, mine], mag[h, mine] = p @ vd, p @ vd.abs()
        check(got, want, mag)
        return k, v, parents

    def free_behind(self):
        """What the window of any next row no longer reaches, but the first rows."""
        first = [-(-SINKS // PAGE)] * len(self.k)
        last = [max(0, n - self.window + 1) // PAGE for n in self.lengths()]
        mh.pages_free(self.table, self.refs, ints(first, self.dev), ints(last, self.dev))
        return first, last

    def fork(self, parents):
        rows = [self.lengths()[p] if 0 <= p < len(parents) else 0 for p in parents]
        self.table, missing = mh.pages_fork(self.pool, self.table, self.refs, ints(parents, self.dev),
                                            ints(rows, self.dev), PAGE)
        assert int(missing) == 0
        empty = self.rows(KV, 0)
        self.k, self.v = ([a[p] if 0 <= p < len(parents) else empty for p in parents] for a in (self.k, self.v))

    def check_pages(self):
        """Every kept row in a page is the stream's; the counts are the table's."""
        table, refs = self.table.tolist(), self.refs.tolist()
        counts = [0] * PAGES
        for s, n in enumerate(self.lengths()):
            for e, page in enumerate(table[s]):
                if page < 0:
                    continue
                counts[page] += 1
                rows = slice(e * PAGE, min(n, e * PAGE + PAGE))
                here = rows.stop - rows.start
                if here > 0:
                    assert torch.equal(self.pool[page, 0, :, :here], self.k[s][:, rows])
                    assert torch.equal(self.pool[page, 1, :, :here], self.v[s][:, rows])
        assert counts == refs


@pytest.mark.parametrize("window", [0, 50])
def test_streams(dev, window):
    p = Program(dev, 4, window, 11 + window)
    text = [70, 33, 16, 1]
    k, v = p.rows(KV, sum(text)), p.rows(KV, sum(text))
    p.append(k, v, text)
    p.check_pages()
    for turn in range(8):
        # Drafts: a path of each stream's tree is accepted.
        k, v, parents = p.step(6, True)
        rows, counts = [], []
        for s in range(4):
            path, at = [], p.rng.randrange(6)
            while at >= 0:
                path.append(s * 6 + at)
                at = parents[s * 6 + at]
            rows += path[::-1]
            counts.append(len(path))
        p.append(k, v, counts, rows)
        # A few rows one after another, all kept; then one alone.
        k, v, _ = p.step(9, False)
        p.append(k, v, [9] * 4)
        k, v, _ = p.step(1, False)
        p.append(k, v, [1] * 4)
        if window:
            p.free_behind()
        if turn % 2:
            p.fork([1, 1, 3, 0] if turn % 4 == 1 else [0, 2, 2, 7])
            p.append(*(p.rows(KV, 40) for _ in range(2)), [0, 11, 24, 5])
        if turn % 3 == 2:
            before = int((p.refs > 0).sum())
            _, used = mh.pages_compact(p.pool, p.table, p.refs)
            assert int(used) == before and bool((p.refs[:before] > 0).all())
        p.check_pages()


def test_a_window_is_the_same_over_pages_and_in_one_piece(dev):
    """A stream's last rows through flash_attn_pages_128, and through flash_attn_128 with attn_window_ranges over all of its
    rows: within the sum of their bounds."""
    p = Program(dev, 1, 60, 5)
    p.append(p.rows(KV, 300), p.rows(KV, 300), [300])
    q, k, v = p.rows(HEADS, 25), p.rows(KV, 25), p.rows(KV, 25)
    a = mh.flash_attn_pages_128(q, k, v, *p.pages(), p.table, ints([300], dev), ints([0, 25], dev), window=60,
                                sinks=ints([SINKS], dev))
    off_q, off_k = ints([0, 25], dev), ints([0, 325], dev)
    ranges, sinks = mh.attn_window_ranges(off_q, off_k, 25, 325, 60, sinks=ints([SINKS], dev))
    ka, va = torch.cat([p.k[0], k], 1), torch.cat([p.v[0], v], 1)
    b = mh.flash_attn_128(q, ka, va, ranges=ranges, sinks=sinks)
    # Each is within 2^-8 of itself and 2^-8 + 2^-11 of the sum of p |v|, at most the largest |v|, of the exact value.
    bound = 2 ** -8 * (a.float().abs() + b.float().abs()) + 2 * (2 ** -8 + 2 ** -11) * float(va.float().abs().max())
    assert bool(((a.float() - b.float()).abs() <= bound).all())
    # Far closer on average: the probabilities' roundings are independent.
    assert float((a.float() - b.float()).abs().mean()) < 2 ** -8 * float(b.float().abs().mean()) * 2


def test_a_step_captured(dev):
    """A step of single rows in a graph (places, attention, the rows into their pages, what the window has left behind freed,
    lengths counted on), replayed: every replay gives the eager bits."""
    state = []
    for _ in range(2):
        p = Program(dev, 3, 40, 8)
        p.append(p.rows(KV, 90), p.rows(KV, 90), [50, 10, 30])
        state.append(p)
    x = [[torch.randn((h, 3, 128), generator=state[0].g, device=dev).to(torch.bfloat16) for h in (HEADS, KV, KV)]
         for _ in range(5)]
    off, sinks, zero = ints([0, 1, 2, 3], dev), ints([SINKS] * 3, dev), ints([-(-SINKS // PAGE)] * 3, dev)

    def step(p, q, k, v, lengths):
        first = ((lengths + PAGE - 1) // PAGE).int()
        mh.pages_take(p.table, p.refs, first, ((lengths + PAGE) // PAGE).int())
        out = mh.flash_attn_pages_128(q, k, v, *p.pages(), p.table, lengths, off, window=40, sinks=sinks)
        mh.pages_write(k, v, *p.pages(), p.table, lengths, off)
        lengths += 1
        mh.pages_free(p.table, p.refs, zero, ((lengths - 39).clamp(min=0) // PAGE).int())
        return out

    eager, replayed = state
    lengths = [ints(eager.lengths(), dev) for _ in range(2)]
    static = [t.clone() for t in x[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    keep = [t.clone() for t in (replayed.table, replayed.refs, lengths[1])]
    with torch.cuda.stream(side):
        step(replayed, *static, lengths[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(replayed, *static, lengths[1])
    for t, was in zip((replayed.table, replayed.refs, lengths[1]), keep):
        t.copy_(was)
    for q, k, v in x:
        for t, new in zip(static, (q, k, v)):
            t.copy_(new)
        graph.replay()
        want = step(eager, q, k, v, lengths[0])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(replayed.table, eager.table) and torch.equal(replayed.refs, eager.refs)
