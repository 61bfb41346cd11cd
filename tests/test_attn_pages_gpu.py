"""flash_attn_pages_128 against a float64 restatement, key by key; the bounds are those of test_attn_dense_gpu."""
import math
import random

import pytest
import torch

import mako_h3 as mh
from test_attn_dense_gpu import check, make

pytestmark = pytest.mark.gpu

NAN = float("nan")


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Streams:
    """Streams of some kept and new rows over shuffled pages, what the pools hold outside of them NaN."""

    def __init__(self, seed, dev, heads, kv_heads, page, kept, new, tree=False, page_layout="heads", sinks=None):
        rng, g = random.Random(seed), torch.Generator(device=dev).manual_seed(seed)
        self.dev, self.page, self.kept, self.new, self.page_layout = dev, page, kept, new, page_layout
        counts = [-(-n // page) for n in kept]
        self.pages = sum(counts) + 3
        numbers = rng.sample(range(self.pages), sum(counts))
        cols = max(counts) + 2
        self.lines = [[-1] * cols for _ in kept]
        for line, n in zip(self.lines, counts):
            for e in range(n):
                line[e] = numbers.pop()
        self.q_off = [2]
        for n in new:
            self.q_off.append(self.q_off[-1] + n)
        rows = self.q_off[-1] + 3
        self.q, self.k, self.v = make(g, heads, rows, dev), make(g, kv_heads, rows, dev), make(g, kv_heads, rows, dev)
        shape = (self.pages, kv_heads, page, 128) if page_layout == "heads" else (self.pages, page, kv_heads * 128)
        self.k_pages, self.v_pages = (torch.full(shape, NAN, device=dev, dtype=torch.bfloat16) for _ in range(2))
        for s, n in enumerate(kept):
            for pool in (self.k_pages, self.v_pages):
                self.place(pool, s, make(g, kv_heads, n, dev))
        self.parents = None
        if tree:
            self.parents = [0] * rows
            for a, n in zip(self.q_off, new):
                for i in range(n):
                    self.parents[a + i] = rng.choice([-1, i - 1, rng.randint(-1, max(i - 1, -1)), i, i + 5, -9]) if i else \
                        rng.choice([-1, 0, 3])
        self.sinks = sinks

    def place(self, pool, s, x):
        for at in range(0, x.shape[1], self.page):
            part = x[:, at:at + self.page]
            page = pool[self.lines[s][at // self.page]]
            if self.page_layout == "heads":
                page[:, :part.shape[1]] = part
            else:
                page[:part.shape[1]] = part.transpose(0, 1).reshape(part.shape[1], -1)

    def kept_rows(self, pool, s):
        """(rows [heads][kept][128], which of them have a page)."""
        heads = self.k.shape[0]
        rows = torch.zeros((heads, self.kept[s], 128), dtype=torch.bfloat16, device=self.dev)
        there = torch.zeros(self.kept[s], dtype=torch.bool, device=self.dev)
        for at in range(0, self.kept[s], self.page):
            page, n = self.lines[s][at // self.page], min(self.page, self.kept[s] - at)
            if 0 <= page < self.pages:
                x = pool[page, :, :n] if self.page_layout == "heads" else pool[page, :n].view(n, heads, 128).transpose(0, 1)
                rows[:, at:at + n], there[at:at + n] = x, True
        return rows, there

    def line(self, s, i):
        """The new rows that row i attends, from itself to its first ancestor."""
        if self.parents is None:
            return list(range(i, -1, -1))
        rows = [i]
        while 0 <= self.parents[self.q_off[s] + rows[-1]] < rows[-1]:
            rows.append(self.parents[self.q_off[s] + rows[-1]])
        return rows

    def seen(self, s, window):
        """bool [new][kept + new], without regard to missing pages."""
        kept, new = self.kept[s], self.new[s]
        seen = torch.zeros((new, kept + new), dtype=torch.bool)
        sinks = self.sinks[s] if self.sinks else 0
        at = torch.arange(kept)
        for i in range(new):
            line = self.line(s, i)
            place = kept + len(line) - 1
            seen[i, :kept] = (at < sinks) | (at > place - window) if window else True
            for back, j in enumerate(line):
                seen[i, kept + j] = not window or back < window or place - back < sinks
        return seen.to(self.dev)

    def run(self, window=0, **kw):
        if self.parents is not None:
            kw["parents"] = ints(self.parents, self.dev)
        if self.sinks:
            kw["sinks"] = ints(self.sinks, self.dev)
        return mh.flash_attn_pages_128(self.q, self.k, self.v, self.k_pages, self.v_pages, ints(self.lines, self.dev),
                                       ints(self.kept, self.dev), ints(self.q_off, self.dev), window=window,
                                       page_layout=self.page_layout, **kw)

    def want(self, window=0, scale=None, cap=0.0):
        """(out, sum of p |v|) in float64; rows of no stream zero."""
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=self.dev)
        mag = torch.zeros_like(out)
        share = self.q.shape[0] // self.k.shape[0]
        for s in range(len(self.kept)):
            mine = slice(self.q_off[s], self.q_off[s + 1])
            ks, there = self.kept_rows(self.k_pages, s)
            vs, _ = self.kept_rows(self.v_pages, s)
            seen = self.seen(s, window)
            seen[:, :self.kept[s]] &= there
            for h in range(self.q.shape[0]):
                kd = torch.cat([ks[h // share], self.k[h // share, mine]]).double()
                vd = torch.cat([vs[h // share], self.v[h // share, mine]]).double()
                x = self.q[h, mine].double() @ kd.T.contiguous() * (scale or 1 / math.sqrt(128))
                if cap:
                    x = cap * torch.tanh(x / cap)
                p = torch.softmax(torch.where(seen, x, -math.inf), -1)
                p = torch.where(seen, p, 0.0)
                clean = torch.where(torch.isfinite(vd).all(1, keepdim=True), vd, 0.0)
                out[h, mine], mag[h, mine] = p @ clean, p @ clean.abs()
        return out, mag


CASES = [
    # heads, key heads, page, kept, new
    (1, 1, 16, [0], [1]), (1, 1, 16, [1], [1]), (2, 1, 16, [64], [1]), (5, 1, 32, [65], [3]), (40, 8, 64, [777, 0, 15], 1),
    (3, 3, 16, [129, 64, 1000], [0, 5, 64]), (4, 2, 48, [500, 0, 0, 33], [65, 130, 1, 0]), (56, 56, 64, [300], [8]),
    (7, 1, 112, [2000, 1999], [33, 2]), (8, 8, 64, [4096], [100]), (2, 2, 16, [10] * 70, 1), (6, 3, 256, [3000, 77], 7),
    (16, 2, 1024, [5000, 1024, 1023], 4), (2, 1, 16, [20000], [200]), (12, 2, 32, [50] * 130 + [9000], 2),
    (64, 1, 16, [100, 3000], [1, 70]), (4, 4, 64, [0, 0], [300, 1]),
    # Runs of more tiles than either kernel looks up at a time.
    (2, 2, 16, [40], [1100]), (64, 64, 16, [20000], [70]), (64, 64, 32, [20000, 5], 1), (48, 48, 128, [9000, 9001], [33, 100]),
]


def streams(i, dev, **kw):
    heads, kv_heads, page, kept, new = CASES[i]
    new = [new] * len(kept) if isinstance(new, int) else new
    return Streams(i, dev, heads, kv_heads, page, kept, new, **kw)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("cap,page_layout", [(0.0, "heads"), (5.0, "rows")])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_all_kept_rows(dev, i, tree, cap, page_layout):
    st = streams(i, dev, tree=tree, page_layout=page_layout)
    out = torch.full_like(st.q, 7.0)
    assert st.run(cap=cap, out=out) is out
    want, mag = st.want(cap=cap)
    assert bool((out[:, :2] == 7).all()) and bool((out[:, st.q_off[-1]:] == 7).all())   # rows of no stream
    out[:, :2], out[:, st.q_off[-1]:] = 0, 0
    check(out, want, mag)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("window", [1, 2, 17, 64, 500, 4294967295])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_window_and_first_rows(dev, i, window, tree):
    """Windows from the row alone to all there is, with none, a few and many first rows, which may be new ones."""
    kept = CASES[i][3]
    st = streams(i, dev, tree=tree, sinks=[(0, 1, 5, 70, 400, 2 ** 31 - 1, -3)[(s + window + i) % 7]
                                           for s in range(len(kept))])
    out = st.run(window=window, scale=0.2)
    check(out, *st.want(window=window, scale=0.2))


@pytest.mark.parametrize("i", [4, 5, 6, 8, 13, 14])
def test_missing_pages(dev, i):
    """Entries that are no page (those that a window has left behind, or any): their rows are not attended."""
    st = streams(i, dev, tree=i % 2 == 0)
    rng = random.Random(i)
    for line in st.lines:
        for e in range(len(line)):
            if rng.random() < 0.4:
                line[e] = rng.choice([-1, st.pages, -2 ** 31, 2 ** 31 - 1])
    check(st.run(), *st.want())
    check(st.run(window=90), *st.want(window=90))


@pytest.mark.parametrize("i", [5, 6, 8])
def test_unattended_rows_leave_no_trace(dev, i):
    """NaN in kept and new rows that a row does not attend, behind the window or off its line, change none of its bits."""
    st = streams(i, dev, tree=True, sinks=[20] * len(CASES[i][3]))
    clean = st.run(window=60)
    for s, (kept, new) in enumerate(zip(st.kept, st.new)):
        for back in (61 + new, 200, kept - 21):     # behind every row's window, and no first row
            at = kept - back
            if 20 <= at < kept - 60 - new:
                for pool in (st.k_pages, st.v_pages):
                    pool[st.lines[s][at // st.page], :, at % st.page] = NAN
    assert torch.equal(st.run(window=60), clean)
    for s, new in enumerate(st.new):
        j = new // 2
        if new < 2:
            continue
        k, v = st.k.clone(), st.v.clone()
        st.k[:, st.q_off[s] + j], st.v[:, st.q_off[s] + j] = NAN, NAN
        got = st.run(window=60)
        st.k, st.v = k, v
        off = [st.q_off[t] + r for t in range(len(st.new)) for r in range(st.new[t]) if t != s or j not in st.line(s, r)]
        assert torch.equal(got[:, off], clean[:, off])
        on = [st.q_off[s] + r for r in range(new) if j in st.line(s, r)[:60]]
        assert bool(torch.isnan(got[:, on]).all())


def test_a_row_is_its_own_stream(dev):
    """A stream's rows do not depend on the streams beside it but for the order of their sums: within twice the bound of a
    rounding. With the same cuts they are the same bits: streams of no rows between them move none."""
    st = streams(14, dev)
    want, mag = st.want()
    one = mh.flash_attn_pages_128(st.q[:, -5:-3], st.k[:, -5:-3], st.v[:, -5:-3], st.k_pages, st.v_pages,
                                  ints(st.lines[-1:], dev), ints(st.kept[-1:], dev), ints([0, 2], dev))
    check(one, want[:, -5:-3], mag[:, -5:-3])
    wide = mh.flash_attn_pages_128(st.q[:, -5:-3], st.k[:, -5:-3], st.v[:, -5:-3], st.k_pages, st.v_pages,
                                   ints(st.lines[:100] + st.lines[-1:], dev), ints(st.kept[:100] + st.kept[-1:], dev),
                                   ints([0] * 101 + [2], dev))
    assert torch.equal(one, wide)


@pytest.mark.parametrize("i,gap", [(6, 32), (6, 8), (8, 8), (4, 24)])
def test_layouts_strides_and_slices(dev, i, gap):
    """Heads side by side in wider rows (by 8 elements, and by 64), one layer's slices of pages that hold several, a table in
    a wider one; with streams of many rows and of few."""
    st = streams(i, dev, tree=True)
    want = st.run()
    rows = st.q.shape[1]
    wide = [torch.full((rows, x.shape[0] * 128 + 2 * gap), NAN, dtype=torch.bfloat16, device=dev) for x in (st.q, st.k, st.v)]
    q, k, v = (w[:, gap:-gap] for w in wide)
    for t, x in zip((q, k, v), (st.q, st.k, st.v)):
        t.copy_(x.transpose(0, 1).reshape(rows, -1))
    heads, page = st.k_pages.shape[1:3]
    pool = torch.full((st.pages, 3, 2, page, heads, 128 + gap), NAN, dtype=torch.bfloat16, device=dev)
    k_pages, v_pages = (pool[:, 1, x, :, :, :128].transpose(2, 1) for x in range(2))     # rows of heads, each wider
    k_pages.copy_(st.k_pages)
    v_pages.copy_(st.v_pages)
    table = torch.full((len(st.lines), len(st.lines[0]) + 9), 1, dtype=torch.int32, device=dev)
    table[:, 4:-5] = ints(st.lines, dev)
    out = torch.zeros((rows, st.q.shape[0] * 128), dtype=torch.bfloat16, device=dev)
    mh.flash_attn_pages_128(q, k, v, k_pages, v_pages, table[:, 4:-5], ints(st.kept, dev), ints(st.q_off, dev),
                            parents=ints(st.parents, dev), layout="rows", out=out)
    assert torch.equal(out.view(rows, -1, 128).transpose(0, 1), want)


def test_stream_and_graph(dev):
    """Another stream, and a captured step replayed while its lengths grow, each replay against the eager call."""
    st = streams(8, dev)
    table, off = ints(st.lines, dev), ints(st.q_off, dev)
    lengths = ints([100, 64], dev)
    ws = torch.empty(mh.flash_attn_pages_128_workspace_bytes(st.q, st.k, st.v, st.k_pages, st.v_pages, table),
                     dtype=torch.uint8, device=dev)
    run = lambda **kw: mh.flash_attn_pages_128(st.q, st.k, st.v, st.k_pages, st.v_pages, table, lengths, off, window=700,  # noqa: E731
                                               **kw)
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for n in (0, 700, 1999):
        lengths.copy_(ints([n, max(0, n - 300)], dev))
        graph.replay()
        eager = run()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)


def test_nothing_to_do(dev):
    """No query rows; no streams with rows: out stays as it is."""
    st = streams(3, dev)
    out = torch.full_like(st.q, 3.0)
    t, n = ints(st.lines, dev), ints(st.kept, dev)
    mh.flash_attn_pages_128(st.q, st.k, st.v, st.k_pages, st.v_pages, t, n, ints([5, 5], dev), out=out)
    assert bool((out == 3).all())
    out = mh.flash_attn_pages_128(st.q, st.k, st.v, st.k_pages, st.v_pages, t, n, ints([5, 5], dev))
    assert not bool(out.any())
    e = st.q[:, :0], st.k[:, :0], st.v[:, :0]
    assert mh.flash_attn_pages_128(*e, st.k_pages, st.v_pages, t, n, ints([0, 0], dev)).shape == (5, 0, 128)


def test_most_streams(dev):
    """As many streams as a call takes, a few of them without kept or new rows."""
    n = mh.MAX_STREAMS
    st = Streams(77, dev, 2, 1, 16, [(7 * s) % 41 for s in range(n)], [0 if s % 97 == 5 else 1 + (s % 50 == 0) for s in range(n)])
    out = torch.zeros_like(st.q)
    st.run(out=out, window=20)
    check(out, *st.want(window=20))


def far_pool(like, dev, storage):
    """A pool of `like`'s pages, 2.5 GB from one to the next."""
    step = 1_250_000_008
    pool = storage.as_strided(like.shape, (step, *like.stride()[1:]))
    pool.copy_(like)
    return pool


def test_pages_past_32_bits_of_offsets(dev):
    """Pages that lie gigabytes apart: attention, rows into them, copies, forks and compactions are those of close ones."""
    st = Streams(5, dev, 4, 2, 32, [70], [3])
    assert st.pages == 6
    size = 5 * 1_250_000_008 + st.k_pages[0].numel()
    k_far = far_pool(st.k_pages, dev, torch.empty(size, dtype=torch.bfloat16, device=dev))
    v_far = far_pool(st.v_pages, dev, torch.empty(size, dtype=torch.bfloat16, device=dev))
    near, far = [st.k_pages, st.v_pages], [k_far, v_far]
    same = lambda: all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(near, far))  # noqa: E731
    want = st.run()
    st.k_pages, st.v_pages = far
    assert torch.equal(st.run(), want)
    table, off = ints([st.lines[0] * 1, [-1] * len(st.lines[0])], dev), ints([0, 5, 5], dev)
    for pools in (near, far):
        refs = torch.zeros(6, dtype=torch.int32, device=dev)
        refs[ints(st.lines[0][:3], dev).long()] = 1
        t = table.clone()
        mh.pages_write(st.k[:, :5].contiguous(), st.v[:, :5].contiguous(), *pools, t, ints([62, 0], dev), off)
        t, missing = mh.pages_fork(pools, t, refs, ints([0, 0], dev), ints([0, 67], dev), 32)
        assert int(missing) == 0
        mh.pages_copy(pools, t[0, :1].contiguous(), t[1, 2:3].contiguous())
        mh.pages_free(t, refs, ints([0, 0], dev), ints([3, 0], dev))
        mh.pages_compact(pools, t, refs)
    assert same()


def test_two_at_once(dev):
    """Two calls on two streams, each with a workspace of its own, again and again."""
    sts = [streams(i, dev, tree=True) for i in (7, 17)]
    want = [st.run(window=90) for st in sts]
    side = [torch.cuda.Stream() for _ in sts]
    ws = [torch.empty(mh.flash_attn_pages_128_workspace_bytes(st.q, st.k, st.v, st.k_pages, st.v_pages, ints(st.lines, dev)),
                      dtype=torch.uint8, device=dev) for st in sts]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for n, st in enumerate(sts):
            with torch.cuda.stream(side[n]):
                got[n].append(st.run(window=90, workspace=ws[n]))
    torch.cuda.synchronize()
    for n in (0, 1):
        for out in got[n]:
            assert torch.equal(out, want[n])


def test_lengths_and_offsets_past_their_ends(dev):
    """Lengths below zero and past the table, and offsets before the first row and past the last, are those ends'."""
    st = streams(8, dev)  # two streams
    table, rows = ints(st.lines, dev), st.q.shape[1]
    full = len(st.lines[0]) * st.page
    run = lambda n, off: mh.flash_attn_pages_128(st.q, st.k, st.v, st.k_pages, st.v_pages, table, ints(n, dev),  # noqa: E731
                                                 ints(off, dev), window=300, sinks=ints([5, 5], dev))
    assert torch.equal(run([-5, 0], [0, 7, rows]), run([0, 0], [0, 7, rows]))
    assert torch.equal(run([-2 ** 31, 64], [-9, 7, rows + 100]), run([0, 64], [0, 7, rows]))
    # What the pages hold past the rows that were kept is NaN, so that only finite places are compared.
    st.k_pages, st.v_pages = st.k_pages.nan_to_num(0.25), st.v_pages.nan_to_num(0.25)
    assert torch.equal(run([2 ** 31 - 1, full + 1], [0, 7, rows]), run([full, full], [0, 7, rows]))
