"""flash_attn_pages_128 over streams of unlike new rows: long runs among single rows, which the one-wave kernel takes where
streams have few list rows on average, slots that are empty at the moment, and counts of row tiles that leave workgroups
over. Against the float64 restatement of test_attn_pages_gpu, whose bounds these are."""
import random

import pytest
import torch

import mako_h3 as mh
from test_attn_dense_gpu import check
from test_attn_pages_gpu import NAN, Streams

pytestmark = pytest.mark.gpu


class Mixed(Streams):
    """As Streams, with the keys that rows see found row by row from their parents'."""

    def seen(self, s, window):
        kept, new = self.kept[s], self.new[s]
        a = self.q_off[s]
        line = torch.zeros((new, new), dtype=torch.bool)      # row i' is i or an ancestor of i
        depth = torch.zeros(new, dtype=torch.long)
        for i in range(new):
            up = i - 1 if self.parents is None else self.parents[a + i]
            if 0 <= up < i:
                line[i], depth[i] = line[up], depth[up] + 1
            line[i, i] = True
        place, sinks = kept + depth, self.sinks[s] if self.sinks else 0
        at = torch.arange(kept)
        near = lambda p: (p < sinks) | (p > place[:, None] - window) if window else torch.ones((new, 1), dtype=torch.bool)  # noqa: E731
        return torch.cat([near(at).expand(new, kept), line & near(place)], 1).to(self.dev)


def test_the_restatements_agree():
    """Mixed.seen is Streams.seen."""
    dev = torch.device("cpu")
    for tree in (False, True):
        st = Mixed(3, dev, 1, 1, 16, [40, 0, 5], [30, 70, 1], tree=tree, sinks=[3, 50, 6])
        for window in (0, 1, 20, 64):
            for s in range(3):
                assert torch.equal(st.seen(s, window), Streams.seen(st, s, window))


# heads, key heads, page, kept, new: of up to 64 list rows a stream on average, which is what the one-wave kernel takes.
LONG = {
    "chunk last": (8, 8, 16, [300] * 63 + [500], [1] * 63 + [510]),
    "chunk first, shared heads": (10, 2, 64, [130] + [777] * 40, [200] + [1] * 40),
    "parents past what LDS holds": (2, 2, 32, [70] + [40] * 80, [1100] + [1] * 80),
    "two chunks among empty slots": (3, 3, 64, [0] * 20 + [1000] + [0] * 30 + [515] + [0] * 12,
                                     [0] * 20 + [510] + [0] * 30 + [130] + [0] * 12),
    "a chunk and nothing kept": (4, 1, 16, [0] * 70, [1] * 35 + [700] + [0] * 34),
    "past 64 streams": (2, 1, 16, [(37 * s) % 300 for s in range(200)], [(s % 50 == 7) * 290 + s % 2 for s in range(200)]),
}


def few(name, dev, **kw):
    heads, kv_heads, page, kept, new = LONG[name]
    assert max(new) > 64 and sum(new) * (heads // kv_heads) <= 60 * len(new)
    return Mixed(len(name), dev, heads, kv_heads, page, kept, new, **kw)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("name", LONG)
def test_long_runs_among_few_rows(dev, name, tree, cap):
    st = few(name, dev, tree=tree, page_layout="rows" if cap else "heads")
    check(st.run(cap=cap), *st.want(cap=cap))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("window", [1, 17, 100, 600])
@pytest.mark.parametrize("name", LONG)
def test_long_runs_under_a_window(dev, name, window, tree):
    st = few(name, dev, tree=tree, sinks=[(0, 1, 5, 70, 400, 2 ** 31 - 1)[(s + window) % 6] for s in range(len(LONG[name][3]))])
    check(st.run(window=window), *st.want(window=window))


@pytest.mark.parametrize("name", ["chunk last", "parents past what LDS holds"])
def test_long_runs_with_missing_pages(dev, name):
    st = few(name, dev, tree=True)
    rng = random.Random(4)
    for line in st.lines:
        for e in range(len(line)):
            if rng.random() < 0.4:
                line[e] = rng.choice([-1, st.pages, -2 ** 31])
    check(st.run(), *st.want())
    check(st.run(window=90), *st.want(window=90))


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("new", [344, 520, 1020])
def test_row_tiles_that_leave_workgroups_over(dev, new, tree, window):
    """64 query heads share a key head: 86, 130 and 255 row tiles of one stream."""
    st = Mixed(new, dev, 64, 1, 32, [500], [new], tree=tree, sinks=[40])
    check(st.run(window=window), *st.want(window=window))


@pytest.mark.parametrize("name", ["chunk last", "chunk first, shared heads", "a chunk and nothing kept"])
def test_unattended_new_rows_leave_no_trace(dev, name):
    """NaN in a new row of a long run changes no bit of the rows whose line it is not on."""
    st = few(name, dev, tree=True)
    clean = st.run(window=400)
    s = max(range(len(st.new)), key=lambda i: st.new[i])
    seen = st.seen(s, 400)[:, st.kept[s]:]
    for j in (st.new[s] - 2, st.new[s] // 2, 3):
        k, v = st.k.clone(), st.v.clone()
        st.k[:, st.q_off[s] + j], st.v[:, st.q_off[s] + j] = NAN, NAN
        got = st.run(window=400)
        st.k, st.v = k, v
        on = torch.zeros(st.q.shape[1], dtype=torch.bool, device=dev)
        on[st.q_off[s]:st.q_off[s + 1]] = seen[:, j]
        assert torch.equal(got[:, ~on], clean[:, ~on])
        assert bool(torch.isnan(got[:, on]).all())


@pytest.mark.parametrize("i", range(3))
def test_infinities_that_rows_attend(dev, i):
    """An infinite value in a kept row and in a new one is in the rows that attend it, and in no other."""
    heads, kv_heads, page, kept, new = [(8, 8, 16, [300] * 5, [2] * 5), (6, 2, 32, [900, 70], [130, 40]), LONG["chunk last"]][i]
    st = Mixed(i, dev, heads, kv_heads, page, kept, new)
    clean = st.run(window=64)
    s, back = len(new) - 1, 40
    at = kept[s] - back
    st.v_pages[st.lines[s][at // page], :, at % page, 5] = float("inf")
    st.v[:, st.q_off[s] + 1, 9] = -float("inf")
    got = st.run(window=64)
    seen = st.seen(s, 64)
    for column, on, value in ((5, seen[:, at], float("inf")), (9, seen[:, kept[s] + 1], -float("inf"))):
        rows = torch.zeros(st.q.shape[1], dtype=torch.bool, device=dev)
        rows[st.q_off[s]:st.q_off[s + 1]] = on
        assert bool((got[:, rows, column] == value).all())
        assert torch.equal(got[:, ~rows, column], clean[:, ~rows, column])
    others = [d for d in range(128) if d not in (5, 9)]
    assert torch.equal(got[:, :, others], clean[:, :, others])


@pytest.mark.parametrize("scale,cap", [(2.0 ** 20, 0.0), (2.0 ** 100, 0.0), (2.0 ** -40, 0.0), (2.0 ** 30, 7.0), (0.1, 2.0 ** -60),
                                       (0.1, 1024.0)])
@pytest.mark.parametrize("heads,kv_heads,kept,new", [(8, 2, [700, 33], [3, 40]), (16, 2, [1500], [90])])
def test_scores_to_the_ends_of_their_range(dev, heads, kv_heads, kept, new, scale, cap):
    """Values of -1, 0 and 1 make the products exact and tie many of them: with a large scale the ties of each row's maximum
    share its probability, whichever tile or part they lie in; with a tiny one, or under a tiny cap, all keys do."""
    st = Mixed(9, dev, heads, kv_heads, 32, kept, new, sinks=[20] * len(kept))
    for x in (st.q, st.k, st.k_pages):
        x.copy_(x.nan_to_num(0.0).clamp(-1.4, 1.4).round())
    for window in (0, 200):
        check(st.run(window=window, scale=scale, cap=cap), *st.want(window=window, scale=scale, cap=cap))
    # The same rows in one piece, under the same window.
    s = len(kept) - 1
    mine = slice(st.q_off[s], st.q_off[s + 1])
    k, v = (torch.cat([st.kept_rows(p, s)[0], x[:, mine]], 1) for p, x in ((st.k_pages, st.k), (st.v_pages, st.v)))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    ranges, first = mh.attn_window_ranges(ints([0, new[s]]), ints([0, kept[s] + new[s]]), new[s], kept[s] + new[s], 200,
                                          sinks=ints([20]))
    want, mag = st.want(window=200, scale=scale, cap=cap)
    check(mh.flash_attn_128(st.q[:, mine].contiguous(), k, v, ranges=ranges, sinks=first, scale=scale, cap=cap),
          want[:, mine], mag[:, mine])
