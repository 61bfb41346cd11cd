"""flash_attn_128 over two ranges a row (`sinks`) and attn_window_ranges, against float64 restatements; the bounds are
those of test_attn_dense_gpu."""
import math

import pytest
import torch

import mako_h3 as mh
from test_attn_dense_gpu import CASES, check, make, random_ranges

pytestmark = pytest.mark.gpu


def seen_of(ranges, sinks, keys):
    at = torch.arange(keys, device=ranges.device)
    seen = torch.zeros((ranges.shape[0], keys), dtype=torch.bool, device=ranges.device)
    for r in (ranges, sinks):
        lo, hi = r[:, 0].long().clamp(0, keys), r[:, 1].long().clamp(0, keys)
        seen |= (at >= lo[:, None]) & (at < hi[:, None])
    return seen


def attention64(q, k, v, seen, scale=None, cap=0.0, slopes=None, q_pos=None, k_pos=None):
    """(out, sum of p |v|), float64, over the keys that `seen` [rows][keys] says; the others are left out, whatever they
    hold."""
    heads, rows, n = q.shape[0], q.shape[1], k.shape[1]
    dev, share = q.device, heads // k.shape[0]
    out = torch.zeros((heads, rows, 128), dtype=torch.float64, device=dev)
    mag = torch.zeros_like(out)
    for h in range(heads):
        kd, vd = k[h // share].double(), v[h // share].double()
        s = q[h].double() @ kd.T.contiguous() * (scale or 1 / math.sqrt(128))
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            qp = torch.arange(rows, device=dev) if q_pos is None else q_pos.long()
            kp = torch.arange(n, device=dev) if k_pos is None else k_pos.long()
            s = s - slopes[h].double() * (qp[:, None] - kp).abs().double()
        s = torch.where(seen, s, -math.inf)
        p = torch.where(seen, torch.softmax(s, -1), 0.0)
        finite = torch.isfinite(vd).all(1)
        clean = torch.where(finite[:, None], vd, 0.0)
        out[h], mag[h] = p @ clean, p @ clean.abs()
        for j in torch.nonzero(~finite).flatten().tolist():     # non-finite keys, into the rows that attend them
            out[h, seen[:, j]] += p[seen[:, j], j, None] * vd[j]
    return out, mag


@pytest.mark.parametrize("cap,bias", [(0.0, False), (5.0, False), (0.0, True), (20.0, True)])
@pytest.mark.parametrize("heads,kv_heads,rows,keys", CASES)
def test_two_ranges(dev, heads, kv_heads, rows, keys, cap, bias):
    """Two ranges of any kind: apart in either order, touching, one in the other, empty."""
    g = torch.Generator(device=dev).manual_seed(7 + heads + rows * keys)
    q, k, v = make(g, heads, rows, dev), make(g, kv_heads, keys, dev), make(g, kv_heads, keys, dev)
    ranges, sinks = (random_ranges(g, rows, keys, dev) for _ in range(2))
    kind = torch.randint(0, 4, (rows,), generator=g, device=dev)
    sinks[kind == 0, 1] = ranges[kind == 0, 0]                      # one behind the other, if not empty
    sinks[kind == 1] = sinks[kind == 1].clamp(max=keys // 8)        # few, in front
    kw = {"cap": cap, "scale": 0.2}
    if bias:
        kw["slopes"] = torch.rand(heads, generator=g, device=dev) * 0.2
        if rows % 2:
            kw["q_pos"] = torch.randint(-50, 50, (rows,), generator=g, device=dev, dtype=torch.int32)
            kw["k_pos"] = torch.randint(-50, 50, (keys,), generator=g, device=dev, dtype=torch.int32)
    out = mh.flash_attn_128(q, k, v, ranges=ranges, sinks=sinks, out=torch.full_like(q, float("nan")), **kw)
    seen = seen_of(ranges, sinks, keys)
    check(out, *attention64(q, k, v, seen, **kw))
    assert not bool(out[:, ~seen.any(1)].any())


WINDOWS = [
    # document lengths, query rows of each (0: all), window, sinks, heads, key heads
    ([1], 0, 1, 0, 1, 1), ([5], 0, 3, 1, 2, 1), ([200], 0, 64, 4, 5, 1), ([64, 0, 130, 33], 0, 16, 3, 2, 2),
    ([300, 200], 0, 1000, 40, 4, 2), ([1100, 40, 777], 0, 100, 77, 8, 2), ([5000], 0, 700, 130, 2, 2),
    ([900, 40, 77], 1, 32, 4, 40, 8), ([4000, 300], 7, 200, 64, 7, 1), ([129, 257, 1], 0, 1, 0, 3, 3),
    ([2500], 0, 64, 1, 56, 8), ([700, 900], 0, 4000000000, 5, 2, 1), ([30000, 100], 3, 4080, 435, 8, 8),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,new,window,sinks,heads,kv_heads", WINDOWS)
def test_window(dev, lengths, new, window, sinks, heads, kv_heads, causal):
    """Packed documents under a window (rows before the first document and behind the last, first rows of uneven numbers)
    from attn_window_ranges, against the definition key by key."""
    g = torch.Generator(device=dev).manual_seed(sum(lengths) + new + window % 1000)
    queries = [min(new, n) if new else n for n in lengths]
    q_cuts, k_cuts = [3], [2]
    for a, b in zip(queries, lengths):
        q_cuts.append(q_cuts[-1] + a)
        k_cuts.append(k_cuts[-1] + b)
    rows, keys = q_cuts[-1] + 5, k_cuts[-1] + 4
    off = lambda c: torch.tensor(c, dtype=torch.int32, device=dev)  # noqa: E731
    front = [max(0, sinks - d) for d in range(len(lengths))]
    ranges, first = mh.attn_window_ranges(off(q_cuts), off(k_cuts), rows, keys, window, causal=causal,
                                          sinks=off(front) if sinks else None)
    at, seen = torch.arange(keys, device=dev), torch.zeros((rows, keys), dtype=torch.bool, device=dev)
    for d, n in enumerate(lengths):
        for i in range(queries[d]):
            own = k_cuts[d] + n - queries[d] + i
            line = (at - own).abs() < window
            line |= at < k_cuts[d] + front[d]
            line &= (at >= k_cuts[d]) & (at < k_cuts[d] + n)
            if causal:
                line &= at <= own
            seen[q_cuts[d] + i] = line
    assert torch.equal(seen_of(ranges, first, keys), seen)
    q, k, v = make(g, heads, rows, dev), make(g, kv_heads, keys, dev), make(g, kv_heads, keys, dev)
    out = mh.flash_attn_128(q, k, v, ranges=ranges, sinks=first)
    check(out, *attention64(q, k, v, seen))
    assert not bool(out[:, :3].any()) and not bool(out[:, q_cuts[-1]:].any())


def test_window_past_the_keys(dev):
    """Offsets before the first key and past the last: what lies among the keys remains. More query rows than keys: the
    first ones sit before the document and see nothing."""
    off = lambda c: torch.tensor(c, dtype=torch.int32, device=dev)  # noqa: E731
    ranges, first = mh.attn_window_ranges(off([0, 4]), off([-6, 14]), 4, 10, 5, sinks=off([8]))
    assert ranges.tolist() == [[6, 10], [7, 10], [8, 10], [9, 10]] and first.tolist() == [[0, 2]] * 4
    ranges, first = mh.attn_window_ranges(off([0, 6]), off([3, 6]), 6, 10, 2, sinks=off([1]))
    assert ranges.tolist() == [[0, 0]] * 3 + [[3, 4], [3, 5], [4, 6]] and first.tolist() == [[0, 0]] * 5 + [[3, 4]]
    ranges, first = mh.attn_window_ranges(off([0, 6]), off([3, 6]), 6, 10, 2, sinks=off([-4]), causal=False)
    assert ranges.tolist() == [[0, 0]] * 2 + [[3, 4], [3, 5], [3, 6], [4, 6]] and not bool(first.any())


@pytest.mark.parametrize("heads,kv_heads,rows,keys", [(4, 2, 40, 900), (2, 2, 700, 1500), (8, 8, 900, 900)])
def test_unattended_keys_leave_no_trace(dev, heads, kv_heads, rows, keys):
    """Infinities and NaN in keys and values that a row does not attend change none of its bits, and the row's neighbours'
    ranges and q neither."""
    g = torch.Generator(device=dev).manual_seed(rows)
    q, k, v = make(g, heads, rows, dev), make(g, kv_heads, keys, dev), make(g, kv_heads, keys, dev)
    own = torch.arange(rows, device=dev) * keys // rows
    ranges = torch.stack([(own - 90).clamp(min=0), own + 1], 1).int().contiguous()
    sinks = torch.tensor([[0, 70]], dtype=torch.int32, device=dev).expand(rows, 2).contiguous()
    clean = mh.flash_attn_128(q, k, v, ranges=ranges, sinks=sinks)
    for bad in (float("nan"), float("inf"), -3e38):
        k2, v2 = k.clone(), v.clone()
        k2[:, 300], v2[:, 300], v2[:, 301, 5], k2[:, 69] = bad, bad, bad, bad
        out = mh.flash_attn_128(q, k2, v2, ranges=ranges, sinks=sinks)
        seen = seen_of(ranges, sinks, keys)
        away = ~(seen[:, 300] | seen[:, 301] | seen[:, 69])
        assert torch.equal(out[:, away], clean[:, away])
        near = mh.flash_attn_128(q, k2, v2, ranges=ranges, sinks=torch.zeros_like(sinks))
        alone = mh.flash_attn_128(q, k, v, ranges=ranges, sinks=torch.zeros_like(sinks))
        assert torch.equal(near[:, ~seen[:, 300] & ~seen[:, 301]][:, 200:], alone[:, ~seen[:, 300] & ~seen[:, 301]][:, 200:])
        if bad == math.inf:     # 128 products with -3e38 leave a float's range, but not float64's
            check(out, *attention64(q, k2, v2, seen))


def test_layouts_and_graph(dev):
    """Rows of heads side by side, a workspace of the caller's, another stream, and a captured call replayed on new
    inputs."""
    g = torch.Generator(device=dev).manual_seed(4)
    q, k, v = make(g, 8, 120, dev), make(g, 2, 3000, dev), make(g, 2, 3000, dev)
    off_q, off_k = (torch.tensor(c, dtype=torch.int32, device=dev) for c in ([0, 50, 120], [0, 1000, 3000]))
    text = torch.tensor([20, 300], dtype=torch.int32, device=dev)
    ranges, sinks = mh.attn_window_ranges(off_q, off_k, 120, 3000, 500, sinks=text)
    want = mh.flash_attn_128(q, k, v, ranges=ranges, sinks=sinks)
    rows = [x.transpose(0, 1).reshape(x.shape[1], -1) for x in (q, k, v)]
    ws = torch.empty(max(1, mh.flash_attn_128_workspace_bytes(q, k, v)), dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mh.flash_attn_128(*rows, ranges=ranges, sinks=sinks, layout="rows", out_layout="heads", workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, s = mh.attn_window_ranges(off_q, off_k, 120, 3000, 500, sinks=text)
        captured = mh.flash_attn_128(q, k, v, ranges=r, sinks=s)
    for i in range(3):
        q.copy_(make(g, 8, 120, dev))
        text.copy_(torch.tensor([i, 77 * i], dtype=torch.int32))
        graph.replay()
        r, s = mh.attn_window_ranges(off_q, off_k, 120, 3000, 500, sinks=text)
        eager = mh.flash_attn_128(q, k, v, ranges=r, sinks=s)
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)
