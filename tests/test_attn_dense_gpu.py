"""flash_attn_128 and attn_ranges against a float64 restatement.

The bound of an output element: its rounding to bf16 (2^-8 of it), the rounding of each probability to bf16 (2^-8 of the
sum of p |v|), and for the scores' float errors (some 128 roundings of 2^-24 at |q . k| scale up to 10, the exponential's
and the cap's 2^-22) another 2^-11 of that sum."""
import math

import pytest
import torch

import mako_h3 as mh

pytestmark = pytest.mark.gpu


def make(g, heads, rows, dev, scale=1.0):
    return (torch.randn((heads, rows, 128), generator=g, device=dev) * scale).to(torch.bfloat16)


def attention64(q, k, v, ranges=None, scale=None, cap=0.0, slopes=None, q_pos=None, k_pos=None):
    """(out, sum of p |v|), float64 [heads][rows][128]; masked keys are left out, whatever they hold."""
    heads, rows, n = q.shape[0], q.shape[1], k.shape[1]
    dev, share = q.device, heads // k.shape[0]
    at = torch.arange(n, device=dev)
    if ranges is None:
        seen = torch.ones((rows, n), dtype=torch.bool, device=dev)
    else:
        lo, hi = ranges[:, 0].long().clamp(0, n), ranges[:, 1].long().clamp(0, n)
        seen = (at >= lo[:, None]) & (at < hi[:, None])
    out = torch.zeros((heads, rows, 128), dtype=torch.float64, device=dev)
    mag = torch.zeros_like(out)
    some = seen.any(1)
    for h in range(heads):
        kd, vd = k[h // share].double(), v[h // share].double()
        s = q[h].double() @ kd.T.contiguous() * (scale or 1 / math.sqrt(128))
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            qp = torch.arange(rows, device=dev) if q_pos is None else q_pos.long()
            kp = at if k_pos is None else k_pos.long()
            s = s - slopes[h].double() * (qp[:, None] - kp).abs().double()
        s = torch.where(seen, s, -math.inf)
        p = torch.softmax(s, -1) if n else s
        p = torch.where(seen, p, 0.0)
        p[~some] = 0.0
        finite = torch.isfinite(vd).all(1) if n else torch.ones(0, dtype=torch.bool, device=dev)
        clean = torch.where(finite[:, None], vd, 0.0)
        out[h], mag[h] = p @ clean, p @ clean.abs()
        for j in torch.nonzero(~finite).flatten().tolist():     # non-finite keys, into the rows that attend them
            rows_j = seen[:, j]
            out[h, rows_j] += p[rows_j, j, None] * vd[j]
    return out, mag


def check(got, want, mag, what=""):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN"
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin].nan_to_num(), want[~fin].nan_to_num()), f"{what}: infinities"
    err = (got - want).abs()[fin]
    bound = (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * mag)[fin]
    assert bool((err <= bound).all()), f"{what}: worst {float((err / bound.clamp_min(1e-300)).max()):.3g} of the bound"


CASES = [
    # heads, key heads, query rows, key rows
    (1, 1, 1, 1), (1, 1, 1, 64), (2, 1, 1, 65), (5, 1, 1, 1000), (40, 8, 1, 777), (3, 3, 31, 63), (2, 2, 32, 64),
    (2, 2, 33, 129), (7, 1, 20, 500), (4, 2, 127, 128), (4, 2, 128, 127), (3, 1, 129, 300), (56, 56, 77, 212),
    (2, 2, 257, 1025), (40, 8, 260, 333), (56, 8, 300, 100), (40, 40, 945, 945), (1, 1, 2000, 130), (6, 3, 700, 2000),
    (12, 2, 3, 20000), (64, 64, 1100, 200),
]


@pytest.mark.parametrize("heads,kv_heads,rows,keys", CASES)
def test_every_row_over_every_key(dev, heads, kv_heads, rows, keys):
    g = torch.Generator(device=dev).manual_seed(heads + rows * keys)
    q, k, v = make(g, heads, rows, dev), make(g, kv_heads, keys, dev), make(g, kv_heads, keys, dev)
    out = torch.full_like(q, float("nan"))
    assert mh.flash_attn_128(q, k, v, out=out) is out
    check(out, *attention64(q, k, v))


def random_ranges(g, rows, keys, dev):
    """Ranges of all kinds: whole, empty, one key, either end, random."""
    r = torch.randint(0, keys + 1, (rows, 2), generator=g, device=dev).sort(1).values
    kind = torch.randint(0, 7, (rows,), generator=g, device=dev)
    lo, hi = r[:, 0].clone(), r[:, 1].clone()
    lo[kind == 0], hi[kind == 0] = 0, keys
    hi[kind == 1] = lo[kind == 1]
    hi[kind == 2] = (lo[kind == 2] + 1).clamp(max=keys)
    lo[kind == 3], hi[kind == 4] = 0, keys
    return torch.stack([lo, hi], 1).int().contiguous()


@pytest.mark.parametrize("cap,bias", [(0.0, False), (5.0, False), (0.0, True), (20.0, True)])
@pytest.mark.parametrize("heads,kv_heads,rows,keys", CASES)
def test_ranges_cap_and_bias(dev, heads, kv_heads, rows, keys, cap, bias):
    g = torch.Generator(device=dev).manual_seed(1 + heads + rows * keys)
    q, k, v = make(g, heads, rows, dev), make(g, kv_heads, keys, dev), make(g, kv_heads, keys, dev)
    kw = {"ranges": random_ranges(g, rows, keys, dev), "cap": cap, "scale": 0.2}
    if bias:
        kw["slopes"] = torch.rand(heads, generator=g, device=dev) * 0.2
        if rows % 2:
            kw["q_pos"] = torch.randint(-50, 50, (rows,), generator=g, device=dev, dtype=torch.int32)
            kw["k_pos"] = torch.randint(-50, 50, (keys,), generator=g, device=dev, dtype=torch.int32)
    out = mh.flash_attn_128(q, k, v, out=torch.full_like(q, float("nan")), **kw)
    check(out, *attention64(q, k, v, **kw))
    empty = kw["ranges"][:, 0] >= kw["ranges"][:, 1]
    assert not bool(out[:, empty].any())


@pytest.mark.parametrize("causal,prefix", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("lengths,new", [([5], 0), ([1, 1, 1], 0), ([64, 0, 130, 33], 0), ([300, 200], 0),
                                         ([900, 40, 77], 1), ([500, 300], 7), ([129, 257, 1], 0)])
def test_documents(dev, lengths, new, causal, prefix):
    """Packed documents (some empty, rows before the first and behind the last) through attn_ranges, against each
    document on its own."""
    g = torch.Generator(device=dev).manual_seed(sum(lengths) + new)
    queries = [min(new, n) if new else n for n in lengths]
    q_cuts, k_cuts = [3], [2]
    for a, b in zip(queries, lengths):
        q_cuts.append(q_cuts[-1] + a)
        k_cuts.append(k_cuts[-1] + b)
    rows, keys = q_cuts[-1] + 5, k_cuts[-1] + 4
    off = lambda c: torch.tensor(c, dtype=torch.int32, device=dev)  # noqa: E731
    pre = [min(n // 2, 70) for n in lengths] if prefix else None
    ranges = mh.attn_ranges(off(q_cuts), off(k_cuts), rows, keys, causal=causal, prefix=off(pre) if prefix else None)
    want = torch.zeros((rows, 2), dtype=torch.int64)
    for d, n in enumerate(lengths):
        for i in range(queries[d]):
            own = n - queries[d] + i + 1
            hi = n if not causal else min(n, max(own, pre[d] if prefix else 0))
            want[q_cuts[d] + i] = torch.tensor([k_cuts[d], k_cuts[d] + hi])
    assert torch.equal(ranges.cpu().long(), want)
    q, k, v = make(g, 4, rows, dev), make(g, 2, keys, dev), make(g, 2, keys, dev)
    out = mh.flash_attn_128(q, k, v, ranges=ranges)
    check(out, *attention64(q, k, v, ranges=ranges))
    assert not bool(out[:, :3].any()) and not bool(out[:, q_cuts[-1]:].any())


@pytest.mark.parametrize("rows,keys,heads", [(5, 200, 2), (64, 300, 1), (140, 700, 3), (1, 3000, 4), (600, 600, 64)])
def test_nothing_comes_from_masked_keys(dev, rows, keys, heads):
    """Infinities and NaN in keys and values that a row does not attend change none of its bits; a row that attends them
    gets what the formula gives."""
    g = torch.Generator(device=dev).manual_seed(rows)
    q, k, v = make(g, heads, rows, dev), make(g, heads, keys, dev), make(g, heads, keys, dev)
    # Rows 0 :: 2 attend the front, the others the back; the poisoned keys lie in the back.
    cut = keys // 3 + 5
    ranges = torch.tensor([[0, cut], [cut, keys]], dtype=torch.int32, device=dev).repeat((rows + 1) // 2, 1)[:rows]
    ranges = ranges.contiguous()
    clean = mh.flash_attn_128(q, k, v, ranges=ranges)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, cut + 1], bad_k[:, keys - 1] = float("nan"), float("inf")
    bad_v[:, cut], bad_v[:, keys - 2] = float("inf"), float("nan")
    got = mh.flash_attn_128(q, bad_k, bad_v, ranges=ranges)
    assert torch.equal(got[:, 0::2], clean[:, 0::2])
    assert bool(torch.isnan(got[:, 1::2]).all())
    # Poisoned values alone: infinite in one key, NaN in another of a few columns.
    bad_v = v.clone()
    bad_v[:, cut + 2, 3], bad_v[:, cut + 9, 70], bad_v[:, keys - 1, 127] = float("inf"), float("nan"), -float("inf")
    got = mh.flash_attn_128(q, k, bad_v, ranges=ranges)
    assert torch.equal(got[:, 0::2], clean[:, 0::2])
    want, mag = attention64(q, k, bad_v, ranges=ranges)
    check(got, want, mag + 1e-3)


def test_lowest_values_and_infinite_scores(dev):
    """Scores that are all -inf make a row NaN (0 / 0), some leave it to the others; equal lowest scores share evenly."""
    q = torch.ones((1, 4, 128), dtype=torch.bfloat16, device=dev)
    k = torch.zeros((1, 70, 128), dtype=torch.bfloat16, device=dev)
    v = torch.arange(70, device=dev).to(torch.bfloat16)[None, :, None].expand(1, 70, 128).contiguous()
    k[0, :35] = -float("inf")
    ranges = torch.tensor([[0, 70], [0, 35], [35, 70], [3, 3]], dtype=torch.int32, device=dev)
    out = mh.flash_attn_128(q, k, v, ranges=ranges)[0].float()
    assert float(out[0, 0]) == float(out[2, 0]) == 52.0
    assert bool(torch.isnan(out[1]).all()) and not bool(out[3].any())
    k[0, :] = -3.0e36  # 128 of them scaled: beyond -3e37, float still
    out = mh.flash_attn_128(q, k, v)[0].float()
    assert abs(float(out[0, 0]) - 34.5) <= 34.5 * 2.0 ** -8


@pytest.mark.parametrize("rows,keys", [(1, 900), (90, 400), (700, 333)])
def test_layouts_and_strides(dev, rows, keys):
    """Head tiles, the model's row order, slices of a fused [q | k | v] row, a key head stride of zero and an output in the
    other layout: the same bits."""
    g = torch.Generator(device=dev).manual_seed(rows)
    heads = 6
    n = max(rows, keys)
    fused = torch.randn((n, 3 * heads * 128), generator=g, device=dev).to(torch.bfloat16)
    part = lambda i, m: fused[:m, i * heads * 128:(i + 1) * heads * 128]  # noqa: E731
    tiles = lambda t: t.reshape(t.shape[0], heads, 128).transpose(0, 1).contiguous()  # noqa: E731
    q, k, v = part(0, rows), part(1, keys), part(2, keys)
    want = mh.flash_attn_128(tiles(q), tiles(k), tiles(v))
    flat = want.transpose(0, 1).reshape(rows, heads * 128)
    assert torch.equal(mh.flash_attn_128(q, k, v, layout="rows"), flat)
    assert torch.equal(mh.flash_attn_128(q, k, v, layout="rows", out_layout="heads"), want)
    wide = torch.zeros((rows, 2 * heads * 128), dtype=torch.bfloat16, device=dev)
    mh.flash_attn_128(tiles(q), tiles(k), tiles(v), out=wide[:, heads * 128:], out_layout="rows")
    assert torch.equal(wide[:, heads * 128:], flat) and not bool(wide[:, :heads * 128].any())
    one_k, one_v = tiles(k)[:1].expand(heads, keys, 128), tiles(v)[:1].expand(heads, keys, 128)
    assert torch.equal(mh.flash_attn_128(tiles(q), one_k, one_v),
                       mh.flash_attn_128(tiles(q), one_k.contiguous(), one_v.contiguous()))


def test_offsets_past_32_bits(dev):
    """Key rows 256 KB apart: byte offsets up to 5 GB."""
    g = torch.Generator(device=dev).manual_seed(2)
    keys, stride = 20000, 1 << 17
    store = torch.zeros(keys * stride, dtype=torch.bfloat16, device=dev)
    k, v = (torch.as_strided(store, (1, keys, 128), (0, stride, 1), o) for o in (0, 4096))
    k.copy_(make(g, 1, keys, dev))
    v.copy_(make(g, 1, keys, dev))
    for rows in (2, 200):
        q = make(g, 1, rows, dev)
        out = mh.flash_attn_128(q, k, v)
        check(out, *attention64(q, k.contiguous(), v.contiguous()))


def test_no_rows_and_no_keys(dev):
    q, none = torch.ones((2, 5, 128), dtype=torch.bfloat16, device=dev), torch.empty((2, 0, 128), dtype=torch.bfloat16,
                                                                                    device=dev)
    assert not bool(mh.flash_attn_128(q, none, none).any())
    assert mh.flash_attn_128(none, q, q).shape == (2, 0, 128)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_a_poisoned_workspace_and_two_streams(dev, rows):
    """What the workspace holds before a call does not matter, and calls on two streams with their own do not meet."""
    g = torch.Generator(device=dev).manual_seed(rows)
    q, k, v = make(g, 8, rows, dev), make(g, 2, 5000, dev), make(g, 2, 5000, dev)
    want = mh.flash_attn_128(q, k, v)
    n = mh.flash_attn_128_workspace_bytes(q, k, v)
    spaces = [torch.full((max(n, 16),), 255, dtype=torch.uint8, device=dev) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s, w in zip(streams, spaces):
        with torch.cuda.stream(s):
            outs.append([mh.flash_attn_128(q, k, v, workspace=w) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for several in outs for o in several)


def test_replayed_from_graphs(dev):
    """Two captured graphs (long and few rows) replayed in turn, each with its own buffers, against eager calls."""
    g = torch.Generator(device=dev).manual_seed(8)
    sets = [(make(g, 8, r, dev), make(g, 2, 3000, dev), make(g, 2, 3000, dev)) for r in (2, 400)]
    off = torch.tensor([0, 1000, 3000], dtype=torch.int32, device=dev)
    q_off = [torch.tensor([0, r // 2, r], dtype=torch.int32, device=dev) for r in (2, 400)]

    def run(i):
        q, k, v = sets[i]
        return mh.flash_attn_128(q, k, v, ranges=mh.attn_ranges(q_off[i], off, q.shape[1], 3000, causal=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(0), run(1)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(i))
        graphs.append(graph)
    for _ in range(3):
        for i in range(2):
            for t in sets[i]:
                t.copy_(torch.randn(t.shape, generator=g, device=dev))
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], run(i))


@pytest.mark.parametrize("rows,keys", [(700, 1000), (6, 900), (130, 70)])
@pytest.mark.parametrize("cap", [0.0, 15.0])
def test_positions_near_and_far(dev, rows, keys, cap):
    """Positions whose differences a float holds, ones that it does not, both in one call (key tiles of either kind,
    query rows of either kind), and both ends of int32."""
    g = torch.Generator(device=dev).manual_seed(rows + keys)
    q, k, v = make(g, 6, rows, dev), make(g, 2, keys, dev), make(g, 2, keys, dev)
    near_q = torch.randint(0, 100, (rows,), generator=g, device=dev, dtype=torch.int32)
    near_k = torch.randint(0, 100, (keys,), generator=g, device=dev, dtype=torch.int32)
    far_q = torch.randint(-(1 << 31), 1 << 31, (rows,), generator=g, device=dev).int()
    far_k = torch.randint(-(1 << 31), 1 << 31, (keys,), generator=g, device=dev).int()
    far_k[:2] = torch.tensor([-(1 << 31), (1 << 31) - 1], device=dev).int()
    far_q[0] = -(1 << 31)
    mixed_k = torch.where(torch.arange(keys, device=dev) // 64 % 3 == 1, far_k, near_k)
    mixed_q = torch.where(torch.arange(rows, device=dev) // 40 % 2 == 1, far_q, near_q)
    shifted = 1 << 30
    for slope, qp, kp in ((0.1, near_q, near_k), (0.1, near_q + shifted, near_k + shifted), (3e-9, far_q, far_k),
                          (3e-9, near_q, mixed_k), (3e-9, mixed_q, near_k), (3e-9, mixed_q, mixed_k),
                          (2e-6, near_q * 300000, near_k * 300000), (0.0, far_q, near_k), (-0.05, near_q, near_k)):
        slopes = slope * (1 + torch.rand(6, generator=g, device=dev))
        kw = {"slopes": slopes, "q_pos": qp.contiguous(), "k_pos": kp.contiguous(), "cap": cap,
              "ranges": random_ranges(g, rows, keys, dev)}
        check(mh.flash_attn_128(q, k, v, **kw), *attention64(q, k, v, **kw), f"slope {slope}")


@pytest.mark.parametrize("heads,kv_heads,rows", [(40, 8, 900), (8, 8, 600), (8, 1, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_steep_slopes(dev, heads, kv_heads, rows, causal):
    """Scores that rise or fall by tens a key tile: a bias of up to 450, whose 2^-24 is inside the bound's 2^-11."""
    g = torch.Generator(device=dev).manual_seed(heads * rows)
    q, k, v = make(g, heads, rows, dev), make(g, kv_heads, rows, dev), make(g, kv_heads, rows, dev)
    off = torch.tensor([0, rows], dtype=torch.int32, device=dev)
    ranges = mh.attn_ranges(off, off, rows, rows, causal=causal)
    for sign in (1.0, -1.0):
        slopes = sign * 0.5 ** torch.linspace(1.0, 8.0, heads, device=dev)
        check(mh.flash_attn_128(q, k, v, ranges=ranges, slopes=slopes), *attention64(q, k, v, ranges=ranges, slopes=slopes))


@pytest.mark.parametrize("lengths", [[300, 64, 500, 129], [700, 5], [64, 64, 64, 512, 256]])
@pytest.mark.parametrize("causal,bias,cap", [(False, False, 0.0), (True, False, 0.0), (True, True, 0.0), (False, True, 9.0)])
def test_infinite_values_in_masked_and_whole_tiles(dev, lengths, causal, bias, cap):
    """Infinities and NaN in the values of some keys of every document: they reach the rows that attend them, and no
    others, whether their tile is masked, whole, or between the two."""
    g = torch.Generator(device=dev).manual_seed(sum(lengths))
    n = sum(lengths)
    q, k, v = make(g, 4, n, dev), make(g, 2, n, dev), make(g, 2, n, dev)
    off = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=dev)
    for i, (start, length) in enumerate(zip(off.tolist(), lengths)):
        v[i % 2, start + length // 2, 3 * i] = float("inf")
        v[(i + 1) % 2, start + length - 1, 40 + i] = float("-inf") if i % 2 else float("nan")
    ranges = mh.attn_ranges(off, off, n, n, causal=causal)
    kw = {"ranges": ranges, "cap": cap}
    if bias:
        kw["slopes"] = torch.rand(4, generator=g, device=dev) * 0.02
    check(mh.flash_attn_128(q, k, v, **kw), *attention64(q, k, v, **kw))


@pytest.mark.parametrize("heads,kv_heads,keys,news", [
    (16, 16, [60000], [40]), (16, 16, [20000, 20001, 19999], [12, 12, 12]), (16, 16, [1, 30000, 63, 0, 30000], [1, 30, 5, 0, 20]),
    (40, 8, [100000], [28]), (40, 8, [30000, 40000, 30000], [4, 4, 4]), (40, 8, [2000] * 50, [1] * 50),
    (40, 8, [50000, 50000], [28, 28])])
@pytest.mark.parametrize("causal,cap,bias", [(True, 0.0, False), (False, 30.0, False), (True, 0.0, True)])
def test_a_batch_of_streams_with_new_rows(dev, heads, kv_heads, keys, news, causal, cap, bias):
    """New rows of one or many streams against long kept keys: the sizes where the ranges decide which of the two kernels
    runs, with one, few or many rows a stream, empty streams, and rows of none in front."""
    g = torch.Generator(device=dev).manual_seed(sum(keys) + sum(news))
    rows, n = 3 + sum(news), sum(keys)
    q, k, v = make(g, heads, rows, dev), make(g, kv_heads, n, dev), make(g, kv_heads, n, dev)
    cut = lambda a, at: torch.tensor([at, *(torch.tensor(a).cumsum(0) + at).tolist()], dtype=torch.int32, device=dev)  # noqa: E731
    kw = {"ranges": mh.attn_ranges(cut(news, 3), cut(keys, 0), rows, n, causal=causal), "cap": cap}
    if bias:
        kw["slopes"] = 0.5 ** torch.linspace(4.0, 12.0, heads, device=dev)
        kw["q_pos"] = torch.randint(0, 40, (rows,), generator=g, device=dev, dtype=torch.int32)
        kw["k_pos"] = torch.arange(n, device=dev, dtype=torch.int32) // 510
    ws = torch.full((mh.flash_attn_128_workspace_bytes(q, k, v),), 0xff, dtype=torch.uint8, device=dev)
    out = mh.flash_attn_128(q, k, v, workspace=ws, **kw)
    ws.fill_(0xff)
    assert torch.equal(mh.flash_attn_128(q, k, v, workspace=ws, **kw), out)
    for h in range(0, heads, heads // 4):
        j = h // (heads // kv_heads)
        part = {**kw, **({"slopes": kw["slopes"][h:h + 1]} if bias else {})}
        check(out[h:h + 1], *attention64(q[h:h + 1], k[j:j + 1], v[j:j + 1], **part), f"head {h}")


def test_streams_that_change_under_a_graph(dev):
    """One captured call, replayed for one stream and for many: each replay takes the kernel of its own ranges."""
    g = torch.Generator(device=dev).manual_seed(77)
    rows, n = 28, 100000
    q, k, v = make(g, 40, rows, dev), make(g, 8, n, dev), make(g, 8, n, dev)
    ranges = torch.zeros((rows, 2), dtype=torch.int32, device=dev)
    run = lambda: mh.flash_attn_128(q, k, v, ranges=ranges)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for docs in (1, 28, 2, 0, 7):
        ranges.zero_()
        if docs:
            lo = torch.arange(rows, device=dev) * docs // rows * (n // docs)
            ranges.copy_(torch.stack([lo, lo + n // docs], 1))
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check(out[:1], *attention64(q[:1], k[:1], v[:1], ranges=ranges), f"{docs} streams")


@pytest.mark.parametrize("cap,scale", [(2.0 ** -60, None), (1e-6, None), (1024.0, None), (1024.0, 3.0), (30.0, 1e-30), (0.0, 1e-40),
                                       (0.0, 0.5)])
def test_ends_of_the_caps_and_scales(dev, cap, scale):
    """The whole domain of both: a cap of 1024 is off by 2^-23 of it, inside the bound's 2^-11."""
    g = torch.Generator(device=dev).manual_seed(3)
    q, k, v = make(g, 2, 300, dev), make(g, 2, 200, dev), make(g, 2, 200, dev)
    q[0, 7], k[1, 5] = 0.0, 0.0
    for rows in (300, 5):
        kw = {"cap": cap, **({"scale": scale} if scale else {})}
        check(mh.flash_attn_128(q[:, :rows], k, v, **kw), *attention64(q[:, :rows], k, v, **kw), f"{rows} rows")


@pytest.mark.parametrize("rows", [300, 5])
@pytest.mark.parametrize("cap,scale", [(2.0 ** -60, 2.0 ** 100), (2.0 ** -60, 2.0 ** 67), (1e-9, 2.0 ** 100), (1024.0, 2.0 ** 100),
                                       (0.0, 2.0 ** 100)])
def test_the_largest_scales_under_caps(dev, rows, cap, scale):
    """scale / cap beyond what a float holds: a dot product of zero is still a score of zero, others are at the cap."""
    g = torch.Generator(device=dev).manual_seed(4)
    q, k, v = make(g, 2, rows, dev), make(g, 2, 200, dev), make(g, 2, 200, dev)
    q[0, 3], q[1], k[:, 7], k[1, 150:] = 0.0, 0.0, 0.0, 0.0
    kw = {"cap": cap, "scale": scale}
    check(mh.flash_attn_128(q, k, v, **kw), *attention64(q, k, v, **kw))
    kw["ranges"] = random_ranges(g, rows, 200, dev)
    check(mh.flash_attn_128(q, k, v, **kw), *attention64(q, k, v, **kw))


@pytest.mark.parametrize("causal,prefix", [(False, None), (True, None), (True, [30, 0]), (True, [-5, 1 << 30])])
@pytest.mark.parametrize("k_cuts,keys", [([0, 100, 180], 90), ([-20, 40, 130], 90), ([-50, -10, 20], 200), ([5, 300, 310], 100),
                                         ([120, 150, 200], 100), ([-(1 << 31), 0, (1 << 31) - 1], 50), ([0, 60, 130], 130)])
def test_documents_that_the_keys_cut_off(dev, k_cuts, keys, causal, prefix):
    """Offsets before the first key and past the last: the documents' rows, diagonals and prefixes lie where the offsets say,
    and of the resulting ranges what the keys hold remains."""
    q_cuts = [4, 64, 131]
    rows = 140
    off = lambda c: torch.tensor(c, dtype=torch.int64, device=dev).int()  # noqa: E731
    got = mh.attn_ranges(off(q_cuts), off(k_cuts), rows, keys, causal=causal, prefix=None if prefix is None else off(prefix))
    want = torch.zeros((rows, 2), dtype=torch.int64)
    for d in range(2):
        start, end = k_cuts[d], k_cuts[d + 1]
        for i in range(q_cuts[d], q_cuts[d + 1]):
            hi = end
            if causal:
                hi = min(end, max(end - q_cuts[d + 1] + i + 1, start + max(prefix[d] if prefix else 0, 0)))
            lo = min(max(start, 0), keys)
            want[i] = torch.tensor([lo, min(max(hi, lo), keys)])
    assert torch.equal(got.cpu().long(), want)


@pytest.mark.parametrize("heads,kv_heads,rows,keys", [(56, 56, 51, 14922), (40, 40, 57, 18626), (35, 7, 11, 69694),
                                                      (16, 16, 39, 29920), (40, 8, 28, 116105)])
def test_few_rows_without_ranges(dev, heads, kv_heads, rows, keys):
    """Sizes at which ranges would decide the kernel, and a call that has none: the splits of a call with ranges, in a
    workspace that holds garbage."""
    g = torch.Generator(device=dev).manual_seed(rows)
    q, k, v = make(g, heads, rows, dev), make(g, kv_heads, keys, dev), make(g, kv_heads, keys, dev)
    ws = torch.full((mh.flash_attn_128_workspace_bytes(q, k, v),), 0xff, dtype=torch.uint8, device=dev)
    out = mh.flash_attn_128(q, k, v, workspace=ws)
    for h in (0, heads - 1):
        j = h // (heads // kv_heads)
        check(out[h:h + 1], *attention64(q[h:h + 1], k[j:j + 1], v[j:j + 1]), f"head {h}")


def causal_ranges(rows, keys, dev):
    """The last row on the last key."""
    hi = torch.arange(rows, device=dev) + keys - rows + 1
    return torch.stack([torch.zeros_like(hi), hi], 1).int().contiguous()


@pytest.mark.parametrize("heads,kv_heads,rows,keys", [(2, 2, 100, 100), (8, 2, 30, 300), (1, 1, 20, 9000), (6, 6, 700, 700),
                                                     (40, 8, 300, 333), (16, 16, 40, 30000)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (5.0, False), (0.0, True), (20.0, True)])
def test_no_bit_of_a_row_comes_from_keys_that_its_neighbours_attend(dev, heads, kv_heads, rows, keys, cap, bias):
    """Causal rows, one key poisoned at a time (NaN, infinite, scores past 2^20 and 2^10, values, a far position): the rows
    before it attend the rest of its tile, and are the same bits. Then one query row, and its position."""
    g = torch.Generator(device=dev).manual_seed(rows + keys + heads)
    q, k, v = make(g, heads, rows, dev), make(g, kv_heads, keys, dev), make(g, kv_heads, keys, dev)
    kw = {"ranges": causal_ranges(rows, keys, dev), "cap": cap}
    if bias:
        kw["slopes"] = torch.rand(heads, generator=g, device=dev) * 0.2
        kw["q_pos"] = torch.randint(-50, 50, (rows,), generator=g, device=dev, dtype=torch.int32)
        kw["k_pos"] = torch.randint(-50, 50, (keys,), generator=g, device=dev, dtype=torch.int32)
    clean = mh.flash_attn_128(q, k, v, **kw)
    first = keys - rows
    check(clean[:1], *attention64(q[:1], k[:1], v[:1], **{**kw, **({"slopes": kw["slopes"][:1]} if bias else {})}))
    for row in {1, 5, rows // 3, rows // 2 + 3, rows - 1}:
        for what in (float("nan"), float("inf"), 1e6, 300.0):
            bad = k.clone()
            bad[:, first + row] = torch.where(bad[:, first + row] > 0, what, -what)
            assert torch.equal(mh.flash_attn_128(q, bad, v, **kw)[:, :row], clean[:, :row]), f"key of row {row}: {what}"
        bad = v.clone()
        bad[:, first + row] = float("inf")
        assert torch.equal(mh.flash_attn_128(q, k, bad, **kw)[:, :row], clean[:, :row]), f"value of row {row}"
        others = torch.arange(rows, device=dev) != row
        for what in (float("nan"), 1e6, 300.0):
            bad = q.clone()
            bad[:, row] = what
            assert torch.equal(mh.flash_attn_128(bad, k, v, **kw)[:, others], clean[:, others]), f"row {row}: {what}"
            no_ranges = {**kw, "ranges": None}
            assert torch.equal(mh.flash_attn_128(bad, k, v, **no_ranges)[:, others],
                               mh.flash_attn_128(q, k, v, **no_ranges)[:, others]), f"row {row}: {what}, all keys"
        if bias:
            for what in (1 << 30, -(1 << 31)):
                bad = kw["k_pos"].clone()
                bad[first + row] = what
                assert torch.equal(mh.flash_attn_128(q, k, v, **{**kw, "k_pos": bad})[:, :row], clean[:, :row])
                bad = kw["q_pos"].clone()
                bad[row - 1] = what
                others = torch.arange(rows, device=dev) != row - 1
                assert torch.equal(mh.flash_attn_128(q, k, v, **{**kw, "q_pos": bad})[:, others], clean[:, others])


def test_scores_far_beyond_and_ordinary_ones_in_a_wave(dev):
    """Rows of the first tiles' large scores (past 2^20) beside ordinary rows, in rising and falling order, each against
    float64 and against itself alone."""
    g = torch.Generator(device=dev).manual_seed(5)
    rows, keys = 64, 500
    q, k, v = make(g, 2, rows, dev), make(g, 2, keys, dev), make(g, 2, keys, dev)
    q[:, 1::3] *= 2.0 ** 18
    q[:, 2::3] *= 2.0 ** 9
    for kw in ({}, {"ranges": causal_ranges(rows, keys, dev)}, {"ranges": random_ranges(g, rows, keys, dev)}):
        out = mh.flash_attn_128(q, k, v, **kw)
        for part in (slice(0, None, 3), slice(1, None, 3), slice(2, None, 3)):
            pw = {n: t[part].contiguous() for n, t in kw.items()}
            alone = q.clone()
            alone[:] = q[:, part][:, :1].expand_as(q)   # a call of the same sizes, all rows of one kind
            alone[:, part] = q[:, part]
            assert torch.equal(mh.flash_attn_128(alone, k, v, **kw)[:, part], out[:, part])
            if part.start == 0:
                check(out[:, part], *attention64(q[:, part], k, v, **pw))
