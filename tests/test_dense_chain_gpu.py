"""The dense path of a block as it is run: the 4-bit qkv projection, heads with positions on three axes, attention over
packed clips, the out projection into the residual, fc1 with SwiGLU and fc2 into a float residual; and a stream that keeps
its keys and values and takes one row at a time. Every step is checked against float64 of what the step before left, within
the bounds of that operator's own tests, and the run captured in a graph gives the eager bits."""
import pytest
import torch

import mako_h3 as mh
from test_attn_dense_gpu import attention64, check as check_attention
from test_mx4_gpu import check_quant, products
from test_rotary_gpu import heads64

pytestmark = pytest.mark.gpu

PAIRS, HEADS, DIM, FFN = (16, 16, 16), 4, 512, 768


def weights(g, dev):
    def mx4(n, k):
        return mh.quant_rows_mx4((torch.randn((n, k), generator=g, device=dev) / k ** 0.5).to(torch.bfloat16))
    return {"qkv": mx4(3 * HEADS * 128, DIM), "out": mx4(DIM, HEADS * 128), "fc1": mx4(2 * FFN, DIM), "fc2": mx4(DIM, FFN),
            "q_w": 1 + 0.1 * torch.randn(128, generator=g, device=dev),
            "k_w": 1 + 0.1 * torch.randn(128, generator=g, device=dev),
            "gate": 0.5 + 0.1 * torch.randn((1, DIM), generator=g, device=dev)}


def positions(lengths, dev):
    """Clips on a grid 5 wide and 4 high, each from its own first frame."""
    at = torch.cat([torch.arange(n) for n in lengths])
    return torch.stack([at // 20, at // 5 % 4, at % 5], 1).int().to(dev)


def block(w, x, pos, ranges):
    """One pass; returns every step's result."""
    t = {}
    t["xq"] = mh.quant_rows_mx4(x)
    t["qkv"] = mh.gemm_mx4(*t["xq"], *w["qkv"])
    t["q"], t["k"], t["v"] = mh.heads_partial_axes(t["qkv"], HEADS, pos, PAIRS, w["q_w"], w["k_w"])
    t["att"] = mh.flash_attn_128(t["q"], t["k"], t["v"], ranges=ranges, out_layout="rows")
    t["aq"] = mh.quant_rows_mx4(t["att"])
    t["x1"] = mh.gemm_mx4_gate_add(*t["aq"], *w["out"], x.clone(), w["gate"])
    t["hq"] = mh.quant_rows_mx4(t["x1"])
    t["h"] = mh.gemm_mx4_swiglu(*t["hq"], *w["fc1"])
    t["fq"] = mh.quant_rows_mx4(t["h"])
    t["x2"] = mh.gemm_mx4_gate_add(*t["fq"], *w["fc2"], t["x1"].float(), w["gate"])
    return t


def inputs(lengths, seed, dev, causal):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = sum(lengths)
    off = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=dev)
    return (weights(g, dev), torch.randn((n, DIM), generator=g, device=dev).to(torch.bfloat16), positions(lengths, dev),
            mh.attn_ranges(off, off, n, n, causal=causal))


def check_heads(w, qkv, pos, q, k, v):
    want = heads64(qkv, HEADS, pos, PAIRS, (10000.0,) * 3, (1.0,) * 3, w["q_w"], w["k_w"], 1e-6)
    for got, y in zip((q, k, v), want):
        err = (got.transpose(0, 1).double() - y).abs()
        assert bool((err <= 2.0 ** -8 * y.abs() + 2e-5 * y.abs().amax(-1, keepdim=True)).all())


@pytest.mark.parametrize("lengths,causal", [([1], False), ([40, 3, 100], False), ([300, 217], True)])
def test_every_step_of_a_block(dev, lengths, causal):
    w, x, pos, ranges = inputs(lengths, sum(lengths), dev, causal)
    t = block(w, x, pos, ranges)
    for m in (x, t["att"], t["x1"], t["h"]):
        check_quant(m)
    y, tol = products(t["xq"], w["qkv"], DIM)
    assert bool(((t["qkv"].double() - y).abs() <= 2.0 ** -8 * y.abs() + tol).all())
    check_heads(w, t["qkv"], pos, t["q"], t["k"], t["v"])
    want, mag = attention64(t["q"], t["k"], t["v"], ranges=ranges)
    rows = lambda a: a.transpose(0, 1).reshape(len(x), HEADS * 128)  # noqa: E731
    check_attention(t["att"], rows(want), rows(mag))
    gate = w["gate"].double()
    y, tol = products(t["aq"], w["out"], HEADS * 128)
    want = x.double() + gate * y
    assert bool(((t["x1"].double() - want).abs() <= 2.0 ** -8 * want.abs() + gate.abs() * (tol + 2.0 ** -24 * y.abs())).all())
    y, tol = products(t["hq"], w["fc1"], DIM)
    a, u, ta, tu = y[:, :FFN], y[:, FFN:], tol[:, :FFN], tol[:, FFN:]
    want = a * torch.sigmoid(a) * u
    slack = 1.1 * ta * (u.abs() + tu) + (a * torch.sigmoid(a)).abs() * tu + 2.0 ** -21 * (1 + a.abs()) * want.abs()
    assert bool(((t["h"].double() - want).abs() <= 2.0 ** -8 * want.abs() + slack).all())
    y, tol = products(t["fq"], w["fc2"], FFN)
    want = t["x1"].double() + gate * y
    assert bool(((t["x2"].double() - want).abs() <= 2.0 ** -23 * want.abs() + gate.abs() * (tol + 2.0 ** -24 * y.abs())).all())


def test_the_block_in_a_graph(dev):
    w, x, pos, ranges = inputs([70, 130], 7, dev, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(w, x, pos, ranges)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = block(w, x, pos, ranges)
    g = torch.Generator(device=dev).manual_seed(8)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device=dev))
        graph.replay()
        want = block(w, x, pos, ranges)
        torch.cuda.synchronize()
        assert torch.equal(t["x2"], want["x2"]) and torch.equal(t["att"], want["att"])


def test_a_stream_row_by_row(dev):
    """A stream's first rows at once, then one row at a time against the kept keys and values."""
    w, x, pos, _ = inputs([150], 9, dev, True)
    n, first = len(x), 140
    keys, values = (torch.full((HEADS, n, 128), float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2))
    start = 0
    while start < n:
        end = first if start == 0 else start + 1
        xq = mh.quant_rows_mx4(x[start:end].contiguous())
        qkv = mh.gemm_mx4(*xq, *w["qkv"])
        y, tol = products(xq, w["qkv"], DIM)
        assert bool(((qkv.double() - y).abs() <= 2.0 ** -8 * y.abs() + tol).all())
        here = pos[start:end].contiguous()
        q, k, v = mh.heads_partial_axes(qkv, HEADS, here, PAIRS, w["q_w"], w["k_w"])
        check_heads(w, qkv, here, q, k, v)
        keys[:, start:end], values[:, start:end] = k, v
        off = [torch.tensor([0, m], dtype=torch.int32, device=dev) for m in (end - start, end)]
        r = mh.attn_ranges(*off, end - start, end, causal=True)
        got = mh.flash_attn_128(q, keys, values, ranges=r)  # rows behind `end` hold NaN
        check_attention(got, *attention64(q, keys[:, :end], values[:, :end], ranges=r))
        start = end
