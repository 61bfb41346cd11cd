"""quant_rows_mx4 against the nearest of the eight magnitudes in float64 (exact, every bf16 pattern among the inputs), and
gemm_mx4 with its epilogues against float64 products of the values that the operands stand for.

A product's bound: its rounding (2^-8 of a bf16 result), and for its float accumulation (k / 128 + 16) 2^-22 of the sum of
its terms' magnitudes: one addition to the accumulator an MFMA of 128 k, and some 16 inside one, each off by at most 2^-23
of that sum, doubled for truncation."""
import numpy as np
import pytest
import torch

import mako_h3 as mh

pytestmark = pytest.mark.gpu

MAGS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def values(q, scale):
    """Float64 values of a matrix in its 4-bit form (scale byte 255: NaN)."""
    rows = q.shape[0]
    table = torch.tensor(MAGS + [-m for m in MAGS], dtype=torch.float64, device=q.device)
    v = table[torch.stack([q & 15, q >> 4], -1).long()].view(rows, -1, 32)
    e = scale.transpose(0, 1).reshape(rows, -1, 1).double()
    v = v * torch.exp2(e - 127)
    return torch.where(e == 255, float("nan"), v).view(rows, -1)


def quantized64(w):
    """(values, scale bytes [rows][blocks]) by the definition, in float64."""
    rows = w.shape[0]
    b = w.double().view(rows, -1, 32)
    top = b.abs().amax(-1)
    # floor(log2) by comparison with the powers themselves
    powers = torch.exp2(torch.arange(-149, 128, dtype=torch.float64, device=w.device))
    e = torch.searchsorted(powers, top.nan_to_num(posinf=1.0), right=True).double() - 1 - 149
    e = torch.where(top > 0, (e - 2).clamp_min(-127), -127.0)
    a = b.abs() / torch.exp2(e)[..., None]
    mags = torch.tensor(MAGS, dtype=torch.float64, device=w.device)
    mids = (mags[1:] + mags[:-1]) / 2
    lo, hi = torch.searchsorted(mids, a.contiguous()), torch.searchsorted(mids, a.contiguous(), right=True)
    v = torch.sign(b) * mags[torch.where(lo % 2 == 0, lo, hi)] * torch.exp2(e)[..., None]
    bad = ~torch.isfinite(b).all(-1)
    return torch.where(bad[..., None], float("nan"), v).view(rows, -1), torch.where(bad, 255.0, e + 127)


def check_quant(w):
    q, s = mh.quant_rows_mx4(w)
    want, byte = quantized64(w)
    assert torch.equal(s.transpose(0, 1).reshape(w.shape[0], -1).double(), byte)
    got = values(q, s)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 256), (3, 512), (945, 5376), (67, 13824), (2985, 256)])
def test_quant_matches_the_definition(dev, rows, cols, dtype):
    g = torch.Generator(device=dev).manual_seed(rows + cols)
    w = torch.randn((rows, cols), generator=g, device=dev) * torch.exp2(
        torch.randint(-20, 20, (rows, cols // 32), generator=g, device=dev).float()).repeat_interleave(32, 1)
    check_quant(w.to(dtype))


def test_quant_of_every_bf16_pattern(dev):
    """All 65,536 patterns: sorted by magnitude 32 to a block (neighbours share a block: all codes, ties, subnormals,
    infinities and NaN), and each against a block maximum of 1 .. 8 times a power of two above it."""
    bits = torch.arange(65536, device=dev)
    by_size = bits[torch.argsort(bits & 0x7fff, stable=True)].to(torch.int32)
    bf16 = lambda t: (t << 16).view(torch.float32).to(torch.bfloat16)  # noqa: E731
    check_quant(bf16(by_size).view(256, 256))
    for up in (1, 2, 3):
        w = bf16(by_size).view(-1, 16)
        top = ((((by_size.view(-1, 16).amax(1) & 0x7fff) >> 7) + up).clamp(max=254) << 7).to(torch.int32)
        w = torch.cat([w, bf16(top)[:, None].expand(-1, 16)], 1)
        check_quant(w.reshape(-1, 256).contiguous())


def test_quant_of_zero_and_nonfinite_blocks(dev):
    w = torch.zeros((4, 512), device=dev)
    w[1, 40] = float("inf")
    w[2, 100] = float("nan")
    w[3, 0], w[3, 32] = 1e-45, -3.4e38
    check_quant(w)
    q, s = mh.quant_rows_mx4(w.to(torch.bfloat16))
    assert int(q[0].max()) == 0 and int(s[:, 0].max()) == 0


def operand(g, rows, k, dev, scale=1.0):
    return mh.quant_rows_mx4((torch.randn((rows, k), generator=g, device=dev) * scale).to(torch.bfloat16))


def products(x, w, k):
    """y and the bound of its accumulation, float64."""
    xv, wv = values(*x), values(*w)
    y = xv @ wv.T.contiguous()
    return y, (k / 128 + 16) * 2.0 ** -22 * (xv.abs() @ wv.abs().T.contiguous())


SHAPES = [(1, 256, 256), (3, 256, 512), (16, 512, 768), (17, 256, 5120), (64, 512, 1024), (65, 1280, 256), (128, 256, 2560),
          (200, 768, 1536), (256, 512, 512), (257, 256, 13824), (945, 1536, 5376), (1500, 2048, 768), (3000, 5120, 512)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm_store(dev, m, n, k):
    g = torch.Generator(device=dev).manual_seed(m + n + k)
    x, w = operand(g, m, k, dev), operand(g, n, k, dev, 0.02)
    out = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device=dev)
    mh.gemm_mx4(*x, *w, out=out)
    y, tol = products(x, w, k)
    assert bool(((out.double() - y).abs() <= 2.0 ** -8 * y.abs() + tol).all())


@pytest.mark.parametrize("m,n,k", [(1, 128, 256), (5, 256, 1024), (33, 128, 5120), (100, 384, 512), (257, 1152, 768),
                                   (945, 1024, 1280), (2100, 2048, 256)])
def test_gemm_swiglu(dev, m, n, k):
    g = torch.Generator(device=dev).manual_seed(m * n + k)
    x, w = operand(g, m, k, dev), operand(g, 2 * n, k, dev, 1.5 / k ** 0.5)
    out = mh.gemm_mx4_swiglu(*x, *w)
    y, tol = products(x, w, k)
    a, u, ta, tu = y[:, :n], y[:, n:], tol[:, :n], tol[:, n:]
    silu = a * torch.sigmoid(a)
    want = silu * u
    # |d silu| <= 1.1; the exponential and the reciprocal are within 2^-22 of theirs, scaled by the argument's size.
    slack = 1.1 * ta * (u.abs() + tu) + silu.abs() * tu + 2.0 ** -21 * (1 + a.abs()) * want.abs()
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + slack).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k,sets", [(1, 256, 512, 1), (3, 5120, 1024, 3), (20, 256, 256, 2), (100, 512, 768, 1),
                                        (300, 768, 1280, 3), (945, 5376, 512, 2)])
def test_gemm_gate_add(dev, m, n, k, sets, dtype):
    g = torch.Generator(device=dev).manual_seed(m + n * k)
    x, w = operand(g, m, k, dev), operand(g, n, k, dev, 0.05)
    residual = torch.randn((m, n), generator=g, device=dev).to(dtype)
    table = 0.5 * torch.randn((sets, 6, n), generator=g, device=dev)
    which = torch.randint(0, sets + 2, (m,), generator=g, device=dev, dtype=torch.uint8) if sets > 1 else None
    got = mh.gemm_mx4_gate_add(*x, *w, residual.clone(), table[:, 2], set_of_row=which, n_sets=sets)
    y, tol = products(x, w, k)
    gate = table[which.long().clamp(max=sets - 1), 2].double() if which is not None else table[:1, 2].double()
    want = residual.double() + gate * y
    # A float residual rounds twice (the product's sum, the addition), at most 2^-24 of each.
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    assert bool(((got.double() - want).abs() <= unit * want.abs() + gate.abs() * (tol + 2.0 ** -24 * y.abs())).all())


@pytest.mark.parametrize("m,n", [(1, 20480), (32, 16384), (33, 16384), (33, 20480), (63, 512), (300, 10240), (383, 10240), (577, 16384),
                                 (769, 16384), (1024, 16384), (1025, 512)])
def test_every_kernel_with_every_epilogue(dev, m, n):
    """Sizes that take each of the kernels (few rows, tiles of 64, 128, 192 and 256 rows), with whole and cut tiles."""
    g = torch.Generator(device=dev).manual_seed(m + n)
    for k in (256, 768):
        x, w = operand(g, m, k, dev), operand(g, n, k, dev, 1.5 / k ** 0.5)
        y, tol = products(x, w, k)
        out = mh.gemm_mx4(*x, *w)
        assert bool(((out.double() - y).abs() <= 2.0 ** -8 * y.abs() + tol).all())
        res = torch.randn((m, n), generator=g, device=dev)
        gate = torch.randn(n, generator=g, device=dev)
        want = res.double() + gate.double() * y
        got = mh.gemm_mx4_gate_add(*x, *w, res, gate[None])
        assert got is res
        slack = gate.double().abs() * (tol + 2.0 ** -24 * y.abs())
        assert bool(((got.double() - want).abs() <= 2.0 ** -23 * want.abs() + slack).all())
        h = n // 2
        out = mh.gemm_mx4_swiglu(*x, *w)
        a, u, ta, tu = y[:, :h], y[:, h:], tol[:, :h], tol[:, h:]
        want = a * torch.sigmoid(a) * u
        slack = 1.1 * ta * (u.abs() + tu) + (a * torch.sigmoid(a)).abs() * tu + 2.0 ** -21 * (1 + a.abs()) * want.abs()
        assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + slack).all())


def test_nan_scales_stay_in_their_rows_and_columns(dev):
    """A block of scale 255 makes its row of x (its row of w) NaN and nothing else."""
    g = torch.Generator(device=dev).manual_seed(5)
    m, n, k = 70, 512, 768
    for rows in (m, 5):
        x, w = operand(g, rows, k, dev), operand(g, n, k, dev)
        y = mh.gemm_mx4(*x, *w)
        x[1][1, 3, 5], w[1][2, 300, 0] = 255, 255
        z = mh.gemm_mx4(*x, *w)
        bad = torch.zeros((rows, n), dtype=torch.bool, device=dev)
        bad[3], bad[:, 300] = True, True
        assert torch.equal(torch.isnan(z), bad)
        assert torch.equal(z[~bad], y[~bad])


@pytest.mark.parametrize("m", [2, 40, 300])
def test_extreme_scales(dev, m):
    """Exponents at both ends whose products are ordinary numbers, and a zero block of the least exponent."""
    g = torch.Generator(device=dev).manual_seed(m)
    n, k = 256, 512
    x, w = operand(g, m, k, dev), operand(g, n, k, dev)
    x[1][:], w[1][:] = 127 + 100, 127 - 100
    x[1][:, 0], x[0][0] = 0, 0
    y, tol = products(x, w, k)
    out = mh.gemm_mx4(*x, *w)
    assert bool(((out.double() - y).abs() <= 2.0 ** -8 * y.abs() + tol).all())


def test_rows_do_not_depend_on_the_batch(dev):
    """A row's product in any batch of one tile variant is the same bits; all variants agree within the bound."""
    g = torch.Generator(device=dev).manual_seed(9)
    n, k = 512, 2560
    x, w = operand(g, 600, k, dev), operand(g, n, k, dev, 0.02)
    full = mh.gemm_mx4(*x, *w).double()
    y, tol = products(x, w, k)
    for m in (1, 2, 8, 16, 17, 32, 33, 64, 100, 192, 300, 512):
        part = mh.gemm_mx4(x[0][:m], x[1][:, :m].contiguous(), *w).double()
        assert bool(((part - full[:m]).abs() <= 2.0 ** -7 * y[:m].abs() + 2 * tol[:m]).all())


def test_replayed_from_a_graph(dev):
    g = torch.Generator(device=dev).manual_seed(11)
    w = operand(g, 512, 768, dev, 0.02)
    src = torch.randn((130, 768), generator=g, device=dev).to(torch.bfloat16)
    few = src[:4].clone()
    run = lambda: (mh.gemm_mx4(*mh.quant_rows_mx4(src), *w), mh.gemm_mx4(*mh.quant_rows_mx4(few), *w))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(3):
        src.copy_(torch.randn((130, 768), generator=g, device=dev))
        few.copy_(src[7:11])
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def tile_of_sizes(m, w_rows, k):
    """The kernel that a product's sizes take (the rule of gemm_mx4.hip, in float as there)."""
    f = np.float32
    tiles = (("256x256", 256, 256, 1.65), ("192x256", 192, 256, 1.5), ("128x128", 128, 128, 0.71), ("64x128", 64, 128, 0.48),
             ("64x64", 64, 64, 0.35))
    w_us, best, least = f(w_rows) * f(k) * f(0.53125 / 6.2e6), None, f(np.inf)
    for name, rows, cols, step in tiles:
        rounds = (-(-m // rows) * (w_rows // cols) + 255) // 256
        us = f(4) + max(f(rounds) * f(k // 256) * f(step), w_us)
        if us < least:
            best, least = name, us
    few = f(4) + w_us + f(w_rows // 32) * f(m) * f(k) * f(0.35 / 6.2e6)
    return ("few 16" if m <= 16 else "few 32") if m <= 32 and few <= least else best


LONG = [("few 16", 5, 512), ("few 16", 16, 1024), ("few 32", 17, 512), ("few 32", 32, 2048), ("64x64", 65, 512),
        ("64x64", 129, 512), ("64x128", 129, 8192), ("64x128", 300, 4096), ("128x128", 385, 5120), ("128x128", 700, 3328),
        ("192x256", 769, 10240), ("192x256", 2100, 4096), ("256x256", 769, 16384), ("256x256", 3000, 5120)]


@pytest.mark.parametrize("k", [2560, 2816])
@pytest.mark.parametrize("kernel,m,n", LONG)
def test_every_kernel_over_many_steps_with_every_epilogue(dev, kernel, m, n, k):
    """Ten and eleven K-steps of 256, several times round every kernel's ring of stages, with cut row tiles and all four
    epilogues."""
    assert tile_of_sizes(m, n, k) == kernel
    g = torch.Generator(device=dev).manual_seed(m + n + k)
    x, w = operand(g, m, k, dev), operand(g, n, k, dev, 1.5 / k ** 0.5)
    y, tol = products(x, w, k)
    out = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device=dev)
    mh.gemm_mx4(*x, *w, out=out)
    assert bool(((out.double() - y).abs() <= 2.0 ** -8 * y.abs() + tol).all())
    table, which = 0.5 * torch.randn((3, n), generator=g, device=dev), torch.randint(0, 3, (m,), generator=g, device=dev).byte()
    gate = table[which.long()].double()
    slack = gate.abs() * (tol + 2.0 ** -24 * y.abs())
    for dtype, unit in ((torch.bfloat16, 2.0 ** -8), (torch.float32, 2.0 ** -23)):
        res = torch.randn((m, n), generator=g, device=dev).to(dtype)
        want = res.double() + gate * y
        got = mh.gemm_mx4_gate_add(*x, *w, res, table, set_of_row=which, n_sets=3)
        assert bool(((got.double() - want).abs() <= unit * want.abs() + slack).all())
    h = n // 2
    out = torch.full((m, h), float("nan"), dtype=torch.bfloat16, device=dev)
    mh.gemm_mx4_swiglu(*x, *w, out=out)
    a, u, ta, tu = y[:, :h], y[:, h:], tol[:, :h], tol[:, h:]
    want = a * torch.sigmoid(a) * u
    slack = 1.1 * ta * (u.abs() + tu) + (a * torch.sigmoid(a)).abs() * tu + 2.0 ** -21 * (1 + a.abs()) * want.abs()
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + slack).all())


@pytest.mark.parametrize("kernel,n,sizes", [("few 16", 512, (16, 1, 7)), ("few 32", 512, (32, 17)), ("64x64", 512, (130, 33, 65)),
                                            ("64x128", 10240, (129, 65)), ("128x128", 5120, (500, 385)),
                                            ("192x256", 4096, (3000, 2100)), ("256x256", 16384, (900, 769))])
def test_a_row_is_the_same_bits_in_any_batch_of_its_kernel(dev, kernel, n, sizes):
    """Of fewer rows, and at another place among them."""
    k = 2304
    g = torch.Generator(device=dev).manual_seed(n)
    x, w = operand(g, sizes[0], k, dev), operand(g, n, k, dev, 0.02)
    full = mh.gemm_mx4(*x, *w)
    for m in sizes:
        assert tile_of_sizes(m, n, k) == kernel
        assert torch.equal(mh.gemm_mx4(x[0][:m], x[1][:, :m].contiguous(), *w), full[:m])
        for by in (1, m // 2):
            got = mh.gemm_mx4(x[0][:m].roll(by, 0), x[1][:, :m].contiguous().roll(by, 1), *w)
            assert torch.equal(got.roll(-by, 0), full[:m])


def test_first_rows_with_all_rows_scales_of_256_columns(dev):
    """One run of scales a matrix: the first rows' lead it. Of more columns the binding refuses the same call."""
    g = torch.Generator(device=dev).manual_seed(12)
    for k in (256, 512):
        x, w = operand(g, 90, k, dev), operand(g, 512, k, dev)
        if k == 256:
            assert torch.equal(mh.gemm_mx4(x[0][:70], x[1], *w), mh.gemm_mx4(x[0][:70], x[1][:, :70].contiguous(), *w))
        else:
            with pytest.raises(ValueError, match="x_scale"):
                mh.gemm_mx4(x[0][:70], x[1], *w)
