"""rotary_axes against angles of 45 decimal digits, and heads_partial_axes against rotary_axes + heads_partial (bit for
bit) and a float64 restatement.

The tables' bound, 1e-7: the polynomials are cut below 2e-9, and a result below 1 takes at most two roundings of half a
step of [1/2, 1) (2^-25 each) and what its last polynomial term adds (2^-26)."""
import math
from decimal import Decimal, getcontext

import numpy as np
import pytest
import torch

import mako_h3 as mh
from helpers import from_bits, randn_bf16_bits

pytestmark = pytest.mark.gpu

PI = Decimal("3.14159265358979323846264338327950288419716939937510582")


def exact_tables(pos, pairs, theta, step):
    """Float64 cos and sin of the angles, reduced modulo a turn in decimal."""
    getcontext().prec = 45
    angles = []
    for a, n in enumerate(pairs):
        for j in range(n):
            f = Decimal(step[a]) * (-(Decimal(theta[a]).ln()) * j / n).exp()
            angles.append([float((Decimal(int(p)) * f) % (2 * PI)) for p in pos[:, a]])
    ang = np.array(angles).reshape(sum(pairs), len(pos)).T
    return np.cos(ang), np.sin(ang)


FAR = [0, 1, -1, 2, 7, 511, 4095, 65535, 1 << 24, (1 << 24) + 1, -123456789, (1 << 31) - 1, -(1 << 31)]


@pytest.mark.parametrize("pairs,theta,step", [
    ((16, 16, 16), (10000.0, 10000.0, 10000.0), (0.25, 1.0, 1.0)),
    ((48,), (10000.0,), (1.0,)),
    ((1,), (1.0,), (2 * math.pi / 8,)),
    ((8, 0, 24, 32), (500000.0, 7.0, 10000.0, 256.0), (1.0, 1.0, -0.5, 1 / 3)),
    ((22, 42), (1e6, 1e4), (0.1, 6.0)),
])
def test_tables_at_near_and_far_positions(dev, pairs, theta, step):
    rng = np.random.default_rng(len(pairs))
    pos = np.array([[FAR[(i + 3 * a) % len(FAR)] for a in range(len(pairs))] for i in range(len(FAR))] +
                   [[int(rng.integers(-3000, 3000)) for _ in pairs] for _ in range(20)], dtype=np.int64)
    cos, sin = mh.rotary_axes(torch.from_numpy(pos.astype(np.int32)).to(dev), pairs, theta=theta, step=step)
    want_c, want_s = exact_tables(pos, pairs, theta, step)
    for got, want in ((cos, want_c), (sin, want_s)):
        assert np.abs(got.cpu().numpy().astype(np.float64) - want).max() <= 1e-7


def test_eighths_of_a_turn_are_exact_where_a_float_is(dev):
    pos = torch.arange(-16, 17, dtype=torch.int32, device=dev).view(-1, 1)
    cos, sin = mh.rotary_axes(pos, (1,), theta=1.0, step=math.pi / 2)
    # A step of pi / 2 as a double is a quarter of a turn less 2^-55 or so.
    assert np.array_equal(cos.cpu().numpy().ravel().round(6) + 0.0, [(1.0, 0.0, -1.0, 0.0)[i % 4] for i in range(-16, 17)])
    assert np.array_equal(sin.cpu().numpy().ravel().round(6) + 0.0, [(0.0, 1.0, 0.0, -1.0)[i % 4] for i in range(-16, 17)])


@pytest.mark.parametrize("rows", [1, 5, 212, 945, 70001])
def test_table_rows_and_one_axis_split_in_three(dev, rows):
    """Every row is written, and axes that share their positions and frequencies give what one axis gives."""
    p = torch.randint(-5000, 5000, (rows, 1), dtype=torch.int32, device=dev)
    cos, sin = (torch.full((rows, 24), float("nan"), device=dev) for _ in range(2))
    mh.rotary_axes(p.expand(rows, 3).contiguous(), (8, 8, 8), cos=cos, sin=sin)
    one = mh.rotary_axes(p, (8,))
    for t, o in ((cos, one[0]), (sin, one[1])):
        for a in range(3):
            assert torch.equal(t[:, 8 * a:8 * a + 8], o)


def heads64(qkv, heads, pos, pairs, theta, step, q_w, k_w, eps):
    rows, half = qkv.shape[0], sum(pairs)
    cos, sin = (torch.from_numpy(t).to(qkv.device)[:, None]
                for t in exact_tables(pos.cpu().numpy().astype(np.int64), pairs, theta, step))
    x = qkv[:, :3 * heads * 128].double().view(rows, 3, heads, 128)
    out = []
    for i, w in ((0, q_w), (1, k_w)):
        y = x[:, i] * torch.rsqrt(x[:, i].square().mean(-1, keepdim=True) + eps)
        y = y if w is None else y * w.double()
        a, b = y[..., :half].clone(), y[..., half:2 * half].clone()
        y[..., :half], y[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
        out.append(y)
    return out + [x[:, 2]]


@pytest.mark.parametrize("rows,heads,pairs,weights,with_v,layout,gather", [
    (1, 1, (16, 16, 16), True, True, "heads", False),
    (1, 56, (16, 16, 16), True, True, "rows", False),
    (33, 3, (8,), False, False, "heads", False),
    (130, 5, (24, 20, 20), True, True, "rows", True),
    (67, 40, (16, 16, 16), True, True, "heads", True),
    (212, 2, (4, 4, 0, 8), False, True, "rows", False),
])
def test_heads_partial_axes(dev, rows, heads, pairs, weights, with_v, layout, gather):
    rng = np.random.default_rng(rows + heads)
    theta, step = [10000.0, 500.0, 10000.0, 300.0][:len(pairs)], [0.25, 1.0, 1.0, 0.5][:len(pairs)]
    qkv = from_bits(randn_bf16_bits(rng, (rows, 3 * heads * 128 + 24), 1.5), dev)
    q_w, k_w = (torch.from_numpy((1 + 0.1 * rng.standard_normal(128)).astype(np.float32)).to(dev) if weights else None
                for _ in range(2))
    pos = torch.from_numpy(rng.integers(-2000, 100000, (rows, len(pairs))).astype(np.int32)).to(dev)
    index = None
    if gather:
        index = torch.from_numpy(rng.integers(-2, rows + 2, rows + 9).astype(np.int32)).to(dev)
    kw = dict(map=index, with_v=with_v, layout=layout)
    got = mh.heads_partial_axes(qkv, heads, pos, pairs, q_w, k_w, theta=theta, step=step, **kw)
    tables = mh.rotary_axes(pos, pairs, theta=theta, step=step)
    two = mh.heads_partial(qkv, heads, q_w, k_w, *tables, rot=2 * sum(pairs), **kw)
    for g, t in zip(got, two):
        assert (g is None) == (t is None) and (g is None or torch.equal(g, t))
    want = heads64(qkv, heads, pos, pairs, theta, step, q_w, k_w, 1e-6)
    src = torch.arange(rows, device=dev) if index is None else index.long()
    real = (src >= 0) & (src < rows)
    for g, w in zip(got, want):
        if g is None:
            continue
        g = (g.transpose(0, 1) if layout == "heads" else g.view(-1, heads, 128)).double()
        w = torch.where(real[:, None, None], w[src.clamp(0, rows - 1)], 0.0)
        # One rounding to bf16, and float sums of 128 squares (128 of 2^-24) at the row's scale.
        assert bool(((g - w).abs() <= 2.0 ** -8 * w.abs() + 2e-5 * w.abs().amax(-1, keepdim=True)).all())


def test_in_place_and_no_rotary(dev):
    rng = np.random.default_rng(3)
    qkv = from_bits(randn_bf16_bits(rng, (45, 3 * 4 * 128)), dev)
    pos = torch.randint(0, 50, (45, 3), dtype=torch.int32, device=dev)
    want = mh.heads_partial_axes(qkv, 4, pos, (16, 16, 16), layout="rows")
    none = mh.heads_partial_axes(qkv, 4, pos[:, :1].contiguous(), (0,), layout="rows")
    for a, b in zip(none, mh.heads_partial(qkv, 4, rot=0, layout="rows")):
        assert torch.equal(a, b)
    import ctypes as C
    a, ax = mh.HeadsArgs(), mh.AxesArgs()
    a.rows = a.model_rows = 45
    a.heads, a.head_dim, a.rot, a.eps, a.qkv_stride, a.out_head_stride, a.out_row_stride = 4, 128, 96, 1e-6, 1536, 128, 1536
    ax.axes = 3
    for i in range(3):
        ax.pairs[i], ax.theta[i], ax.step[i] = 16, 10000.0, 1.0
    p = qkv.data_ptr()
    assert mh.lib.mh3_heads_partial_axes(C.byref(a), C.byref(ax), p, None, None, pos.data_ptr(), None, p, p + 1024,
                                         p + 2048, torch.cuda.current_stream().cuda_stream) == mh.OK
    assert torch.equal(qkv, torch.cat(want, 1))
