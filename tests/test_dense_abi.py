"""Refusals of the dense path's entry points (rotary positions with several axes, attention over whole rows, 4-bit
microscaled products) through the C-ABI and through the Python binding. No call here reaches a kernel."""
import ctypes as C

import pytest
import torch

import mako_h3 as mh

FAKE = C.c_void_p(0x1000)  # aligned; never dereferenced: every call below fails validation first
ODD16 = C.c_void_p(0x1008)
ODD4 = C.c_void_p(0x1002)


def at(i):
    """Distinct aligned addresses, 16 GB apart."""
    return C.c_void_p(i << 34)


def axes(**kw):
    a = mh.AxesArgs()
    a.axes = 3
    for i, n in enumerate((16, 16, 16)):
        a.pairs[i], a.theta[i], a.step[i] = n, 10000.0, 1.0
    for k, v in kw.items():
        if isinstance(v, dict):
            for i, x in v.items():
                getattr(a, k)[i] = x
        else:
            setattr(a, k, v)
    return a


BAD_AXES = [{"axes": 0}, {"axes": 5}, {"axes": 2}, {"pairs": {3: 1}}, {"pairs": {0: 65}}, {"pairs": {0: 40}},
            {"pairs": {1: 0xffffffff}}, {"theta": {0: 0.5}}, {"theta": {0: float("nan")}}, {"theta": {2: float("inf")}},
            {"step": {0: float("nan")}}, {"step": {1: 1.1e6}}, {"step": {1: float("-inf")}}]


@pytest.mark.parametrize("kw", BAD_AXES)
def test_axes_domain(kw):
    assert mh.lib.mh3_rotary_axes(C.byref(axes(**kw)), 4, FAKE, at(1), at(2), None) == mh.ERR_PARAM
    h = heads()
    assert mh.lib.mh3_heads_partial_axes(C.byref(h), C.byref(axes(**kw)), at(1), None, None, at(2), None, at(3), at(4),
                                         at(5), None) == mh.ERR_PARAM


def test_rotary_axes_pointers():
    f, a = mh.lib.mh3_rotary_axes, axes()
    assert f(None, 4, FAKE, at(1), at(2), None) == mh.ERR_POINTER
    for i in range(3):
        p = [at(1), at(2), at(3)]
        p[i] = None
        assert f(C.byref(a), 4, *p, None) == mh.ERR_POINTER
        p[i] = ODD4
        assert f(C.byref(a), 4, *p, None) == mh.ERR_ALIGN
    assert f(C.byref(a), 4, at(1), at(1), at(3), None) == mh.ERR_PARAM
    assert f(C.byref(a), 4, at(1), at(2), C.c_void_p(at(2).value + 4 * 48 * 4 - 4), None) == mh.ERR_PARAM
    assert f(C.byref(a), 1 << 31, at(1), at(2), at(3), None) == mh.ERR_SHAPE
    assert f(C.byref(a), 0, None, None, None, None) == mh.OK
    assert f(C.byref(axes(pairs={0: 0, 1: 0, 2: 0})), 4, None, None, None, None) == mh.OK


def heads(**kw):
    a = mh.HeadsArgs()
    a.rows = a.model_rows = 5
    a.heads, a.head_dim, a.rot, a.eps, a.qkv_stride = 2, 128, 96, 1e-6, 768
    a.out_head_stride, a.out_row_stride = 640, 128
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_heads_partial_axes():
    f = mh.lib.mh3_heads_partial_axes
    ax = axes()

    def call(h, a=ax, qkv=at(1), pos=at(2), q=at(3), k=at(4), v=at(5), mp=None):
        return f(None if h is None else C.byref(h), None if a is None else C.byref(a), qkv, None, None, pos, mp, q, k, v,
                 None)

    assert call(None) == mh.ERR_POINTER
    assert call(heads(), a=None) == mh.ERR_POINTER
    assert call(heads(rot=80)) == mh.ERR_PARAM         # the axes hold 48 pairs
    assert call(heads(rot=136)) == mh.ERR_PARAM
    assert call(heads(rot=8)) == mh.ERR_PARAM
    assert call(heads(head_dim=64)) == mh.ERR_UNSUPPORTED
    assert call(heads(eps=0.0)) == mh.ERR_PARAM
    assert call(heads(), pos=None) == mh.ERR_POINTER
    assert call(heads(), pos=ODD4) == mh.ERR_ALIGN
    assert call(heads(), qkv=None) == mh.ERR_POINTER
    assert call(heads(), q=C.c_void_p(at(3).value + 8)) == mh.ERR_ALIGN
    assert call(heads(), q=at(2)) == mh.ERR_PARAM      # q over the positions
    assert call(heads(rows=0), q=None, k=None) in (mh.OK, mh.ERR_POINTER)


def dense(**kw):
    a = mh.DenseAttnArgs(8, 2, 128, 100, 200, 0.0, 0.0, 0, 100 * 128, 128, 200 * 128, 128, 200 * 128, 128, 100 * 128, 128)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


DENSE_BAD = [({"heads": 0}, mh.ERR_SHAPE), ({"kv_heads": 0}, mh.ERR_SHAPE), ({"kv_heads": 3}, mh.ERR_SHAPE),
             ({"kv_heads": 16}, mh.ERR_SHAPE), ({"head_dim": 0}, mh.ERR_SHAPE), ({"head_dim": 64}, mh.ERR_UNSUPPORTED),
             ({"scale": -1.0}, mh.ERR_PARAM), ({"scale": float("nan")}, mh.ERR_PARAM),
             ({"scale": float("inf")}, mh.ERR_PARAM), ({"cap": -1.0}, mh.ERR_PARAM), ({"cap": float("nan")}, mh.ERR_PARAM),
             ({"cap": float("inf")}, mh.ERR_PARAM), ({"cap": 1025.0}, mh.ERR_PARAM), ({"cap": 1e-19}, mh.ERR_PARAM),
             ({"scale": 2e30}, mh.ERR_PARAM), ({"heads": 8192, "kv_heads": 8192}, mh.ERR_SHAPE),
             ({"q_rows": 1 << 30}, mh.ERR_SHAPE), ({"kv_rows": 1 << 30}, mh.ERR_SHAPE),
             ({"q_rows": 1 << 28}, mh.ERR_SHAPE),  # 2^28 rows of four heads a key head
             ({"q_row_stride": 132}, mh.ERR_ALIGN), ({"k_row_stride": 120}, mh.ERR_SHAPE),
             ({"v_row_stride": 1 << 23}, mh.ERR_SHAPE), ({"out_head_stride": 12}, mh.ERR_ALIGN),
             ({"k_head_stride": 4}, mh.ERR_ALIGN)]


@pytest.mark.parametrize("kw,code", DENSE_BAD)
def test_flash_attn_128_domain(kw, code):
    a = dense(**kw)
    assert mh.lib.mh3_flash_attn_128_workspace_bytes(C.byref(a)) == code
    assert mh.lib.mh3_flash_attn_128(C.byref(a), at(1), at(2), at(3), None, None, None, None, at(4), 1 << 30, at(5),
                                     None) == code


def attn(a, q=at(1), k=at(2), v=at(3), ranges=None, slopes=None, q_pos=None, k_pos=None, ws=at(4), n=1 << 33, out=at(5)):
    return mh.lib.mh3_flash_attn_128(None if a is None else C.byref(a), q, k, v, ranges, slopes, q_pos, k_pos, ws, n, out,
                                     None)


def test_flash_attn_128_pointers():
    a = dense()
    assert mh.lib.mh3_flash_attn_128_workspace_bytes(None) == mh.ERR_POINTER
    assert attn(None) == mh.ERR_POINTER
    for name in ("q", "k", "v", "out"):
        assert attn(a, **{name: None}) == mh.ERR_POINTER
        assert attn(a, **{name: ODD16}) == mh.ERR_ALIGN
    assert attn(a, ranges=C.c_void_p(0x1004)) == mh.ERR_ALIGN
    assert attn(a, slopes=ODD4) == mh.ERR_ALIGN
    assert attn(a, slopes=FAKE, q_pos=ODD4, k_pos=at(6)) == mh.ERR_ALIGN
    assert attn(a, slopes=FAKE, q_pos=FAKE) == mh.ERR_POINTER      # one position list alone
    assert attn(a, slopes=FAKE, k_pos=FAKE) == mh.ERR_POINTER
    assert attn(a, q_pos=FAKE, k_pos=at(6)) == mh.ERR_POINTER      # positions without slopes
    assert attn(dense(q_rows=0), q=None, k=None, v=None, out=None, ws=None, n=0) == mh.OK
    assert attn(dense(kv_rows=0), k=None, v=None, out=None) == mh.ERR_POINTER


def test_flash_attn_128_overlaps():
    a = dense()
    for name in ("q", "k", "v"):
        assert attn(a, **{name: at(5)}) == mh.ERR_PARAM
    assert attn(a, ranges=C.c_void_p(at(5).value + 64)) == mh.ERR_PARAM
    assert attn(a, slopes=C.c_void_p(at(5).value + 64)) == mh.ERR_PARAM
    assert attn(a, slopes=FAKE, q_pos=C.c_void_p(at(5).value + 64), k_pos=FAKE) == mh.ERR_PARAM
    assert attn(a, out=C.c_void_p(at(3).value + 2 * 200 * 256 - 16)) == mh.ERR_PARAM  # on v's last bytes
    # Rows of out that lie over each other: equal heads, and heads that begin inside the one before.
    for kw in ({"out_head_stride": 0}, {"out_head_stride": 128}, {"out_head_stride": 99 * 128},
               {"out_head_stride": 128, "out_row_stride": 7 * 128}):
        assert attn(dense(**kw)) == mh.ERR_PARAM


def test_flash_attn_128_workspace():
    few = dense(heads=8, kv_heads=1, q_rows=1, kv_rows=1 << 20, q_head_stride=128, out_head_stride=128,
                k_head_stride=1 << 27, v_head_stride=1 << 27)
    n = mh.lib.mh3_flash_attn_128_workspace_bytes(C.byref(few))
    assert n > 0
    assert attn(few, ws=None) == mh.ERR_POINTER
    assert attn(few, n=n - 1) == mh.ERR_SHAPE
    assert attn(few, ws=C.c_void_p(at(4).value + 8), n=n) == mh.ERR_ALIGN
    assert attn(few, ws=at(5), n=n) == mh.ERR_PARAM
    assert attn(few, ws=C.c_void_p(at(2).value + (1 << 20)), n=n) == mh.ERR_PARAM


def test_attn_ranges():
    f = mh.lib.mh3_attn_ranges
    a = mh.RangeArgs(100, 200, 3, 1)
    ok = [at(1), at(2), at(3), at(4)]
    assert f(None, *ok, None) == mh.ERR_POINTER
    for i, code in ((0, mh.ERR_POINTER), (1, mh.ERR_POINTER), (3, mh.ERR_POINTER)):
        p = list(ok)
        p[i] = None
        assert f(C.byref(a), *p, None) == code
    for i in range(4):
        p = list(ok)
        p[i] = ODD4 if i < 3 else C.c_void_p(0x1004)
        assert f(C.byref(a), *p, None) == mh.ERR_ALIGN
        p[i] = ok[3] if i < 3 else ok[0]
        assert f(C.byref(a), *p, None) == mh.ERR_PARAM
    for bad in ((100, 200, 0, 1), (1 << 30, 200, 3, 1), (100, 1 << 30, 3, 1), (100, 200, 1 << 30, 1)):
        assert f(C.byref(mh.RangeArgs(*bad)), *ok, None) == mh.ERR_SHAPE
    assert f(C.byref(mh.RangeArgs(100, 200, 3, 2)), *ok, None) == mh.ERR_PARAM
    assert f(C.byref(mh.RangeArgs(100, 200, 3, 0)), *ok, None) == mh.ERR_PARAM  # a prefix without causal
    assert f(C.byref(mh.RangeArgs(0, 200, 3, 1)), None, None, None, None, None) == mh.OK


def quant(**kw):
    a = mh.QuantArgs()
    a.rows, a.cols, a.dtype = 7, 512, mh.BF16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_quant_rows_mx4():
    f = mh.lib.mh3_quant_rows_mx4
    assert f(None, at(1), at(2), at(3), None) == mh.ERR_POINTER
    assert f(C.byref(quant(dtype=2)), at(1), at(2), at(3), None) == mh.ERR_PARAM
    for cols in (0, 16, 128, 511, 1 << 30):
        assert f(C.byref(quant(cols=cols)), at(1), at(2), at(3), None) == mh.ERR_SHAPE
    assert f(C.byref(quant(rows=1 << 31)), at(1), at(2), at(3), None) == mh.ERR_SHAPE
    for i in range(3):
        p = [at(1), at(2), at(3)]
        p[i] = None
        assert f(C.byref(quant()), *p, None) == mh.ERR_POINTER
        p[i] = ODD16
        assert f(C.byref(quant()), *p, None) == mh.ERR_ALIGN
    assert f(C.byref(quant()), at(1), at(1), at(3), None) == mh.ERR_PARAM
    assert f(C.byref(quant()), at(1), at(2), C.c_void_p(at(2).value + 16), None) == mh.ERR_PARAM
    assert f(C.byref(quant(rows=0)), None, None, None, None) == mh.OK


def gemm(m=3, n=512, k=768, sets=0, stride=0):
    a = mh.GemmArgs()
    a.m, a.n, a.k, a.n_sets, a.gate_stride = m, n, k, sets, stride
    return a


def products(a, x=at(1), xs=at(2), w=at(3), ws=at(4), gate=at(5), sets=None, out=at(6)):
    """The codes of the four entry points."""
    r = None if a is None else C.byref(a)
    return (mh.lib.mh3_gemm_mx4(r, x, xs, w, ws, out, None), mh.lib.mh3_gemm_mx4_swiglu(r, x, xs, w, ws, out, None),
            mh.lib.mh3_gemm_mx4_gate_add(r, x, xs, w, ws, gate, sets, out, None),
            mh.lib.mh3_gemm_mx4_gate_add_f32(r, x, xs, w, ws, gate, sets, out, None))


def test_gemm_mx4_sizes():
    assert set(products(None)) == {mh.ERR_POINTER}
    for kw in ({"m": 0}, {"n": 0}, {"k": 0}, {"k": 32}, {"k": 640}, {"n": 64}, {"m": 1 << 31},
               {"n": (1 << 32) - 256}):
        assert set(products(gemm(**kw))) == {mh.ERR_SHAPE}
    code = products(gemm(n=384))  # a multiple of 128: SwiGLU's columns alone
    assert code[0] == code[2] == code[3] == mh.ERR_SHAPE
    # w of 2^31 bytes and more; SwiGLU's w has twice the rows
    assert set(products(gemm(n=1 << 20, k=4096))) == {mh.ERR_UNSUPPORTED}
    assert mh.lib.mh3_gemm_mx4_swiglu(C.byref(gemm(n=1 << 19, k=4096)), at(1), at(2), at(3), at(4), at(6), None) == \
        mh.ERR_UNSUPPORTED
    assert set(products(gemm(k=1 << 24))) == {mh.ERR_UNSUPPORTED}          # 256 rows of x
    assert set(products(gemm(m=1 << 26, k=1024))) == {mh.ERR_UNSUPPORTED}  # x's scales


def test_gemm_mx4_pointers():
    for name in ("x", "xs", "w", "ws", "out"):
        assert set(products(gemm(), **{name: None})) == {mh.ERR_POINTER}
        assert set(products(gemm(), **{name: ODD16})) == {mh.ERR_ALIGN}
    for name in ("x", "xs", "w", "ws"):
        assert set(products(gemm(), **{name: at(6)})) == {mh.ERR_PARAM}
    assert products(gemm(), gate=None)[2:] == (mh.ERR_POINTER, mh.ERR_POINTER)
    assert products(gemm(), gate=ODD4)[2:] == (mh.ERR_ALIGN, mh.ERR_ALIGN)
    assert products(gemm(), gate=at(6))[2:] == (mh.ERR_PARAM, mh.ERR_PARAM)
    assert products(gemm(), sets=C.c_void_p(at(6).value + 2))[2:] == (mh.ERR_PARAM, mh.ERR_PARAM)
    assert products(gemm(sets=257))[2:] == (mh.ERR_PARAM, mh.ERR_PARAM)
    assert products(gemm(stride=511))[2:] == (mh.ERR_PARAM, mh.ERR_PARAM)


# ---- the binding ----------------------------------------------------------------------------------------------------

def test_binding_refuses_host_tensors_and_shapes():
    bf, i32, u8 = torch.bfloat16, torch.int32, torch.uint8
    q = torch.zeros((2, 5, 128), dtype=bf)
    pos = torch.zeros((5, 3), dtype=i32)
    x, xs = torch.zeros((3, 128), dtype=u8), torch.zeros((1, 3, 8), dtype=u8)
    w, ws = torch.zeros((256, 128), dtype=u8), torch.zeros((1, 256, 8), dtype=u8)
    off = torch.zeros(3, dtype=i32)
    calls = [lambda: mh.rotary_axes(pos, (16, 16, 16)), lambda: mh.rotary_axes(pos, (16, 16)),
             lambda: mh.rotary_axes(pos, ()), lambda: mh.rotary_axes(pos, (16, 16, -1)),
             lambda: mh.rotary_axes(pos, (16, 16, 16), theta=(1e4, 1e4)),
             lambda: mh.heads_partial_axes(torch.zeros((5, 768), dtype=bf), 2, pos, (16, 16, 16)),
             lambda: mh.heads_partial_axes(torch.zeros((4, 768), dtype=bf), 2, pos, (16, 16, 16)),
             lambda: mh.flash_attn_128(q, q, q), lambda: mh.flash_attn_128(q, q, q, layout="row"),
             lambda: mh.flash_attn_128(q.float(), q, q), lambda: mh.flash_attn_128(q, q[:1], q),
             lambda: mh.flash_attn_128(q[..., :64], q, q), lambda: mh.flash_attn_128(q.transpose(1, 2), q, q),
             lambda: mh.attn_ranges(off, off, 4, 4), lambda: mh.attn_ranges(off[:1], off[:1], 4, 4),
             lambda: mh.quant_rows_mx4(torch.zeros((2, 256), dtype=bf)), lambda: mh.quant_rows_mx4(torch.zeros((2, 96))),
             lambda: mh.quant_rows_mx4(torch.zeros(256)), lambda: mh.quant_rows_mx4(torch.zeros((2, 256), dtype=i32)),
             lambda: mh.gemm_mx4(x, xs, w, ws), lambda: mh.gemm_mx4(x, xs, w[:, :64], ws),
             lambda: mh.gemm_mx4_swiglu(x, xs, w, ws),
             lambda: mh.gemm_mx4_gate_add(x, xs, w, ws, torch.zeros((3, 256), dtype=bf), torch.zeros(256))]
    for call in calls:
        with pytest.raises((ValueError, RuntimeError)):
            call()


class OnGpu(torch.Tensor):
    """A host tensor that says that it is on a GPU."""
    is_cuda = True

    def get_device(self):
        return 0


@pytest.mark.parametrize("place", [0, 1, 2])
def test_a_host_tensor_among_the_operands_is_refused(place):
    """Wherever it stands, the first included: the kernel would take its host address."""
    host = torch.zeros(4)
    ts = [host if i == place else torch.zeros(4).as_subclass(OnGpu) for i in range(3)]
    with pytest.raises(ValueError, match=f"t{place}: must be on the GPU"):
        mh._operands(*((t, f"t{i}", torch.float32, 4) for i, t in enumerate(ts)))
    with pytest.raises(ValueError, match=f"t{place}: must be on the GPU"):
        mh._one_device(**{f"t{i}": t for i, t in enumerate(ts)})
    assert mh._operands(*((t, "t", torch.float32, 4) for i, t in enumerate(ts) if i != place)) == 0
    assert mh._one_device(none=None, **{f"t{i}": t for i, t in enumerate(ts) if i != place}) == 0


def test_host_tensors_alone_are_refused():
    """Every operand on the host: refused by name before the library or the GPU's runtime is called."""
    bf, i32, u8 = torch.bfloat16, torch.int32, torch.uint8
    q, pos, off = torch.zeros((2, 5, 128), dtype=bf), torch.zeros((5, 3), dtype=i32), torch.zeros(3, dtype=i32)
    x, xs = torch.zeros((3, 128), dtype=u8), torch.zeros((1, 3, 8), dtype=u8)
    w, ws = torch.zeros((256, 128), dtype=u8), torch.zeros((1, 256, 8), dtype=u8)
    for call in (lambda: mh.rotary_axes(pos, (16, 16, 16)), lambda: mh.attn_ranges(off, off, 4, 4),
                 lambda: mh.heads_partial_axes(torch.zeros((5, 768), dtype=bf), 2, pos, (16, 16, 16)),
                 lambda: mh.flash_attn_128(q, q, q), lambda: mh.quant_rows_mx4(torch.zeros((2, 256))),
                 lambda: mh.gemm_mx4(x, xs, w, ws), lambda: mh.gemm_mx4_swiglu(x, xs, w, ws),
                 lambda: mh.gemm_mx4_gate_add(x, xs, w, ws, torch.zeros((3, 256), dtype=bf), torch.zeros(256))):
        with pytest.raises(ValueError, match="must be on the GPU"):
            call()


class OnGpuTable(OnGpu):
    device = torch.device("cuda", 0)


def test_sets_that_are_one_vector_expanded_are_refused():
    """A broadcast gate has a stride of zero, which to the library means the sets lie one behind the other: it would read
    past the one vector that there is. A call of one set reads that vector alone."""
    one = torch.zeros((1, 256)).as_subclass(OnGpuTable)
    for gate in (one.expand(3, 256), one[0].expand(3, 256), one.expand(2, 3, 256)):
        with pytest.raises(ValueError, match="gate: its sets lie over each other"):
            mh._set_stride(gate, "gate", 256, 3)
        assert mh._set_stride(gate, "gate", 256, 1) in (0, 256)
    table = torch.zeros((3, 6, 256)).as_subclass(OnGpuTable)
    assert mh._set_stride(table[:, 2], "gate", 256, 3) == 6 * 256

def test_scales_of_other_rows_are_refused():
    """A scale buffer of more rows than its matrix holds other blocks' bytes from the second 256 columns on. The shapes are
    looked at before the device, so host tensors show it."""
    u8 = torch.uint8
    m, n, k = 3, 256, 512
    x, w = torch.zeros((m, k // 2), dtype=u8), torch.zeros((n, k // 2), dtype=u8)
    xs, ws = torch.zeros((k // 256, m, 8), dtype=u8), torch.zeros((k // 256, n, 8), dtype=u8)
    more_x, more_w = torch.zeros((k // 256, m + 1, 8), dtype=u8), torch.zeros((k // 256, 2 * n, 8), dtype=u8)
    res, gate = torch.zeros((m, n), dtype=torch.bfloat16), torch.zeros((1, n))
    ops = [lambda a, b: mh.gemm_mx4(x, a, w, b), lambda a, b: mh.gemm_mx4_swiglu(x, a, w, b),
           lambda a, b: mh.gemm_mx4_gate_add(x, a, w, b, res, gate)]
    for op in ops:
        for bad in (more_x, more_x.flatten(), xs.flatten()[:-8], xs.view(m, k // 256, 8), torch.zeros((1, 2 * m, 8), dtype=u8)):
            with pytest.raises(ValueError, match="x_scale: .*the scales of 3 rows of 512"):
                op(bad, ws)
        for bad in (more_w, more_w.flatten(), ws[:, :-1]):
            with pytest.raises(ValueError, match="w_scale: .*the scales of 256 rows of 512"):
                op(xs, bad)
        for good in ((xs, ws), (xs.flatten(), ws.flatten())):
            with pytest.raises(ValueError, match="must be on the GPU"):
                op(*good)
    v = torch.zeros((m, k))
    for bad in (more_x, more_x.flatten(), xs[:, :2]):
        with pytest.raises(ValueError, match="scale: .*the scales of 3 rows of 512"):
            mh.quant_rows_mx4(v, scale=bad)
    for good in (xs, xs.flatten()):
        with pytest.raises(ValueError, match="must be on the GPU"):
            mh.quant_rows_mx4(v, scale=good)
    # Of 256 columns there is one run of rows, and the first rows' scales lead it.
    with pytest.raises(ValueError, match="must be on the GPU"):
        mh.gemm_mx4(x[:, :128].contiguous(), torch.zeros((1, m + 4, 8), dtype=u8), w[:, :128].contiguous(), ws[:1])
