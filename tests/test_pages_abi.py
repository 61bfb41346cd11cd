"""Refusals of the calls for kept rows in pages, through the C-ABI and through the Python binding. No call here reaches a
kernel."""
import ctypes as C

import pytest
import torch

import mako_h3 as mh

ODD16 = C.c_void_p((1 << 34) + 8)
ODD4 = C.c_void_p((1 << 34) + 2)


def at(i):
    """Distinct aligned addresses, 16 GB apart."""
    return C.c_void_p(i << 34)


def args(**kw):
    a = mh.PagesArgs(3, 5, 16, 64, 5)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def pools(*which, size=4096, stride=4096):
    return (mh.Pool * len(which))(*[mh.Pool(w.value if w is not None else None, size, stride) for w in which])


def take(a=None, p=None):
    p = p or [at(1), at(2), at(3), at(4), at(5)]
    return mh.lib.mh3_pages_take(C.byref(a or args()), *p, None)


def free(a=None, p=None):
    p = p or [at(1), at(2), at(3), at(4)]
    return mh.lib.mh3_pages_free(C.byref(a or args()), *p, None)


def fork(a=None, p=None, pool=None, n=1, ws=1 << 20):
    p = p or [at(i) for i in range(1, 8)]
    held = pool if pool is not None else pools(at(20))
    return mh.lib.mh3_pages_fork(C.byref(a or args()), held, n, *p, ws, None)


def compact(a=None, p=None, pool=None, n=1, ws=1 << 20):
    p = p or [at(i) for i in range(1, 6)]
    held = pool if pool is not None else pools(at(20))
    return mh.lib.mh3_pages_compact(C.byref(a or args()), held, n, *p, ws, None)


@pytest.mark.parametrize("kw", [{"streams": 0}, {"streams": 4097}, {"cols": 0}, {"cols": 1 << 24}, {"pages": 0},
                                {"pages": 1 << 24}, {"table_stride": 4}, {"table_stride": 1 << 32},
                                {"streams": 4096, "cols": 1 << 20, "table_stride": 1 << 20}])
def test_table_shape(kw):
    a = args(**kw)
    assert take(a) == free(a) == fork(a) == compact(a) == mh.ERR_SHAPE
    assert mh.lib.mh3_pages_fork_workspace_bytes(C.byref(a)) == mh.ERR_SHAPE
    assert mh.lib.mh3_pages_compact_workspace_bytes(C.byref(a)) == mh.ERR_SHAPE


@pytest.mark.parametrize("call,n,optional", [(take, 5, {4}), (free, 4, set()), (fork, 7, {5}), (compact, 5, {3})])
def test_pointers(call, n, optional):
    good = [at(i) for i in range(1, n + 1)]
    for i in range(n):
        p = list(good)
        p[i] = None
        if i not in optional:
            assert call(p=p) == mh.ERR_POINTER, i
        p[i] = ODD4
        assert call(p=p) == mh.ERR_ALIGN, i
    for i in range(n):
        for j in range(i):
            inputs = {take: {2, 3}, free: {2, 3}, fork: {0, 2, 3}, compact: set()}[call]
            if not {i, j} <= inputs:
                p = list(good)
                p[i] = p[j]
                assert call(p=p) == mh.ERR_PARAM, (i, j)
    for f in (mh.lib.mh3_pages_take, mh.lib.mh3_pages_free):
        assert f(None, *good[:len(f.argtypes) - 2], None) == mh.ERR_POINTER if len(good) >= len(f.argtypes) - 2 else True


@pytest.mark.parametrize("call,n", [(fork, 7), (compact, 5)])
def test_pools(call, n):
    assert call(pool=pools(*[at(20)] * 65), n=65) == mh.ERR_SHAPE
    assert call(pool=C.POINTER(mh.Pool)(), n=1) == mh.ERR_POINTER
    assert call(pool=pools(None)) == mh.ERR_POINTER
    assert call(pool=pools(ODD16)) == mh.ERR_ALIGN
    assert call(pool=pools(at(20), size=4088)) == mh.ERR_ALIGN
    assert call(pool=pools(at(20), stride=4104)) == mh.ERR_ALIGN
    assert call(pool=pools(at(20), size=0)) == mh.ERR_SHAPE
    assert call(pool=pools(at(20), size=4112)) == mh.ERR_SHAPE      # pages over each other
    assert call(pool=pools(at(20), stride=1 << 39)) == mh.ERR_SHAPE
    assert call(pool=pools(at(20), at(20)), n=2) == mh.ERR_PARAM
    assert call(pool=pools(at(20), C.c_void_p(at(20).value + 15 * 4096)), n=2) == mh.ERR_PARAM
    for i in range(1, n + 1):     # each table and list in the pool's last page
        assert call(pool=pools(C.c_void_p(at(i).value - 15 * 4096))) == mh.ERR_PARAM, i
    assert call(ws=8) == mh.ERR_SHAPE
    a = args()
    assert mh.lib.mh3_pages_fork_workspace_bytes(C.byref(a)) == 24
    assert mh.lib.mh3_pages_compact_workspace_bytes(C.byref(a)) == 16 + 64


def test_fork_page_rows():
    assert fork(args(page_rows=0)) == mh.ERR_SHAPE
    assert fork(args(page_rows=1 << 30)) == mh.ERR_SHAPE


def test_copy():
    f = mh.lib.mh3_pages_copy
    assert f(pools(at(20)), 1, 0, at(1), at(2), 3, None) == mh.ERR_SHAPE
    assert f(pools(at(20)), 1, 1 << 24, at(1), at(2), 3, None) == mh.ERR_SHAPE
    assert f(pools(at(20)), 1, 16, at(1), at(2), 16385, None) == mh.ERR_SHAPE
    assert f(pools(at(20)), 65, 16, at(1), at(2), 3, None) == mh.ERR_SHAPE
    assert f(None, 1, 16, at(1), at(2), 3, None) == mh.ERR_POINTER
    assert f(pools(at(20)), 1, 16, None, at(2), 3, None) == mh.ERR_POINTER
    assert f(pools(at(20)), 1, 16, at(1), ODD4, 3, None) == mh.ERR_ALIGN
    assert f(pools(at(20)), 1, 16, at(1), C.c_void_p(at(20).value + 64), 3, None) == mh.ERR_PARAM
    assert f(pools(at(20)), 1, 16, None, None, 0, None) == mh.OK


def write(a=None, p=None, **kw):
    w = mh.PagesWriteArgs(args(), 2, 128, 9, 9, 9 * 128, 128, 9 * 128, 128, *[16384, 8192, 128] * 2)
    for k, v in kw.items():
        setattr(w, k, v)
    if a is not None:
        w.table = a
    p = p or [at(i) for i in range(1, 9)]
    return mh.lib.mh3_pages_write(C.byref(w), *p, None)


def test_write():
    assert mh.lib.mh3_pages_write(None, *[at(i) for i in range(1, 9)], None) == mh.ERR_POINTER
    assert write(args(streams=0)) == write(args(page_rows=0)) == write(args(page_rows=1 << 28)) == mh.ERR_SHAPE
    assert write(kv_heads=0) == write(kv_heads=4097) == write(n_rows=1 << 30) == write(n=1 << 31) == mh.ERR_SHAPE
    assert write(head_dim=64) == mh.ERR_UNSUPPORTED
    for t in ("k", "v"):
        for d in ("row", "page_row"):
            assert write(**{f"{t}_{d}_stride": 132}) == mh.ERR_ALIGN
            assert write(**{f"{t}_{d}_stride": 120}) == write(**{f"{t}_{d}_stride": 1 << 23}) == mh.ERR_SHAPE
        for d in ("head", "page", "page_head"):
            assert write(**{f"{t}_{d}_stride": 1028}) == mh.ERR_ALIGN
            assert write(**{f"{t}_{d}_stride": 1 << 36}) == mh.ERR_SHAPE
    good = [at(i) for i in range(1, 9)]
    for i in range(8):
        p = list(good)
        p[i] = None
        if i < 7:
            assert write(p=p) == mh.ERR_POINTER
        p[i] = ODD16 if i < 4 else ODD4
        assert write(p=p) == mh.ERR_ALIGN
        for pool in (2, 3):
            if i != pool:
                p[i] = C.c_void_p(at(pool + 1).value + 4096) if i not in (2, 3) else at(pool + 1)
                assert write(p=p) == mh.ERR_PARAM
    assert write(n=0, p=[None] * 8) == write(n_rows=0, p=[None] * 8) == mh.OK


def test_binding():
    """What the Python layer refuses before it comes to the library."""
    t, r, s = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        mh.pages_take(t, r, s, s)
    with pytest.raises(TypeError):
        mh.pages_take([[0]], r, s, s)
    with pytest.raises(ValueError, match="int32"):
        mh.pages_free(t.long(), r, s, s)
    with pytest.raises(ValueError, match="refs"):
        mh.pages_free(t, r[::2], s, s)
    with pytest.raises(ValueError, match="contiguous"):
        mh.pages_free(torch.zeros((3, 2), dtype=torch.int32).T, r, s, s)
    with pytest.raises(ValueError, match="over each other"):
        mh.pages_free(t[:1].expand(2, 3), r, s, s)
    pool = torch.zeros((8, 4))
    with pytest.raises(ValueError, match="pages"):
        mh.pages_fork(pool[:7], t, r, s, s, 16)
    with pytest.raises(ValueError, match="contiguous"):
        mh.pages_compact(torch.zeros((8, 4, 4)).transpose(1, 2), t, r)
    with pytest.raises(ValueError, match="at most"):
        mh.pages_compact([pool] * 65, t, r)
    with pytest.raises(ValueError, match="GPU"):
        mh.pages_copy(pool, s, s)
    k = torch.zeros((2, 9, 128), dtype=torch.bfloat16)
    kp = torch.zeros((8, 2, 16, 128), dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="layout"):
        mh.pages_write(k, k, kp, kp, t, s, off, layout="columns")
    with pytest.raises(ValueError, match="same heads"):
        mh.pages_write(k, k[:1], kp, kp, t, s, off)
    with pytest.raises(ValueError, match="k_pages"):
        mh.pages_write(k, k, kp.float(), kp, t, s, off)
    with pytest.raises(ValueError, match="heads of k"):
        mh.pages_write(k, k, kp[:, :1], kp[:, :1], t, s, off)
    with pytest.raises(ValueError, match="GPU"):
        mh.pages_write(k, k, kp, kp.clone(), t, s, off)
