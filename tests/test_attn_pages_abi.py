"""Refusals of flash_attn_pages_128, through the C-ABI and the Python binding. No call here reaches a kernel."""
import ctypes as C

import pytest
import torch

import mako_h3 as mh
from test_pages_abi import ODD4, ODD16, args, at

NAMES = ("q", "k", "v", "k_pages", "v_pages", "table", "lengths", "q_off", "parents", "sinks", "ws")


def attn_args(table=None, **kw):
    a = mh.PagesAttnArgs(table or args(), 4, 2, 128, 9, 0, 0.0, 0.0, 0, *[9 * 128, 128] * 4, *[16384, 8192, 128] * 2)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def call(a=None, size=1 << 30, out=at(30), **p):
    ptrs = [p.get(n, at(i + 1)) for i, n in enumerate(NAMES)]
    return mh.lib.mh3_flash_attn_pages_128(C.byref(a or attn_args()), *ptrs, size, out, None)


def test_shapes():
    assert mh.lib.mh3_flash_attn_pages_128(None, *[at(i) for i in range(1, 12)], 1 << 30, at(12), None) == mh.ERR_POINTER
    for kw in ({"heads": 0}, {"kv_heads": 0}, {"head_dim": 0}, {"heads": 5}, {"heads": 4098}, {"q_rows": 1 << 30},
               {"q_rows": 1 << 29, "heads": 8}):
        assert call(attn_args(**kw)) == mh.ERR_SHAPE, kw
    assert call(attn_args(head_dim=64)) == mh.ERR_UNSUPPORTED
    for kw in ({"streams": 0}, {"streams": 4097}, {"cols": 0}, {"pages": 0}, {"pages": 1 << 24}, {"table_stride": 4},
               {"page_rows": 0}, {"page_rows": 24}, {"page_rows": 8}, {"page_rows": 1 << 28}):
        assert call(attn_args(args(**kw))) == mh.ERR_SHAPE, kw
    for kw in ({"scale": -1.0}, {"scale": float("nan")}, {"cap": -1.0}, {"cap": 1025.0}, {"cap": float("inf")},
               {"zero_rest": 2}):
        assert call(attn_args(**kw)) == mh.ERR_PARAM, kw
    for t in ("q", "k", "v", "out"):
        assert call(attn_args(**{f"{t}_row_stride": 132})) == call(attn_args(**{f"{t}_head_stride": 4})) == mh.ERR_ALIGN
        assert call(attn_args(**{f"{t}_row_stride": 120})) == call(attn_args(**{f"{t}_row_stride": 1 << 23})) == mh.ERR_SHAPE
    for t in ("k", "v"):
        for d in ("page", "page_head", "page_row"):
            assert call(attn_args(**{f"{t}_{d}_stride": 1028})) == mh.ERR_ALIGN
        assert call(attn_args(**{f"{t}_page_row_stride": 64})) == call(attn_args(**{f"{t}_page_stride": 1 << 36})) == \
            mh.ERR_SHAPE
    assert mh.lib.mh3_flash_attn_pages_128_workspace_bytes(C.byref(attn_args(heads=5))) == mh.ERR_SHAPE
    assert call(attn_args(q_rows=0), out=None, **{n: None for n in NAMES}) == mh.OK


def test_pointers():
    need = mh.lib.mh3_flash_attn_pages_128_workspace_bytes(C.byref(attn_args()))
    assert need > 0 and call(size=need - 1) == mh.ERR_SHAPE
    for i, n in enumerate(NAMES):
        if n not in ("parents", "sinks"):
            assert call(**{n: None}) == mh.ERR_POINTER, n
        assert call(**{n: ODD16 if n in ("q", "k", "v", "k_pages", "v_pages", "ws") else ODD4}) == mh.ERR_ALIGN, n
        assert call(out=at(i + 1)) == mh.ERR_PARAM, n
        if n != "ws":
            assert call(ws=at(i + 1)) == mh.ERR_PARAM, n
    assert call(out=None) == mh.ERR_POINTER and call(out=ODD16) == mh.ERR_ALIGN
    # out in a pool's last page; its heads over each other.
    assert call(out=C.c_void_p(at(4).value + 15 * 32768 + 64)) == mh.ERR_PARAM
    assert call(attn_args(out_head_stride=128)) == mh.ERR_PARAM


def test_binding():
    h = torch.zeros((4, 9, 128), dtype=torch.bfloat16)
    k, pool = h[:2], torch.zeros((16, 2, 64, 128), dtype=torch.bfloat16)
    t, n, off = torch.zeros((3, 5), dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    f = mh.flash_attn_pages_128
    with pytest.raises(ValueError, match="GPU"):
        f(h, k, k, pool, pool, t, n, off)
    with pytest.raises(ValueError, match="q's rows"):
        f(h, k[:, :8], k[:, :8], pool, pool, t, n, off)
    with pytest.raises(ValueError, match="heads of k"):
        f(h, k, k, pool[:, :1], pool[:, :1], t, n, off)
    with pytest.raises(ValueError, match="heads of k"):
        f(h, k, k, pool, pool[:8], t, n, off)
    with pytest.raises(ValueError, match="window"):
        f(h, k, k, pool, pool, t, n, off, window=-1)
    with pytest.raises(ValueError, match="layout"):
        f(h, k, k, pool, pool, t, n, off, page_layout="pages")
    with pytest.raises(ValueError, match="dtype"):
        f(h.float(), k, k, pool, pool, t, n, off)
    with pytest.raises(TypeError):
        f(h, k, k, pool, pool, [[0]], n, off)
