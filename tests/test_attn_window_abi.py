"""Refusals of flash_attn_128's second ranges and of attn_window_ranges, through the C-ABI and the Python binding. No call
here reaches a kernel."""
import ctypes as C

import pytest
import torch

import mako_h3 as mh
from test_pages_abi import ODD4, at


def sinks_call(**kw):
    a = mh.DenseAttnArgs(4, 2, 128, 8, 64, 0.0, 0.0, 0, 1024, 128, 8192, 128, 8192, 128, 1024, 128)
    p = {"q": at(1), "k": at(2), "v": at(3), "ranges": at(4), "sinks": at(5), "slopes": None, "q_pos": None, "k_pos": None,
         "ws": at(6), "bytes": 1 << 30, "out": at(7)}
    p.update(kw)
    return mh.lib.mh3_flash_attn_128_sinks(C.byref(a), *p.values(), None)


def test_sinks():
    assert sinks_call(ranges=None) == mh.ERR_POINTER        # sinks only with ranges
    assert sinks_call(sinks=C.c_void_p(at(5).value + 4)) == mh.ERR_ALIGN
    assert sinks_call(sinks=C.c_void_p(at(7).value + 64)) == mh.ERR_PARAM
    assert sinks_call(out=C.c_void_p(at(5).value + 48)) == mh.ERR_PARAM
    assert sinks_call(q=None) == mh.ERR_POINTER


def window(a=None, p=None, **kw):
    w = mh.WindowArgs(8, 64, 3, 1, 16, 0)
    for k, v in kw.items():
        setattr(w, k, v)
    p = p or [at(i) for i in range(1, 6)]
    return mh.lib.mh3_attn_window_ranges(C.byref(w), *p, None)


def test_window_ranges():
    assert mh.lib.mh3_attn_window_ranges(None, *[at(i) for i in range(1, 6)], None) == mh.ERR_POINTER
    assert window(causal=2) == window(window=0) == mh.ERR_PARAM
    assert window(docs=0) == window(docs=1 << 30) == window(q_rows=1 << 30) == window(kv_rows=1 << 30) == mh.ERR_SHAPE
    good = [at(i) for i in range(1, 6)]
    for i in range(5):
        p = list(good)
        p[i] = None
        if i != 2:
            assert window(p=p) == mh.ERR_POINTER
        p[i] = ODD4
        assert window(p=p) == mh.ERR_ALIGN
        if i < 3:
            p[i] = C.c_void_p(at(4).value + 32)
            assert window(p=p) == mh.ERR_PARAM
    assert window(p=[*good[:4], C.c_void_p(at(4).value + 32)]) == mh.ERR_PARAM
    assert window(q_rows=0, p=[None] * 5) == mh.OK


def test_binding():
    off = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="window"):
        mh.attn_window_ranges(off, off, 4, 4, 0)
    with pytest.raises(ValueError, match="one document"):
        mh.attn_window_ranges(off[:1], off[:1], 4, 4, 3)
    with pytest.raises(TypeError):
        mh.attn_window_ranges([0, 4], off, 4, 4, 3)
    with pytest.raises(ValueError, match="GPU"):
        mh.attn_window_ranges(off, off, 4, 4, 3)
