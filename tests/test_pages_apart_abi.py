"""pages_write refuses pools whose rows lie over each other, which would keep whichever store came last, and takes every
layout whose rows lie apart. Through the C-ABI; every call here is refused, for one reason or the other, before a kernel."""
import ctypes as C

import pytest

import mako_h3 as mh
from test_pages_abi import ODD4, args, at

HEADS, ROWS, PAGES = 2, 64, 16


def write(k_pages, v_pages, k=None, v=None, table=None, heads=HEADS, n=9, starts=ODD4):
    """Offsets in elements from one address; strides (page, head, row)."""
    k = k or (ROWS * HEADS * 128, ROWS * 128, 128)
    w = mh.PagesWriteArgs(table or args(), heads, 128, 9, n, 9 * 128, 128, 9 * 128, 128, *k, *(v or k))
    pool = [C.c_void_p(at(20).value + 2 * x) for x in (k_pages, v_pages)]
    return mh.lib.mh3_pages_write(C.byref(w), at(1), at(2), *pool, at(5), starts, at(7), at(8), None)


FAR = 1 << 32
PAGE = ROWS * HEADS * 128
OVER = [
    # V's offset from K, strides of both pools
    (FAR, (0, ROWS * 128, 128)),                    # one page for all of them
    (FAR, (PAGE, 0, 128)),                          # one head
    (FAR, (PAGE, 128, 128)),                        # the heads a row apart
    (FAR, (PAGE - 128, ROWS * 128, 128)),           # a page's last row is the next one's first
    (FAR, (128, PAGES * 128, 256)),                 # pages and rows over each other
    (FAR, (PAGE + 8, ROWS * 128 + 8, 136)),         # row 60 of a head, 8160 .. 8287, over the next head's first, from 8200 on
    (128, (PAGE, ROWS * 128, 128)),                 # V a row into K
    (-128, (2 * PAGE, ROWS * 128, 128)),
    (PAGE - 128, (2 * PAGE, ROWS * 128, 128)),
    (PAGE + 128, (2 * PAGE, ROWS * 128, 128)),      # V's last row is the next page's first of K
    (3 * PAGE, (PAGE, ROWS * 128, 128)),            # V's pages are K's other ones
    (HEADS * 128, (PAGE, 128, HEADS * 128)),        # rows of heads side by side: V's are K's next ones
]
APART = [
    (FAR, (PAGE, ROWS * 128, 128)),
    (PAGE, (2 * PAGE, ROWS * 128, 128)),                        # [pages][2][heads][rows]
    (-PAGE, (2 * PAGE, ROWS * 128, 128)),
    (3 * PAGE, (2 * PAGE, ROWS * 128, 128)),                    # V's pages one further on
    (5 * PAGE, (8 * PAGE, ROWS * 128, 128)),                    # a layer's slices of several
    (-7 * PAGE, (8 * PAGE, ROWS * 128, 128)),
    (HEADS * 128, (2 * PAGE, 128, 2 * HEADS * 128)),            # [pages][rows][2][heads * 128]
    (128, (2 * PAGE, 256, 2 * HEADS * 128)),                    # [pages][rows][heads][2][128]
    (ROWS * 128, (2 * PAGE, 2 * ROWS * 128, 128)),              # [pages][heads][2][rows]
    (PAGES * ROWS * 128, (ROWS * 128, 2 * PAGES * ROWS * 128, 128)),    # [heads][2][pages][rows]
    (FAR, (HEADS * (ROWS * 136 + 8), ROWS * 136 + 8, 136)),             # gaps behind rows and heads
]


@pytest.mark.parametrize("offset,strides", OVER)
def test_over_each_other(offset, strides):
    assert write(0, offset, strides) == mh.ERR_PARAM
    if offset == FAR:       # either pool alone
        good = (PAGE, ROWS * 128, 128)
        assert write(0, offset, strides, good) == write(0, offset, good, strides) == mh.ERR_PARAM


@pytest.mark.parametrize("offset,strides", APART)
def test_apart(offset, strides):
    """Layouts that are taken come as far as the lists' alignment."""
    assert write(0, offset, strides) == mh.ERR_ALIGN
    assert write(0, offset, strides, n=0) == mh.OK


def test_single_dimensions_carry_any_stride():
    """One page, one head, one row: their strides are never stepped over."""
    one = args(pages=1, page_rows=1)
    assert write(0, 128, (0, 0, 128), table=one, heads=1) == mh.ERR_ALIGN
    assert write(0, 120, (0, 0, 128), table=one, heads=1) == mh.ERR_PARAM
