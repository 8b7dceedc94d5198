"""Which memory a write into the 8-bit K/V cache takes for its rows, codes and
scales: what would race is refused before anything is launched."""

import ctypes

import pytest

from mtlattn_amd import capi

# Addresses that are never dereferenced: a call that is not refused stops at its grid,
# which is larger than a launch can be.
ROWS_K, ROWS_V, K, V, KS, VS = 1 << 44, 1 << 46, 1 << 50, 1 << 51, 1 << 52, 1 << 53
HEADS, D, PAGE, BLOCK, PAGES, TOTAL = 128, 16, 64, 16, 4, (1 << 31) - 1
ROW = HEADS * D                                   # bytes of a token's codes
SPAN = PAGES * PAGE * ROW                         # of one side's, contiguous
SCALES = PAGES * (PAGE // BLOCK) * HEADS * 4      # of one side's scales


def write(rows_k=ROWS_K, rows_v=ROWS_V, total=TOTAL, **kw):
    c = capi.Cache8(code=capi.CODE_INT8, page_size=PAGE, block=BLOCK, num_heads_kv=HEADS, head_dim=D, num_pages=PAGES,
                    k=K, k_row_stride=ROW, v=V, v_row_stride=ROW, k_scale=KS, v_scale=VS, block_table=1 << 40,
                    block_table_stride=4)
    for name, x in kw.items():
        setattr(c, name, x)
    rc = capi.lib().mtlattn_cache8_write(ctypes.byref(c), capi.DTYPE_BF16, rows_k, ROW, rows_v, ROW, total, 2, 1 << 40,
                                         1 << 40, None)
    return rc, capi.lib().mtlattn_last_error()


def side_by_side(stride, shift):
    return dict(k_row_stride=stride, v_row_stride=stride, v=K + shift)


@pytest.mark.parametrize("kw", [
    dict(),
    # K and V rows side by side in one buffer, either first, with and without a gap
    side_by_side(2 * ROW, ROW), side_by_side(2 * ROW, -ROW), side_by_side(3 * ROW, 2 * ROW), side_by_side(2 * ROW, 3 * ROW),
    side_by_side(2 * ROW + 16, ROW + 8), side_by_side(2 * ROW, PAGES * PAGE * 2 * ROW),
    # one after the other
    dict(v=K + SPAN), dict(v=K - SPAN), dict(v_scale=KS + SCALES), dict(v_scale=KS - SCALES),
    dict(k_scale=K + SPAN), dict(k_scale=K - SCALES), dict(v_scale=K + SPAN), dict(k=ROWS_K - SPAN),
    # scales in the gaps between rows
    dict(k_row_stride=ROW + 2 * SCALES, k_scale=K + ROW, v_scale=K + ROW + SCALES),
    # rows that are only read may be the same
    dict(rows_v=ROWS_K),
])
def test_layouts_that_share_nothing_are_taken(kw):
    rc, text = write(**kw)
    assert rc == capi.ERR_LAUNCH, text


@pytest.mark.parametrize("kw", [
    dict(v=K),
    # a page, a row, half a row, the last row, and the other way round
    dict(v=K + PAGE * ROW), dict(v=K + ROW), dict(v=K + ROW // 2), dict(v=K + SPAN - 8), dict(v=K - ROW // 2),
    dict(v=K - SPAN + 8),
    side_by_side(2 * ROW, 2 * ROW), side_by_side(2 * ROW, ROW - 8), side_by_side(2 * ROW, ROW + 8),
    side_by_side(3 * ROW, 4 * ROW - 16), side_by_side(2 * ROW, PAGE * 2 * ROW),
    # rows of two strides in one buffer
    dict(v=K + ROW, v_row_stride=2 * ROW), dict(k_row_stride=2 * ROW, v=K + ROW),
    # the scales
    dict(v_scale=KS), dict(v_scale=KS + SCALES - 4), dict(v_scale=KS - SCALES + 4),
    # scales among the codes, of either side
    dict(k_scale=K), dict(v_scale=K + SPAN - 4), dict(k_scale=V - 4), dict(v_scale=V + 5 * ROW),
    dict(k_row_stride=ROW + SCALES, k_scale=K + ROW + 4), dict(k_row_stride=ROW + SCALES, v_scale=K + 9 * ROW),
    # rows that the call writes over
    dict(rows_k=K), dict(rows_v=K + SPAN - 16), dict(rows_k=V), dict(rows_v=V), dict(rows_k=KS), dict(rows_v=VS),
])
@pytest.mark.parametrize("total", [TOTAL, 1])
def test_layouts_that_share_memory_are_refused(kw, total):
    rc, text = write(total=total, **kw)
    assert rc == capi.ERR_INVALID and b"share" in text
