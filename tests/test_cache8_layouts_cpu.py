"""The layouts of the decode over the 8-bit K/V cache, without a GPU (for 256 CUs)."""

import ctypes

import pytest

from mtlattn_amd import capi
from tests import cache8_layouts


@pytest.mark.parametrize("name", cache8_layouts.CASES)
def test_cases_take_the_layout_they_are_for(name):
    assert cache8_layouts.layout(name) == cache8_layouts.CASES[name][-1]


def test_layout_and_workspace():
    """The workspace holds two partials of 16 rows for each piece, kv head and head group."""
    x = [ctypes.c_int32() for _ in range(3)]
    ref = [ctypes.byref(i) for i in x]

    def problem(**kw):
        p = capi.Problem(dtype=capi.DTYPE_BF16, num_seqs=40, total_q=40, total_kv=40, num_heads_q=64, num_heads_kv=8,
                         head_dim=128, max_seqlen_q=4, scale=1.0, cu_seqlens_q=0x1000, cu_seqlens_kv=0x1000)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    for d, longest in ((128, 30000), (64, 30000), (64, 500)):
        p = problem(head_dim=d)
        capi.call("mtlattn_decode8_layout", ctypes.byref(p), longest, *ref)
        waves, heads, pieces = (i.value for i in x)
        assert waves % heads == 0 and 8 % heads == 0 and (pieces > 0) == (longest > 2048)
        rows = 8 * 2 * pieces * 2 * 16          # (8 heads a group, 4 tokens: 4 heads to 16 rows)
        assert capi.lib().mtlattn_decode8_workspace_size(ctypes.byref(p), longest) == rows * 4 * (d + 1)
    lib = capi.lib()
    assert lib.mtlattn_decode8_layout(None, 100, *ref) == capi.ERR_INVALID
    for i in range(3):
        args = list(ref)
        args[i] = None
        assert lib.mtlattn_decode8_layout(ctypes.byref(problem()), 100, *args) == capi.ERR_INVALID
    assert lib.mtlattn_decode8_layout(ctypes.byref(problem()), -1, *ref) == capi.ERR_INVALID
    for kw in (dict(dtype=capi.DTYPE_F32), dict(head_dim=96), dict(max_seqlen_q=17), dict(max_seqlen_q=0)):
        assert lib.mtlattn_decode8_layout(ctypes.byref(problem(**kw)), 100, *ref) == capi.ERR_UNSUPPORTED
