"""The 8-bit K/V cache without a GPU: its oracle against what the definition
implies, and the refusals of the C ABI, the binding and the Python API."""

import ctypes
import math

import pytest
import torch

import mtlattn
from mtlattn_amd import capi
from oracle import cache8
from tests.cache8_helpers import CODES, pages_for, random_cache

FAKE = 0x1000   # never dereferenced: every call below stops in validation


def cache(**kw):
    c = capi.Cache8(code=capi.CODE_E4M3, page_size=64, block=32, num_heads_kv=2, head_dim=128, num_pages=8, k=FAKE,
                    k_row_stride=256, v=FAKE, v_row_stride=256, k_scale=FAKE, v_scale=FAKE, block_table=FAKE,
                    block_table_stride=4)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def problem(**kw):
    p = capi.Problem(dtype=capi.DTYPE_BF16, num_seqs=2, total_q=2, total_kv=512, num_heads_q=8, num_heads_kv=2,
                     head_dim=128, max_seqlen_q=1, scale=0.088, causal=1, window=0, cu_seqlens_q=FAKE,
                     cu_seqlens_kv=FAKE)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def write(c, dtype=capi.DTYPE_BF16, k=FAKE, krs=256, v=FAKE, vrs=256, total=4, n=2, cu=FAKE, cu_kv=FAKE):
    return capi.lib().mtlattn_cache8_write(ctypes.byref(c) if c else None, dtype, k, krs, v, vrs, total, n, cu, cu_kv,
                                           None)


def read(c, dtype=capi.DTYPE_BF16, k=FAKE, v=FAKE, total=4, n=2, cu=FAKE, cu_kv=FAKE):
    return capi.lib().mtlattn_cache8_read(ctypes.byref(c) if c else None, dtype, k, v, total, n, cu, cu_kv, None)


def decode(p, c, q=FAKE, qrs=1024, max_kv=256, out=FAKE, ws=None, ws_bytes=0):
    return capi.lib().mtlattn_decode8(ctypes.byref(p), q, qrs, ctypes.byref(c) if c else None, max_kv, out, None, ws,
                                      ws_bytes, None)


BAD_CACHES = [
    (dict(code=0), capi.ERR_INVALID, b"code"),
    (dict(code=5), capi.ERR_INVALID, b"code"),
    (dict(block=0), capi.ERR_INVALID, b"tokens per scale"),
    (dict(block=8), capi.ERR_INVALID, b"tokens per scale"),
    (dict(block=48, page_size=48), capi.ERR_INVALID, b"tokens per scale"),
    (dict(block=512, page_size=512), capi.ERR_INVALID, b"tokens per scale"),
    (dict(page_size=0), capi.ERR_INVALID, b"page_size"),
    (dict(page_size=48), capi.ERR_INVALID, b"page_size"),
    (dict(num_pages=0), capi.ERR_INVALID, b"num_pages"),
    (dict(num_pages=1 << 25), capi.ERR_INVALID, b"num_pages"),
    (dict(block_table_stride=0), capi.ERR_INVALID, b"block_table_stride"),
    (dict(num_heads_kv=0), capi.ERR_UNSUPPORTED, b"head_dim"),
    (dict(head_dim=8), capi.ERR_UNSUPPORTED, b"head_dim"),
    (dict(head_dim=100), capi.ERR_UNSUPPORTED, b"head_dim"),
    (dict(head_dim=264), capi.ERR_UNSUPPORTED, b"head_dim"),
    (dict(num_heads_kv=1024), capi.ERR_UNSUPPORTED, b"65536"),
    (dict(k_row_stride=255), capi.ERR_INVALID, b"cover a row"),
    (dict(v_row_stride=0), capi.ERR_INVALID, b"cover a row"),
    (dict(v_row_stride=1 << 24), capi.ERR_UNSUPPORTED, b"2^24"),
]


@pytest.mark.parametrize("kw,rc,text", BAD_CACHES)
def test_bad_caches_are_refused(kw, rc, text):
    for call in (lambda c: write(c), lambda c: read(c), lambda c: decode(problem(), c)):
        assert call(cache(**kw)) == rc
        assert text in capi.lib().mtlattn_last_error()


def test_bad_calls_are_refused():
    inv, uns = capi.ERR_INVALID, capi.ERR_UNSUPPORTED
    assert write(None) == inv and read(None) == inv and decode(problem(), None) == inv
    for name in ("k", "v", "k_scale", "v_scale", "block_table"):
        c = cache(**{name: None})
        assert write(c) == inv and read(c) == inv and decode(problem(), c) == inv
    for kw in (dict(dtype=3), dict(dtype=-1), dict(total=-1), dict(total=1 << 31), dict(n=0), dict(cu=None),
               dict(cu_kv=None), dict(k=None), dict(v=None)):
        assert write(cache(), **kw) == inv, kw
        assert read(cache(), **kw) == inv, kw
    # rows that overlap or are not aligned
    assert write(cache(), krs=255) == inv
    assert write(cache(), vrs=0) == inv
    assert write(cache(), krs=257) == uns
    assert write(cache(), k=FAKE + 8) == uns
    assert read(cache(), v=FAKE + 8) == uns
    assert write(cache(k=FAKE + 4)) == uns
    assert read(cache(v_row_stride=260)) == uns
    assert write(cache(v_scale=FAKE + 2)) == uns
    assert decode(problem(), cache(k=FAKE + 8)) == uns
    assert decode(problem(), cache(k_row_stride=264)) == uns
    # keys and values in the same memory: their blocks' waves would race
    assert write(cache(v=FAKE)) == inv
    assert write(cache(v=FAKE + (1 << 30))) == inv                       # (the scales)
    assert write(cache(v=FAKE + (1 << 30), v_scale=FAKE + 16)) == inv
    # nothing to do is no error, whatever the row pointers
    assert write(cache(), total=0, k=None, v=None) == capi.OK
    assert read(cache(), total=0, k=None, v=None) == capi.OK
    assert decode(problem(total_q=0), cache(), q=None, out=None) == capi.OK


def test_decode_limits():
    uns, inv = capi.ERR_UNSUPPORTED, capi.ERR_INVALID
    assert decode(problem(dtype=capi.DTYPE_F32), cache()) == uns
    assert decode(problem(max_seqlen_q=17), cache()) == uns
    assert decode(problem(max_seqlen_q=0), cache()) == uns
    assert decode(problem(head_dim=96), cache(head_dim=96)) == uns
    assert decode(problem(head_dim=64), cache()) == inv                  # the cache's is 128
    assert decode(problem(num_heads_kv=4), cache()) == inv
    assert decode(problem(), cache(), max_kv=-1) == inv
    assert decode(problem(), cache(), q=None) == inv
    assert decode(problem(), cache(), out=None) == inv
    assert decode(problem(), cache(), out=FAKE + 8) == uns
    assert decode(problem(), cache(), qrs=1025) == uns
    assert decode(problem(num_heads_q=7), cache()) == inv
    # splits need a workspace of the size that the query says
    p = problem(num_seqs=64, total_q=64, total_kv=64 * 30000)
    need = capi.lib().mtlattn_decode8_workspace_size(ctypes.byref(p), 30000)
    assert need > 0
    assert decode(p, cache(), max_kv=30000, ws=FAKE, ws_bytes=need - 1) == capi.ERR_WORKSPACE
    assert decode(p, cache(), max_kv=30000, ws=None, ws_bytes=need) == capi.ERR_WORKSPACE
    # (which does not grow with the batch)
    p = problem(num_seqs=4096, total_q=4096, total_kv=4096 * 30000)
    assert capi.lib().mtlattn_decode8_workspace_size(ctypes.byref(p), 30000) == need
    assert capi.lib().mtlattn_decode8_workspace_size(ctypes.byref(problem(head_dim=96)), 30000) == 0


def test_python_refusals():
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16)
    codes = torch.zeros(2, 16, 2, 128, dtype=torch.int8)
    sc = torch.ones(2, 1, 2)
    cu = torch.tensor([0, 1])
    table = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="go together"):
        mtlattn.paged_decode(q, codes, codes, cu, cu, table, 1, 1, k_scale=sc)
    with pytest.raises(RuntimeError, match="GPU"):
        mtlattn.paged_decode(q, codes, codes, cu, cu, table, 1, 1, k_scale=sc, v_scale=sc)
    with pytest.raises(RuntimeError, match="GPU"):
        mtlattn.paged_cache_write(q, q, codes, codes, sc, sc, cu, cu, table)
    with pytest.raises(RuntimeError, match="GPU"):
        mtlattn.paged_cache_read(codes, codes, sc, sc, cu, cu, table, 1)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        mtlattn.paged_cache_read(codes, codes, sc, sc, cu, cu, table, 1, dtype=torch.float64)


# ---- the oracle itself ----

@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_oracle_codes_are_the_nearest(kind):
    """nearest_code against a search over all codes."""
    dt = CODES[kind]
    every = torch.arange(256, dtype=torch.uint8).view(dt).double()
    every = every[torch.isfinite(every)]
    if kind == "int8":
        every = every[every >= -127]
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(2000, generator=g, dtype=torch.float64) * cache8.QMAX[dt] / 3,
                   torch.randn(500, generator=g, dtype=torch.float64) * 2.0 ** -6,
                   torch.tensor([0.0, 1e9, -1e9, math.inf, -math.inf])])
    got = cache8.nearest_code(x, dt)
    best = (x.clamp(-1e6, 1e6)[:, None] - every[None, :]).abs().amin(1)
    assert torch.equal((got - x.clamp(-1e6, 1e6)).abs(), best)
    nan = cache8.nearest_code(torch.tensor([math.nan], dtype=torch.float64), dt)
    assert bool(torch.isnan(nan)) if kind == "e4m3" else float(nan) == 0.0


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_oracle_write_read_error(kind):
    """A prompt, then tokens one by one with rising magnitudes: what is read
    back is within half a step of what was written, for int8 plus half a step
    for each time the block's scale grew."""
    g = torch.Generator().manual_seed(1)
    kv, page, block, hkv, d = 37, 32, 16, 2, 32
    table, pages = pages_for([kv], page, g)
    codes, scale = random_cache(kind, pages, page, hkv, d, block, g)
    x = torch.randn(kv, hkv, d, generator=g) * torch.exp2(torch.arange(kv) / 8.0)[:, None, None]
    cache8.write(codes, scale, x[:20], [0, 20], [20], table)
    grown = torch.zeros(hkv)
    for t in range(20, kv):
        before = scale.clone()
        cache8.write(codes, scale, x[t:t + 1], [0, 1], [t + 1], table)
        grown += ((scale > before).sum((0, 1)) > 0).float()
    assert grown.min() >= 2
    got = cache8.read(codes, scale, [0, kv], [kv], table, kv)
    err = (got - x.double()).abs()
    at = cache8.rows(table, 0, 0, kv, page, pages)
    sc = scale.repeat_interleave(block, 1).flatten(0, 1)[at].double()
    if kind == "int8":
        assert bool((err <= sc[:, :, None] * 0.5 * (1 + grown[None, :, None])).all())
    else:               # relative 2^-4 in the normal range; below it half of a step of 2^-9, and of the
        # steps before the scale grew, each at most half the next one
        assert bool((err <= torch.maximum(x.double().abs() * 2.0 ** -4, sc[:, :, None] * 2.0 ** -9)).all())
