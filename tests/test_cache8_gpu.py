"""The 8-bit paged K/V cache on the GPU: writing, reading back and decode
attention against the fp64 oracle, at the sizes and masks where they can go
wrong, under graphs and streams, and together as a server uses them."""

import math

import pytest
import torch

from oracle import cache8
from tests.cache8_helpers import (CODES, check_decode, decode_reference, pages_for, poison_free_rows, random_cache,
                                  same_codes)
from tests.helpers import cu_of

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mt():
    import mtlattn
    return mtlattn


def _clone(ts):
    return [t.clone() for t in ts]


def _dev(ts):
    return [t.cuda() for t in ts]


def _cache(kind, kv_lens, page, hkv, d, block, gen, width=0):
    """CPU (k_cache, v_cache, k_scale, v_scale) and the block table."""
    table, pages = pages_for(kv_lens, page, gen, width=width)
    kc, ks = random_cache(kind, pages, page, hkv, d, block, gen)
    vc, vs = random_cache(kind, pages, page, hkv, d, block, gen)
    return [kc, vc, ks, vs], table


def _same_cache(got, want):
    for a, b in zip(got[:2], want[:2]):
        same = same_codes(a, b)
        assert same
    for a, b in zip(got[2:], want[2:]):
        assert torch.equal(a.cpu(), b)


def _write_both(mt, cache, table, k, v, cu, kv_lens, dev=None):
    """The kernel's write into a copy on the GPU, and the oracle's in place."""
    got = _dev(cache) if dev is None else dev
    mt.paged_cache_write(k.cuda(), v.cuda(), *got, torch.tensor(cu, dtype=torch.int32).cuda(), cu_of(kv_lens, "cuda"),
                         table.cuda())
    cache8.write(cache[0], cache[2], k, cu, kv_lens, table)
    cache8.write(cache[1], cache[3], v, cu, kv_lens, table)
    return got


WRITES = [
    # kind, type, hkv, d, page, block, new tokens, kv lengths
    ("e4m3", BF16, 8, 128, 16, 16, [1, 1, 1, 1], [1, 16, 17, 700]),
    ("int8", F16, 8, 128, 16, 16, [1, 1, 1, 1], [1, 16, 17, 700]),
    ("e4m3", F16, 2, 64, 64, 32, [33, 1, 64, 0], [33, 40, 100, 5]),
    ("int8", BF16, 2, 64, 64, 64, [63, 200, 0, 3], [63, 201, 9, 130]),
    ("e4m3", F32, 3, 80, 128, 128, [129, 5], [300, 128]),
    ("int8", F32, 3, 88, 128, 128, [129, 5], [300, 128]),
    ("e4m3", BF16, 1, 256, 256, 256, [255, 2, 300], [255, 257, 800]),
    ("int8", BF16, 5, 256, 256, 256, [255, 2, 300], [255, 257, 800]),
    ("int8", F32, 1, 256, 512, 256, [700], [700]),
    ("e4m3", F32, 17, 16, 48, 16, [50, 1], [50, 49]),
    ("int8", F16, 16, 96, 32, 32, [0, 0, 31], [0, 3, 31]),
    ("e4m3", BF16, 8, 128, 64, 64, [2000], [5000]),
]


@pytest.mark.parametrize("kind,dt,hkv,d,page,block,new,kv", WRITES)
def test_write(mt, kind, dt, hkv, d, page, block, new, kv):
    """Codes, scales and everything that no row goes to, bit for bit."""
    g = torch.Generator().manual_seed(d + page + len(new))
    cache, table = _cache(kind, kv, page, hkv, d, block, g)
    gain = torch.exp(1.5 * torch.randn(1, hkv, d, generator=g))
    k = (torch.randn(sum(new), hkv, d, generator=g) * gain / 50).to(dt)
    v = (torch.randn(sum(new), hkv, d, generator=g) / 3).to(dt)
    _same_cache(_write_both(mt, cache, table, k, v, cu_of(new).tolist(), kv), cache)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_write_exact_ties(mt, kind):
    """Multiples of a quarter and of 1.5 under the largest magnitudes 448, 127
    and 381 = 3 * 127: quotients that lie on ties, also where 1 / scale is not
    a float."""
    g = torch.Generator().manual_seed(3)
    kv, hkv, d = [48], 2, 64
    cache, table = _cache(kind, kv, 16, hkv, d, 16, g)
    k = torch.randint(-80, 81, (48, hkv, d), generator=g).float() * 1.5
    v = torch.randint(-200, 201, (48, hkv, d), generator=g).float() * 0.25
    for b, top in enumerate((448.0, 127.0, 381.0)):
        k[16 * b, :, 0] = top
        v[16 * b, :, 0] = -top
    _same_cache(_write_both(mt, cache, table, k, v, [0, 48], kv), cache)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("block", [16, 64])
def test_write_token_by_token(mt, kind, block):
    """Appending with rising and falling magnitudes: a block's scale grows, and
    its earlier codes follow; a new block starts anew."""
    g = torch.Generator().manual_seed(7)
    hkv, d, page = 3, 64, 64
    cache, table = _cache(kind, [90, 40], page, hkv, d, block, g)
    lens = [10, 3]
    k0 = torch.randn(13, hkv, d, generator=g).to(BF16)
    dev = _write_both(mt, cache, table, k0, -k0, [0, 10, 13], lens)
    for step in range(30):
        lens = [lens[0] + 2, lens[1] + 1]
        k = (torch.randn(3, hkv, d, generator=g) * 2.0 ** (5 * math.sin(step))).to(BF16)
        v = (torch.randn(3, hkv, d, generator=g) * 2.0 ** (step / 4)).to(BF16)
        _write_both(mt, cache, table, k, v, [0, 2, 3], lens, dev)
    _same_cache(dev, cache)
    # tokens taken back and written again
    lens = [lens[0] - 3, lens[1]]
    k = torch.randn(5, hkv, d, generator=g).to(BF16)
    _write_both(mt, cache, table, k, k, [0, 2, 5], lens, dev)
    _same_cache(dev, cache)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_write_extremes(mt, kind, dt):
    """Zeros, the type's largest and smallest values, infinities and NaN: the
    scale is that of the finite values, a NaN stays where it is."""
    g = torch.Generator().manual_seed(11)
    kv, hkv, d = [96], 2, 64
    cache, table = _cache(kind, kv, 16, hkv, d, 16, g)
    k = torch.randn(96, hkv, d, generator=g).to(dt)
    k[0:16] = 0
    k[16:32, :, ::3] = math.inf
    k[20, 0, 1], k[21, 1, 5] = -math.inf, math.nan
    k[32:48] = (k[32:48].float() * 2.0 ** 120).to(dt)
    k[48:64] = (k[48:64].float() * 2.0 ** -120).to(dt)
    k[64:80] = math.inf
    v = k.flip(0).contiguous()
    v[80:96] = math.nan
    _same_cache(_write_both(mt, cache, table, k, v, [0, 96], kv), cache)


def test_write_places_that_do_not_exist(mt):
    """Pages of -1 and past the cache, tokens past the table, more rows than
    tokens, rows of no sequence: not written, and nothing else is."""
    g = torch.Generator().manual_seed(13)
    hkv, d = 2, 64
    cache, table = _cache("e4m3", [64, 64, 64, 64], 16, hkv, d, 16, g)
    table[0, 1], table[1, 2] = -1, cache[0].shape[0]
    table[3, 0] = 2 ** 31 - 1
    cu, kv = [2, 52, 112, 212, 220], [50, 64, 70, 5]      # sequence 2: past its 4 pages; 3: 8 rows, 5 tokens
    k = torch.randn(230, hkv, d, generator=g).to(BF16)
    _same_cache(_write_both(mt, cache, table, k, k * 2, cu, kv), cache)


def test_write_strided_rows_and_cache(mt):
    """k and v as slices of a packed qkv, caches as slices of wider rows, int64
    offsets and table, a table that is a slice."""
    g = torch.Generator().manual_seed(17)
    hkv, d, kv, new = 4, 128, [40, 100], [40, 7]
    cache, table = _cache("int8", kv, 32, hkv, d, 16, g)
    pages = cache[0].shape[0]
    packed = torch.randn(sum(new), 3, hkv, d, generator=g).to(F16).cuda()
    wide = torch.zeros(pages, 32, 2, hkv, d, dtype=torch.int8).cuda()
    wide[:, :, 0], wide[:, :, 1] = cache[0].cuda(), cache[1].cuda()
    big = torch.full((2, table.shape[1] + 3), -1, dtype=torch.int64).cuda()
    big[:, :table.shape[1]] = table.cuda()
    got = [wide[:, :, 0], wide[:, :, 1], *_dev(cache[2:])]
    mt.paged_cache_write(packed[:, 1], packed[:, 2], *got, cu_of(new, "cuda").long(), cu_of(kv, "cuda").long(),
                         big[:, :table.shape[1]])
    cu = cu_of(new).tolist()
    cache8.write(cache[0], cache[2], packed[:, 1].cpu(), cu, kv, table)
    cache8.write(cache[1], cache[3], packed[:, 2].cpu(), cu, kv, table)
    _same_cache(got, cache)
    k, v = mt.paged_cache_read(*got, cu_of(new, "cuda").long(), cu_of(kv, "cuda").long(), big[:, :table.shape[1]], 47,
                               dtype=F32)
    assert torch.equal(k.cpu(), cache8.read(cache[0], cache[2], cu, kv, table, 47).float())
    assert torch.equal(v.cpu(), cache8.read(cache[1], cache[3], cu, kv, table, 47).float())


READS = [
    ("e4m3", BF16, 8, 128, 16, 16, None, [1, 0, 17, 700]),
    ("int8", F16, 2, 64, 64, 32, [1, 33, 0], [1, 90, 5]),
    ("int8", F32, 3, 80, 48, 16, [48, 2], [100, 2]),
    ("e4m3", F32, 1, 16, 256, 256, None, [600]),
    ("e4m3", F16, 17, 88, 128, 64, [100, 3], [128, 300]),
    ("int8", BF16, 4, 256, 512, 128, None, [511, 513]),
]


@pytest.mark.parametrize("kind,dt,hkv,d,page,block,rows,kv", READS)
def test_read(mt, kind, dt, hkv, d, page, block, rows, kv):
    """code * scale in fp32, rounded to the type, bit for bit; rows past the last sequence 0."""
    g = torch.Generator().manual_seed(d + page)
    cache, table = _cache(kind, kv, page, hkv, d, block, g)
    cu = cu_of(kv if rows is None else rows)
    total = int(cu[-1]) + 5
    k, v = mt.paged_cache_read(*_dev(cache), cu.cuda(), cu_of(kv, "cuda"), table.cuda(), total, dtype=dt)
    for got, c, s in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        # (the product of a code and an fp32 scale is exact in fp64; its
        # rounding to fp32 comes first, as the kernel's)
        want = cache8.read(c, s, cu.tolist(), kv, table, total).float().to(dt)
        assert got.shape == want.shape and torch.equal(got.cpu(), want)


def test_read_clamps_and_gaps(mt):
    """Pages that do not exist are clamped as the attention clamps them, more
    rows than tokens and rows of no sequence are 0."""
    g = torch.Generator().manual_seed(19)
    cache, table = _cache("int8", [64, 64, 64], 16, 2, 64, 16, g)
    table[0, 1], table[1, 0] = -7, 10 ** 6
    cu, kv, total = [3, 63, 100, 110], [60, 90, 4], 120       # sequence 1: past its 4 pages; 2: 10 rows, 4 tokens
    k, v = mt.paged_cache_read(*_dev(cache), torch.tensor(cu).cuda(), cu_of(kv, "cuda"), table.cuda(), total, dtype=F32)
    for got, c, s in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        assert torch.equal(got.cpu(), cache8.read(c, s, cu, kv, table, total).float())


DECODES = [
    # kind, type, hq, hkv, d, page, block, q lengths, kv lengths, causal, window, bias
    ("e4m3", BF16, 32, 8, 128, 16, 16, [1], [1], True, 0, None),
    ("int8", F16, 8, 8, 64, 16, 16, [1, 1, 1], [0, 1, 15], True, 0, None),
    ("e4m3", F16, 32, 8, 128, 16, 16, [1, 1, 1, 1], [16, 17, 33, 700], True, 0, None),
    ("int8", BF16, 16, 2, 128, 64, 32, [4, 1, 3], [3, 900, 65], True, 0, None),       # a row without keys
    ("e4m3", BF16, 28, 4, 64, 48, 16, [2, 0, 5], [100, 40, 31], False, 0, None),      # groups of 7
    ("int8", F16, 12, 4, 128, 256, 256, [1, 8], [257, 2000], True, 0, None),
    ("e4m3", BF16, 16, 16, 128, 128, 64, [16, 1, 7], [40, 3000, 16], True, 0, None),
    ("int8", BF16, 8, 2, 64, 32, 32, [1, 2, 1], [5000, 3000, 31], True, 100, None),
    ("e4m3", F16, 64, 8, 128, 64, 64, [1, 2], [4097, 2500], True, 1000, None),
    ("int8", BF16, 8, 4, 128, 16, 16, [3, 1], [600, 50], False, 64, None),
    ("e4m3", BF16, 8, 2, 128, 64, 64, [2, 1], [700, 1500], True, 0, "head"),
    ("int8", F16, 8, 8, 64, 16, 16, [1, 3], [70, 40], True, 0, "broadcast"),
    ("e4m3", F16, 8, 2, 64, 32, 16, [1, 4], [400, 130], True, 50, "short"),
    ("int8", BF16, 32, 8, 128, 16, 16, [1] * 70, [33 * i % 1900 for i in range(70)], True, 0, None),
    ("e4m3", BF16, 16, 2, 64, 128, 128, [1, 1], [20000, 9000], True, 0, None),
    ("int8", F16, 8, 1, 128, 256, 128, [5], [30001], True, 0, None),
]


@pytest.mark.parametrize("kind,dt,hq,hkv,d,page,block,ql,kv,causal,window,bias", DECODES)
def test_decode(mt, kind, dt, hq, hkv, d, page, block, ql, kv, causal, window, bias):
    """Outputs and LSE against fp64 attention over the cache's values; the rows
    of the cache that no sequence owns hold NaN codes."""
    g = torch.Generator().manual_seed(hq + d + page)
    cache, table = _cache(kind, kv, page, hkv, d, block, g)
    for c in cache[:2]:
        poison_free_rows(c, kv, table)
    q = torch.randn(sum(ql), hq, d, generator=g).to(dt)
    b = None
    if bias is not None:
        cols = max(kv) - 37 if bias == "short" else max(kv)
        b = torch.randn(sum(ql), hq if bias == "head" else 1, cols, generator=g)
        b[torch.rand(b.shape, generator=g) < 0.3] = -math.inf
        b[0, :, :] = -math.inf                               # a row that nothing is left of
    lse = torch.empty(sum(ql), hq, device="cuda")
    out = mt.paged_decode(q.cuda(), cache[0].cuda(), cache[1].cuda(), cu_of(ql, "cuda"), cu_of(kv, "cuda"), table.cuda(),
                          max(ql), max(kv), causal=causal, window=window, attn_bias=None if b is None else b.cuda(),
                          lse_out=lse, k_scale=cache[2].cuda(), v_scale=cache[3].cuda())
    rb = b
    if bias == "short":                                       # columns past the bias read as 0
        rb = torch.cat([b, torch.zeros(sum(ql), 1, 37)], 2)
    ref = decode_reference(q, cache[0], cache[2], cache[1], cache[3], cu_of(ql).tolist(), kv, table, 1 / math.sqrt(d),
                           causal, window, rb)
    check_decode(out, lse, *ref, dt)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_decode_scale_spread(mt, kind):
    """Blocks whose value scales differ by 2^60, the heavy keys among the small
    values: fp16 queries keep the small values' digits."""
    g = torch.Generator().manual_seed(23)
    kv, hq, hkv, d = [200, 90], 8, 2, 64
    cache, table = _cache(kind, kv, 16, hkv, d, 16, g)
    cache[3] = torch.exp2(torch.randint(-40, 21, cache[3].shape, generator=g).float())
    # each sequence's first block: small values, large scores
    for s in range(2):
        pg = int(table[s, 0])
        cache[3][pg] = 2.0 ** -20
    q = torch.randn(2, hq, d, generator=g).to(F16)
    bias = torch.zeros(2, 1, 200)
    bias[:, :, :16] = 60.0
    lse = torch.empty(2, hq, device="cuda")
    for dt in (F16, BF16):
        qd = q.to(dt)
        out = mt.paged_decode(qd.cuda(), cache[0].cuda(), cache[1].cuda(), cu_of([1, 1], "cuda"), cu_of(kv, "cuda"),
                              table.cuda(), 1, 200, attn_bias=bias.cuda(), lse_out=lse, k_scale=cache[2].cuda(),
                              v_scale=cache[3].cuda())
        check_decode(out, lse, *decode_reference(qd, cache[0], cache[2], cache[1], cache[3], [0, 1, 2], kv, table,
                                                 1 / math.sqrt(d), False, 0, bias), dt)


def test_decode_nan_reaches_its_rows(mt):
    """A NaN code in a key or value that a row sees is NaN in that head, in no other
    sequence."""
    g = torch.Generator().manual_seed(29)
    kv, hq, hkv, d = [300, 70], 8, 2, 128
    cache, table = _cache("e4m3", kv, 32, hkv, d, 32, g)
    raw = cache[0].view(torch.uint8)
    raw[int(table[0, 2]), 5, 1, 7] = 0xff
    q = torch.randn(2, hq, d, generator=g).to(BF16)
    lse = torch.empty(2, hq, device="cuda")
    out = mt.paged_decode(q.cuda(), cache[0].cuda(), cache[1].cuda(), cu_of([1, 1], "cuda"), cu_of(kv, "cuda"),
                          table.cuda(), 1, 300, lse_out=lse, k_scale=cache[2].cuda(), v_scale=cache[3].cuda()).cpu()
    assert bool(torch.isnan(out[0, 4:]).all()) and bool(torch.isnan(lse[0, 4:]).all())
    assert bool(torch.isfinite(out[0, :4]).all()) and bool(torch.isfinite(out[1]).all())


@pytest.mark.parametrize("kind,d,block,page,ql,kv,causal,window,max_kv", [
    ("e4m3", 128, 16, 16, [1, 3, 4], [100, 203, 77], True, 40, 203),
    ("e4m3", 64, 32, 96, [4, 1, 2], [333, 640, 65], True, 50, 640),
    ("e4m3", 128, 16, 64, [2, 4, 4, 1], [2500, 4097, 2, 900], True, 70, 4097),
    ("e4m3", 64, 16, 16, [3, 4], [2100, 61], True, 0, 2100),
    ("int8", 128, 16, 32, [1, 4, 2], [500, 130, 2300], True, 33, 2300),
    ("int8", 64, 64, 64, [1, 1], [700, 2900], False, 128, 2900),
])
def test_decode_masked_garbage(mt, kind, d, block, page, ql, kv, causal, window, max_kv):
    """What a row does not see is not in its result, whatever lies there: NaN codes
    and scales that are no numbers before a window (pages given to other uses), a
    NaN in V at keys that only some rows see."""
    gen = torch.Generator().manual_seed(23)
    hkv, g = 2, 2
    cache, table = _cache(kind, kv, page, hkv, d, block, gen)
    q = torch.randn(sum(ql), hkv * g, d, generator=gen).to(BF16)
    cu = [0]
    for n in ql:
        cu.append(cu[-1] + n)
    ref, ref_lse, bound, lse_bound = decode_reference(q, cache[0], cache[2], cache[1], cache[3], cu, kv, table, d ** -0.5,
                                                      causal, window)
    want_nan = torch.zeros(ref.shape, dtype=torch.bool)
    dirty = _clone(cache)
    raw = [t.view(torch.uint8).flatten(0, 1) for t in dirty[:2]]
    for s, n in enumerate(kv):
        first = max(0, n - ql[s] - window + 1) if window else 0
        at = cache8.rows(table, s, 0, n, page, cache[0].shape[0])
        for r in raw:
            r[at[:first]] = 0x7f if kind == "e4m3" else 0x80
        for b in range(first // block):
            row = int(at[b * block]) // block
            dirty[2].flatten(0, 1)[row] = float("nan")
            dirty[3].flatten(0, 1)[row] = math.inf if b % 2 else float("nan")
        if kind == "e4m3":
            # column 5 of the key before the last, column 9 of a key at the window's start
            for key, col in ((n - 2, 5), (first + 1, 9)):
                raw[1][at[key], 0, col] = 0xff
                for i in range(ql[s]):
                    pos = i + n - ql[s]
                    if (not causal or key <= pos) and (not window or key > pos - window):
                        want_nan[cu[s] + i, :g, col] = True
    lse = torch.empty(q.shape[:2], device="cuda")
    dev = _dev(dirty)
    out = mt.paged_decode(q.cuda(), dev[0], dev[1], torch.tensor(cu, dtype=torch.int32).cuda(), cu_of(kv, "cuda"),
                          table.cuda(), max(ql), max_kv, causal=causal, window=window, lse_out=lse, k_scale=dev[2],
                          v_scale=dev[3]).cpu()
    assert torch.equal(torch.isnan(out), want_nan)
    check_decode(torch.where(want_nan, ref.to(out.dtype), out), lse, ref, ref_lse, bound, lse_bound, BF16)


def test_decode_many_sequences(mt):
    """Equal pieces of more sequences than one scan of them takes, some without
    keys, queries or both, ragged over page ends."""
    gen = torch.Generator().manual_seed(24)
    kv = torch.randint(1, 700, (203,), generator=gen).tolist()
    ql = torch.randint(1, 4, (203,), generator=gen).tolist()
    for i in range(0, 203, 7):
        kv[i] = 0
    for i in range(3, 203, 11):
        ql[i] = 0
    kv[70:134] = [0] * 64
    kv[150], kv[202] = 5000, 2600
    cu = [0]
    for n in ql:
        cu.append(cu[-1] + n)
    for kind, page, block, causal, window in (("e4m3", 48, 16, True, 0), ("int8", 64, 32, False, 300)):
        cache, table = _cache(kind, kv, page, 2, 64, block, gen)
        q = torch.randn(cu[-1], 4, 64, generator=gen).to(F16)
        ref = decode_reference(q, cache[0], cache[2], cache[1], cache[3], cu, kv, table, 0.125, causal, window)
        poison_free_rows(cache[0], kv, table)
        poison_free_rows(cache[1], kv, table)
        lse = torch.empty(q.shape[:2], device="cuda")
        dev = _dev(cache)
        out = mt.paged_decode(q.cuda(), dev[0], dev[1], torch.tensor(cu, dtype=torch.int32).cuda(), cu_of(kv, "cuda"),
                              table.cuda(), 3, 5000, causal=causal, window=window, lse_out=lse, k_scale=dev[2], v_scale=dev[3])
        check_decode(out, lse, *ref, F16)


@pytest.mark.parametrize("kind,max_kv", [("e4m3", 60000), ("int8", 60000), ("e4m3", 1000)])
def test_decode_long_waves(mt, kind, max_kv):
    """More tiles to a wave than one fetch of lookups holds: many sequences over the
    same pages; and a max_seqlen_kv that is too small costs time, no keys."""
    gen = torch.Generator().manual_seed(25)
    kv = [59999, 51200 - 7]
    n = 64 if max_kv > 1000 else 2
    cache, table = _cache(kind, kv, 256, 1, 64, 16, gen)
    q = torch.randn(2 * n, 2, 64, generator=gen).to(BF16)
    ref = decode_reference(q, cache[0], cache[2], cache[1], cache[3], [0, n, 2 * n], kv, table, 0.125)
    lens = [kv[0]] * n + [kv[1]] * n
    lse = torch.empty(q.shape[:2], device="cuda")
    dev = _dev(cache)
    out = mt.paged_decode(q.cuda(), dev[0], dev[1], torch.arange(2 * n + 1, dtype=torch.int32).cuda(), cu_of(lens, "cuda"),
                          table.repeat_interleave(n, 0).cuda(), 1, max_kv, lse_out=lse, k_scale=dev[2], v_scale=dev[3])
    check_decode(out, lse, *ref, BF16)


@pytest.mark.parametrize("d,kv,max_kv", [(128, [300, 41, 512], 512), (64, [300, 41, 512], 512),
                                         (128, [3000, 41, 900], 3000), (64, [2600, 1, 33], 2600)])
def test_c_entry_padded_batch(mt, d, kv, max_kv):
    """The C entry on a padded batch: rows before the first and behind the last
    sequence stay as they were, and a workspace of the size that the query says is
    enough."""
    from mtlattn_amd import capi
    gen = torch.Generator().manual_seed(41)
    cache, table = _cache("e4m3", kv, 64, 4, d, 32, gen)
    dev, dtable = _dev(cache), table.cuda()
    cu = torch.tensor([2, 3, 5, 6], dtype=torch.int32, device="cuda")
    ck = cu_of(kv, "cuda")
    q = torch.randn(9, 8, d, generator=gen).to(BF16).cuda()
    want = mt.paged_decode(q, dev[0], dev[1], cu, ck, dtable, 2, max_kv, causal=True, k_scale=dev[2], v_scale=dev[3])
    p = capi.problem_for(q, dev[0][0], cu, ck, 2, d ** -0.5, causal=True)
    p.total_kv = sum(kv)
    c = capi.Cache8(code=capi.CODE_E4M3, page_size=64, block=32, num_heads_kv=4, head_dim=d, num_pages=dev[0].shape[0],
                    k=dev[0].data_ptr(), k_row_stride=4 * d, v=dev[1].data_ptr(), v_row_stride=4 * d,
                    k_scale=dev[2].data_ptr(), v_scale=dev[3].data_ptr(), block_table=dtable.data_ptr(),
                    block_table_stride=dtable.shape[1])
    import ctypes
    need = capi.lib().mtlattn_decode8_workspace_size(ctypes.byref(p), max_kv)
    assert (need > 0) == (max_kv > 2048)
    ws = torch.full((need + 256,), 0xa5, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 7.0)
    lse = torch.full((9, 8), 7.0, device="cuda")
    capi.call("mtlattn_decode8", p, q.data_ptr(), 8 * d, c, max_kv, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), need,
              torch.cuda.current_stream().cuda_stream)
    assert bool((ws[need:] == 0xa5).all())
    assert torch.equal(out[2:6], want[2:6])
    # (the first of two queries on one key sees none: -inf)
    assert not bool(torch.isnan(lse[2:6]).any()) and bool((lse[2:6] != 7.0).all())
    for t in (out, lse):
        assert bool((t[:2] == 7.0).all()) and bool((t[6:] == 7.0).all())


def test_two_streams_at_once(mt):
    """Calls on two streams at the same time do not meet: each result is that of the
    call alone, bit for bit."""
    gen = torch.Generator().manual_seed(42)
    work = []
    for kind, kv in (("e4m3", [2500, 700, 3000, 64]), ("int8", [1000, 2900, 17])):
        cache, table = _cache(kind, kv, 32, 8, 128, 32, gen)
        q = torch.randn(len(kv), 16, 128, generator=gen).to(BF16).cuda()
        dev = _dev(cache)
        args = (q, dev[0], dev[1], cu_of([1] * len(kv), "cuda"), cu_of(kv, "cuda"), table.cuda(), 1, max(kv))
        kw = dict(causal=True, k_scale=dev[2], v_scale=dev[3])
        work.append((args, kw, mt.paged_decode(*args, **kw)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, (args, kw, _) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                got[i].append(mt.paged_decode(*args, **kw))
    torch.cuda.synchronize()
    for i, (_, _, want) in enumerate(work):
        for out in got[i]:
            assert torch.equal(out, want)


@pytest.mark.parametrize("kv,max_kv", [([100, 333], 333), ([2100, 70], 2100)])
def test_decode_mask_by_sequence(mt, kv, max_kv):
    """A 4-D bias, indexed by sequence and sequence-local row: the result of the same
    bias row by row, bit for bit. Keys at -inf for every row of a sequence's head
    leave the row empty."""
    gen = torch.Generator().manual_seed(43)
    cache, table = _cache("int8", kv, 16, 2, 64, 16, gen)
    q = torch.randn(4, 4, 64, generator=gen).to(F16).cuda()
    bias = torch.randn(2, 4, 2, max_kv, generator=gen)
    bias[1, 2, 1] = -math.inf
    rows = bias.permute(0, 2, 1, 3).reshape(4, 4, max_kv).contiguous()
    dev = _dev(cache)
    outs = []
    for b in (bias, rows):
        lse = torch.empty(4, 4, device="cuda")
        out = mt.paged_decode(q, dev[0], dev[1], cu_of([2, 2], "cuda"), cu_of(kv, "cuda"), table.cuda(), 2, max_kv,
                              attn_bias=b.cuda(), lse_out=lse, k_scale=dev[2], v_scale=dev[3])
        outs.append((out, lse))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert bool((outs[0][0][3, 2] == 0).all()) and float(outs[0][1][3, 2]) == -math.inf
    ref = decode_reference(q.cpu(), cache[0], cache[2], cache[1], cache[3], [0, 2, 4], kv, table, 0.125, False, 0, rows)
    check_decode(outs[0][0], outs[0][1], *ref, F16)


@pytest.mark.parametrize("kv", [[3, 700, 5, 0], [3, 2500, 5, 0]])
def test_decode_largest_window(mt, kv):
    """A window of any size that no key lies before, with sequences shorter than
    their queries: the result without a window."""
    gen = torch.Generator().manual_seed(44)
    cache, table = _cache("e4m3", kv, 32, 2, 64, 32, gen)
    ql = [4, 2, 4, 3]
    q = torch.randn(sum(ql), 4, 64, generator=gen).to(BF16).cuda()
    dev = _dev(cache)
    outs = [mt.paged_decode(q, dev[0], dev[1], cu_of(ql, "cuda"), cu_of(kv, "cuda"), table.cuda(), 4, max(kv),
                            causal=True, window=w, k_scale=dev[2], v_scale=dev[3]) for w in (0, 2**31 - 1, 2**40)]
    check = decode_reference(q.cpu(), cache[0], cache[2], cache[1], cache[3], cu_of(ql).tolist(), kv, table, 0.125, True)
    for out in outs:
        check_decode(out, None, *check, BF16)


def test_decode_too_small_max_seqlen_q(mt):
    """Query rows past what max_seqlen_q promised are NaN, the others right --
    both where a workgroup takes whole sequences and where they are cut."""
    for kv in ([40, 64], [9000, 7000]):
        g = torch.Generator().manual_seed(31)
        hq, hkv, d, ql = 8, 1, 64, [5, 1]
        cache, table = _cache("int8", kv, 64, hkv, d, 64, g)
        q = torch.randn(6, hq, d, generator=g).to(BF16)
        lse = torch.zeros(6, hq, device="cuda")
        out = mt.paged_decode(q.cuda(), cache[0].cuda(), cache[1].cuda(), cu_of(ql, "cuda"), cu_of(kv, "cuda"),
                              table.cuda(), 1, max(kv), causal=True, lse_out=lse, k_scale=cache[2].cuda(),
                              v_scale=cache[3].cuda()).cpu()
        ref = decode_reference(q, cache[0], cache[2], cache[1], cache[3], [0, 5, 6], kv, table, 1 / math.sqrt(d), True)
        # 8 heads of one query to a group of 16: n = head * 5 + query < 16 is computed
        done = (torch.arange(hq)[None, :] * 5 + torch.arange(5)[:, None]) < 16
        done = torch.cat([done, torch.ones(1, hq, dtype=torch.bool)])
        assert bool(torch.isnan(out[~done]).all()) and bool(torch.isnan(lse.cpu()[~done]).all())
        check_decode(out[done], lse.cpu()[done], ref[0][done], ref[1][done], ref[2][done], ref[3][done], BF16)


def test_decode_strided_query_and_cache(mt):
    """q as a slice of a packed qkv, K and V caches interleaved in one tensor."""
    g = torch.Generator().manual_seed(37)
    kv, hkv, d = [500, 33], 4, 128
    cache, table = _cache("e4m3", kv, 64, hkv, d, 32, g)
    qkv = torch.randn(2, 3, hkv, d, generator=g).to(BF16)
    wide = torch.stack([cache[0].view(torch.uint8), cache[1].view(torch.uint8)], 2).cuda().view(torch.float8_e4m3fn)
    out = mt.paged_decode(qkv.cuda()[:, 0], wide[:, :, 0], wide[:, :, 1], cu_of([1, 1], "cuda"), cu_of(kv, "cuda"),
                          table.cuda(), 1, 500, k_scale=cache[2].cuda(), v_scale=cache[3].cuda())
    ref = decode_reference(qkv[:, 0], cache[0], cache[2], cache[1], cache[3], [0, 1, 2], kv, table, 1 / math.sqrt(d))
    check_decode(out, None, *ref, BF16)


def test_offsets_past_32_bits(mt):
    """A cache of 4.5 GB a side whose last pages are in use."""
    hkv, d, page = 16, 128, 256
    pages = (9 << 29) // (hkv * d * page)
    g = torch.Generator().manual_seed(41)
    kv = [300, 40]
    small, table = _cache("int8", kv, page, hkv, d, 64, g)
    n = small[0].shape[0]
    dev = [torch.empty(pages, page, hkv, d, dtype=torch.int8, device="cuda") for _ in range(2)]
    dev += [torch.empty(pages, page // 64, hkv, device="cuda") for _ in range(2)]
    for a, b in zip(dev, small):
        a[pages - n:] = b.cuda()
    far = (table + pages - n).cuda()
    k = torch.randn(5, hkv, d, generator=g).to(BF16)
    mt.paged_cache_write(k.cuda(), -k.cuda(), *dev, cu_of([3, 2], "cuda"), cu_of(kv, "cuda"), far)
    cache8.write(small[0], small[2], k, [0, 3, 5], kv, table)
    cache8.write(small[1], small[3], -k, [0, 3, 5], kv, table)
    _same_cache([t[pages - n:] for t in dev], small)
    got, _ = mt.paged_cache_read(*dev, cu_of(kv, "cuda"), cu_of(kv, "cuda"), far, 340)
    assert torch.equal(got.cpu(), cache8.read(small[0], small[2], [0, 300, 340], kv, table, 340).float().to(BF16))
    q = torch.randn(2, 32, d, generator=g).to(BF16)
    out = mt.paged_decode(q.cuda(), dev[0], dev[1], cu_of([1, 1], "cuda"), cu_of(kv, "cuda"), far, 1, 300,
                          k_scale=dev[2], v_scale=dev[3])
    check_decode(out, None, *decode_reference(q, small[0], small[2], small[1], small[3], [0, 1, 2], kv, table,
                                              1 / math.sqrt(d)), BF16)


def test_empty_calls(mt):
    g = torch.Generator().manual_seed(43)
    cache, table = _cache("e4m3", [20], 16, 2, 64, 16, g)
    dev = _dev(cache)
    none = torch.empty(0, 2, 64, dtype=BF16, device="cuda")
    zero = cu_of([0], "cuda")
    mt.paged_cache_write(none, none, *dev, zero, cu_of([20], "cuda"), table.cuda())
    _same_cache(dev, cache)
    k, v = mt.paged_cache_read(*dev, zero, cu_of([20], "cuda"), table.cuda(), 0)
    assert k.shape == (0, 2, 64) and k.dtype == BF16
    out = mt.paged_decode(none, dev[0], dev[1], zero, cu_of([20], "cuda"), table.cuda(), 1, 20, k_scale=dev[2],
                          v_scale=dev[3])
    assert out.shape == (0, 2, 64)


def test_binding_refusals(mt):
    """What needs GPU tensors to be refused; nothing is launched."""
    q = torch.zeros(1, 8, 128, dtype=BF16, device="cuda")
    k = torch.zeros(1, 2, 128, dtype=BF16, device="cuda")
    codes = torch.zeros(2, 32, 2, 128, dtype=torch.int8, device="cuda")
    sc = torch.ones(2, 2, 2, device="cuda")
    cu, table = cu_of([1], "cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")

    def attend(q=q, kc=codes, vc=codes, ks=sc, vs=sc, cu_q=cu, table=table, mq=1, mkv=1, **kw):
        return mt.paged_decode(q, kc, vc, cu_q, cu, table, mq, mkv, k_scale=ks, v_scale=vs, **kw)

    def write(k=k, v=k, kc=codes, vc=codes, ks=sc, vs=sc, cu=cu, table=table):
        mt.paged_cache_write(k, v, kc, vc, ks, vs, cu, cu, table)

    e4 = codes.view(torch.float8_e4m3fn)
    for kw, text in ((dict(kc=codes.half()), "8-bit cache"), (dict(vc=e4), "8-bit cache"),
                     (dict(kc=codes[:1], vc=codes[:1]), "k_scale"), (dict(ks=sc.double()), "k_scale"),
                     (dict(vs=sc[:, :1]), "k_scale"), (dict(ks=sc.transpose(1, 2)), "k_scale"),
                     (dict(ks=torch.ones(2, 3, 2, device="cuda"), vs=torch.ones(2, 3, 2, device="cuda")), "k_scale"),
                     (dict(ks=torch.ones(2, 4, 2, device="cuda"), vs=torch.ones(2, 4, 2, device="cuda")), "tokens per scale"),
                     (dict(ks=sc.cpu()), "same device"), (dict(table=table.repeat(2, 1)), "block_table"),
                     (dict(kc=codes.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous")):
        with pytest.raises(RuntimeError, match=text):
            attend(**kw)
        with pytest.raises(RuntimeError, match=text):
            write(**kw)
    for kw, text in ((dict(mkv=65), "block_table has 2 pages"), (dict(q=q[:, :7]), "multiple of kv heads"),
                     (dict(q=q[:, :, :64].contiguous()), "head dim"), (dict(q=q.float()), "half/bf16"),
                     (dict(mq=17), "max_seqlen_q"), (dict(cu_q=cu_of([1, 0], "cuda")), "cu_seqlens"),
                     (dict(lse_out=torch.empty(2, 8, device="cuda")), "lse_out")):
        with pytest.raises(RuntimeError, match=text):
            attend(**kw)
    for kw, text in ((dict(k=k.half()), "dtype"), (dict(k=k[:, :1], v=k[:, :1]), "heads"),
                     (dict(k=k.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous")):
        with pytest.raises(RuntimeError, match=text):
            write(**kw)
    with pytest.raises(RuntimeError, match="total"):
        mt.paged_cache_read(codes, codes, sc, sc, cu, cu, table, -1)


# ---- graphs, streams, and the operators together ----

class _Server:
    """A batch of sequences over an 8-bit cache, and the same K/V in fp64."""

    def __init__(self, mt, kind, block=16, page=32, hq=8, hkv=2, d=64, batch=3, room=12, dt=BF16, seed=0):
        self.mt, self.kind, self.dt, self.hq, self.hkv, self.d = mt, kind, dt, hq, hkv, d
        self.g = torch.Generator().manual_seed(seed)
        perm = torch.randperm(batch * room + 3, generator=self.g).to(torch.int32)
        self.table = perm[:batch * room].view(batch, room)
        n = batch * room + 3
        self.cpu = [torch.zeros(n, page, hkv, d).to(CODES[kind]) for _ in range(2)]
        self.cpu += [torch.zeros(n, page // block, hkv) for _ in range(2)]
        self.dev = _dev(self.cpu)
        self.lens = [0] * batch
        self.dtable = self.table.cuda()

    def rand(self, n, h):
        return torch.randn(n, h, self.d, generator=self.g).to(self.dt)

    def append(self, new):
        """New tokens of each sequence, written on the GPU and by the oracle."""
        k, v = self.rand(sum(new), self.hkv), self.rand(sum(new), self.hkv)
        self.lens = [a + b for a, b in zip(self.lens, new)]
        cu = cu_of(new)
        self.mt.paged_cache_write(k.cuda(), v.cuda(), *self.dev, cu.cuda(), cu_of(self.lens, "cuda"), self.dtable)
        cache8.write(self.cpu[0], self.cpu[2], k, cu.tolist(), self.lens, self.table)
        cache8.write(self.cpu[1], self.cpu[3], v, cu.tolist(), self.lens, self.table)

    def reference(self, q, new):
        return decode_reference(q, self.cpu[0], self.cpu[2], self.cpu[1], self.cpu[3], cu_of(new).tolist(), self.lens,
                                self.table, 1 / math.sqrt(self.d), True)

    def decode(self, q, new):
        return self.mt.paged_decode(q.cuda(), self.dev[0], self.dev[1], cu_of(new, "cuda"), cu_of(self.lens, "cuda"),
                                    self.dtable, max(new), max(self.lens), causal=True, k_scale=self.dev[2],
                                    v_scale=self.dev[3])


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_serving_run(mt, kind):
    """Prompts written and read back for a prompt's next chunk (varlen_attention
    over what the cache holds), then tokens written and attended one to three at a
    time."""
    s = _Server(mt, kind)
    s.append([50, 33, 128])
    chunk = [40, 0, 70]
    s.append(chunk)
    q = s.rand(sum(chunk), s.hq)
    total = sum(s.lens)
    ck = cu_of(s.lens, "cuda")
    k, v = mt.paged_cache_read(*s.dev, ck, ck, s.dtable, total, dtype=s.dt)
    out = mt.varlen_attention(q.cuda(), k, v, cu_of(chunk, "cuda"), ck, max(chunk), causal=True)
    # the forward rounds the read values and its weights to bf16: 2^-8 each of
    # sum p |v| (scores: 2^-8 of sum |q k| / 8, about 2 at most here, twice)
    ref, _, bound, _ = s.reference(q, chunk)
    size = cache8.values(s.cpu[1], s.cpu[3]).abs().max()
    assert float((out.cpu().double() - ref).abs().max()) <= float(bound.max()) + size * 2.0 ** -8 * 6
    for step in range(6):
        new = [1 + step % 3, 1, 2]
        s.append(new)
        q = s.rand(sum(new), s.hq)
        ref = s.reference(q, new)
        check_decode(s.decode(q, new), None, *ref, s.dt)
    _same_cache(s.dev, s.cpu)


def test_other_stream(mt):
    """All three on a stream that is not the tensors' own, waited for as usual."""
    s = _Server(mt, "int8", seed=5)
    s.append([200, 64, 31])
    q = s.rand(3, s.hq)
    ref = s.reference(q, [1, 1, 1])
    qd, cq, ck = q.cuda(), cu_of([1, 1, 1], "cuda"), cu_of(s.lens, "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = mt.paged_decode(qd, s.dev[0], s.dev[1], cq, ck, s.dtable, 1, max(s.lens), causal=True, k_scale=s.dev[2],
                              v_scale=s.dev[3])
        k, _ = mt.paged_cache_read(*s.dev, ck, ck, s.dtable, sum(s.lens), dtype=F32)
    torch.cuda.current_stream().wait_stream(side)
    check_decode(out, None, *ref, BF16)
    assert torch.equal(k.cpu(), cache8.read(s.cpu[0], s.cpu[2], cu_of(s.lens).tolist(), s.lens, s.table,
                                            sum(s.lens)).float())


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_graph_decode_step(mt, kind):
    """A step -- write, attend -- captured once and replayed as the sequences
    grow, its lengths and rows changed in place, eager work between; then a
    second graph over the same cache, replayed in turn with it."""
    s = _Server(mt, kind, room=20, seed=9)
    s.append([250, 7, 90])
    B, top = 3, 20 * 32
    cq = cu_of([1] * B, "cuda")
    k, v = torch.zeros(B, s.hkv, s.d, dtype=BF16, device="cuda"), torch.zeros(B, s.hkv, s.d, dtype=BF16, device="cuda")
    q, ck = torch.zeros(B, s.hq, s.d, dtype=BF16, device="cuda"), cu_of(s.lens, "cuda")

    def step():
        mt.paged_cache_write(k, v, *s.dev, cq, ck, s.dtable)
        return mt.paged_decode(q, s.dev[0], s.dev[1], cq, ck, s.dtable, 1, top, causal=True, k_scale=s.dev[2],
                               v_scale=s.dev[3])

    # (the captured call itself does not run; the warm-up writes into pages that a
    # later write takes over)
    keep = _clone(s.dev)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    for a, b in zip(s.dev, keep):
        a.copy_(b)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for i in range(6):
        nk, nv, nq = s.rand(B, s.hkv), s.rand(B, s.hkv), s.rand(B, s.hq)
        s.lens = [x + 1 for x in s.lens]
        cache8.write(s.cpu[0], s.cpu[2], nk, [0, 1, 2, 3], s.lens, s.table)
        cache8.write(s.cpu[1], s.cpu[3], nv, [0, 1, 2, 3], s.lens, s.table)
        k.copy_(nk), v.copy_(nv), q.copy_(nq), ck.copy_(cu_of(s.lens))
        gr, out = graphs[i % 2]
        gr.replay()
        check_decode(out, None, *s.reference(nq, [1] * B), BF16)
        eager = s.decode(nq, [1] * B)
        torch.cuda.synchronize()
        check_decode(eager, None, *s.reference(nq, [1] * B), BF16)
    _same_cache(s.dev, s.cpu)


def test_repeatable(mt):
    """The same call gives the same bits."""
    s = _Server(mt, "e4m3", batch=2, room=200, seed=13)
    s.append([6000, 3000])
    q = s.rand(2, s.hq)
    first = s.decode(q, [1, 1])
    for _ in range(3):
        assert torch.equal(s.decode(q, [1, 1]), first)
