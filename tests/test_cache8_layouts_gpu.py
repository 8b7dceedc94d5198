"""Decode over the 8-bit K/V cache in every layout of its work, against the fp64
oracle; writing and reading for batches of more sequences than a wave has lanes."""

import ctypes
import math

import pytest
import torch

from mtlattn_amd import capi
from oracle import cache8
from tests import cache8_layouts
from tests.cache8_helpers import check_decode, decode_reference, pages_for, poison_free_rows, random_cache, same_codes
from tests.helpers import cu_of

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mt():
    import mtlattn
    return mtlattn


def _offsets(lens, start=0):
    c = [start]
    for n in lens:
        c.append(c[-1] + n)
    return c


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("name", cache8_layouts.CASES)
def test_decode(mt, name):
    """Outputs and LSE; rows of the cache that no sequence owns hold NaN codes."""
    kind, dt, hq, hkv, d, page, block, n, most, longest, window, bias, want = cache8_layouts.CASES[name]
    assert cache8_layouts.layout(name) == want
    dt = BF16 if dt == "bf16" else F16
    ql, kv = cache8_layouts.lengths(name)
    g = torch.Generator().manual_seed(n)
    table, pages = pages_for(kv, page, g)
    kc, ks = random_cache(kind, pages, page, hkv, d, block, g)
    vc, vs = random_cache(kind, pages, page, hkv, d, block, g)
    for c in (kc, vc):
        poison_free_rows(c, kv, table)
    q = torch.randn(sum(ql), hq, d, generator=g).to(dt)
    b = None
    if bias is not None:
        b = torch.randn(sum(ql), hq if bias == "head" else 1, longest, generator=g)
        b[torch.rand(b.shape, generator=g) < 0.3] = -math.inf
        b[1] = -math.inf                                         # a row that nothing is left of
    cu = _offsets(ql)
    ref = decode_reference(q, kc, ks, vc, vs, cu, kv, table, d ** -0.5, True, window, b)
    lse = torch.empty(sum(ql), hq, device="cuda")
    args = (q.cuda(), kc.cuda(), vc.cuda(), _int32(cu), cu_of(kv, "cuda"), table.cuda(), most, longest)
    kw = dict(causal=True, window=window, attn_bias=None if b is None else b.cuda(), lse_out=lse, k_scale=ks.cuda(),
              v_scale=vs.cuda())
    out = mt.paged_decode(*args, **kw)
    check_decode(out, lse, *ref, dt)
    assert torch.equal(mt.paged_decode(*args, **kw), out)


def _batch(n, gen):
    """(new tokens, lengths) of n sequences: some without either, runs of 64 without
    new tokens, blocks that hold earlier tokens and blocks that do not."""
    kv = torch.randint(1, 90, (n,), generator=gen).tolist()
    new = [int(torch.randint(1, min(x, 40) + 1, (1,), generator=gen)) for x in kv]
    for i in range(0, n, 5):
        new[i] = 1
    for i in range(2, n, 9):
        new[i] = 0
    for i in range(4, n, 13):
        new[i] = kv[i]
    for i in range(7, n, 17):
        kv[i] = new[i] = 0
    if n > 200:
        new[64:130] = [0] * 66
        new[n - 66:n - 1] = [0] * 65
    return new, kv


@pytest.mark.parametrize("n", [64, 65, 128, 129, 330])
@pytest.mark.parametrize("kind,dt", [("e4m3", BF16), ("int8", F32)])
def test_write_and_read_many_sequences(mt, n, kind, dt):
    """More sequences than a wave's lanes, bit for bit: a gap before the first row and
    rows behind the last sequence."""
    g = torch.Generator().manual_seed(n)
    new, kv = _batch(n, g)
    page, block, hkv, d = 32, 16, 2, 32
    table, pages = pages_for(kv, page, g)
    cache = []
    for _ in range(2):
        cache += random_cache(kind, pages, page, hkv, d, block, g)
    cache = [cache[0], cache[2], cache[1], cache[3]]
    cu = _offsets(new, 3)
    rows = [torch.randn(cu[-1] + 6, hkv, d, generator=g).to(dt) for _ in range(2)]
    dev = [t.cuda() for t in cache]
    mt.paged_cache_write(rows[0].cuda(), rows[1].cuda(), *dev, _int32(cu), cu_of(kv, "cuda"), table.cuda())
    for x in (0, 1):
        cache8.write(cache[x], cache[2 + x], rows[x], cu, kv, table)
        assert torch.equal(dev[2 + x].cpu(), cache[2 + x]) and same_codes(dev[x], cache[x])
    for lens in (new, kv):
        at = _offsets(lens, 5)
        total = at[-1] + 9
        got = mt.paged_cache_read(*dev, _int32(at), cu_of(kv, "cuda"), table.cuda(), total, dtype=dt)
        for x in (0, 1):
            want = cache8.read(cache[x], cache[2 + x], at, kv, table, total).float().to(dt)
            assert torch.equal(got[x].cpu(), want)


def test_malformed_offsets_stay_in_the_workspace(mt):
    """KV offsets that go up and down claim more keys in all than an int counts (a
    multiple of 2^32 less 2^17 units of 32): the call ends, writes nothing but its
    rows, and calls after it are right."""
    n, hq, hkv, d, page = 128, 8, 8, 64, 256
    g = torch.Generator().manual_seed(61)
    kv = [700, 40]
    table, pages = pages_for(kv, page, g)
    kc, ks = random_cache("int8", pages, page, hkv, d, 64, g)
    vc, vs = random_cache("int8", pages, page, hkv, d, 64, g)
    dev = [t.cuda() for t in (kc, vc, ks, vs)]
    wide = torch.zeros(n, 4, dtype=torch.int32, device="cuda")
    cu_kv = torch.tensor([0, 2 ** 31 - 1] * (n // 2) + [0], dtype=torch.int32, device="cuda")
    q = torch.randn(n + 2, hq, d, generator=g).to(BF16).cuda()
    cu = torch.arange(1, n + 2, dtype=torch.int32, device="cuda")
    p = capi.problem_for(q, dev[0][0], cu, cu_kv, 1, d ** -0.5, causal=True)
    p.total_kv = 2 ** 31 - 1
    x = [ctypes.c_int32() for _ in range(3)]
    capi.call("mtlattn_decode8_layout", ctypes.byref(p), 100000, *[ctypes.byref(i) for i in x])
    assert x[0].value == x[1].value and x[2].value > 0      # (a unit is 32 keys, so that the sum wraps to -2^17)
    keys = min(2 ** 31 - 1, 0x7fff0000)
    assert ((n // 2) * -(-keys // 32)) % 2 ** 32 == 2 ** 32 - 2 ** 17
    c = capi.Cache8(code=capi.CODE_INT8, page_size=page, block=64, num_heads_kv=hkv, head_dim=d, num_pages=pages,
                    k=dev[0].data_ptr(), k_row_stride=hkv * d, v=dev[1].data_ptr(), v_row_stride=hkv * d,
                    k_scale=dev[2].data_ptr(), v_scale=dev[3].data_ptr(), block_table=wide.data_ptr(),
                    block_table_stride=wide.shape[1])
    need = capi.lib().mtlattn_decode8_workspace_size(ctypes.byref(p), 100000)
    ws = torch.zeros(need + 256, dtype=torch.uint8, device="cuda")
    ws[need:] = 0xa5
    out = torch.full_like(q, 7.0)
    lse = torch.full((n + 2, hq), 7.0, device="cuda")
    capi.call("mtlattn_decode8", p, q.data_ptr(), hq * d, c, 100000, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), need,
              torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0xa5).all())
    for t in (out, lse):
        assert bool((t[0] == 7.0).all()) and bool((t[n + 1] == 7.0).all())
    # every partial of the workspace is 0, and so are the rows that are written from it
    assert bool(((out[1:n + 1] == 0) | (out[1:n + 1] == 7.0)).all())
    out = mt.paged_decode(q[:2], dev[0], dev[1], cu_of([1, 1], "cuda"), cu_of(kv, "cuda"), table.cuda(), 1, 700,
                          causal=True, k_scale=dev[2], v_scale=dev[3])
    check_decode(out, None, *decode_reference(q[:2].cpu(), kc, ks, vc, vs, [0, 1, 2], kv, table, d ** -0.5, True), BF16)
