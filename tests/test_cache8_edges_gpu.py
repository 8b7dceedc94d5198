"""The 8-bit paged K/V cache on the GPU where its arithmetic and its index code
are at their edges: weights next to each other, quotients next to ties, scales of
the caller's own."""

import math

import pytest
import torch

from oracle import cache8
from tests.cache8_helpers import CODES, check_decode, decode_reference, pages_for, random_cache, same_codes
from tests.helpers import cu_of

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mt():
    import mtlattn
    return mtlattn


def _dev(ts):
    return [t.cuda() for t in ts]


def _offsets(lens, start=0):
    c = [start]
    for n in lens:
        c.append(c[-1] + n)
    return c


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_decode_weights_in_32_bits(mt, kind, dt):
    """Two keys of nearly the same score and opposite values: the result is the
    difference of two weights, of which the output's rounding leaves every digit.

    With scores of at most 2^-7 in sum |q k| the bound of what is left, relative to
    sum p |v|: the scores (d + 8) 2^-24 2^-7, twice; exp2 and the base's subtraction
    2^-22 a weight, and as much in the sum of weights; a weight times its scale
    2^-24; two keys of three products each and the sums of those, 8 roundings of
    2^-23; the division and the product with it, 2^-22: 2^-20 + 2^-23.8 + what the
    weights lose on their way. A weight of 16 bits loses up to 2^-18, which is
    four times that."""
    g = torch.Generator().manual_seed(51)
    n, hq, hkv, d = 64, 16, 8, 64
    kv = [2] * n
    table, pages = pages_for(kv, 16, g)
    codes = torch.randint(-8, 9, (2, pages, 16, hkv, d), generator=g).float()
    codes[0, :, 1] = codes[0, :, 0]
    codes[0, :, 1, :, 5] += 1
    codes[1, :, 1] = -codes[1, :, 0]
    kc, vc = (c.to(CODES[kind]) for c in codes)
    ks = torch.full((pages, 1, hkv), 2.0 ** -14)
    vs = 0.5 + torch.rand(pages, 1, hkv, generator=g)
    q = torch.randn(n, hq, d, generator=g).to(dt)
    assert float((q.double().abs().sum(-1) * 8 * 2.0 ** -14 / 8).max()) <= 2.0 ** -7
    out = mt.paged_decode(q.cuda(), kc.cuda(), vc.cuda(), cu_of([1] * n, "cuda"), cu_of(kv, "cuda"), table.cuda(), 1, 2,
                          k_scale=ks.cuda(), v_scale=vs.cuda())
    ref, ref_lse, _, _ = decode_reference(q, kc, ks, vc, vs, _offsets([1] * n), kv, table, 1 / math.sqrt(d))
    size = cache8.values(vc, vs).view(pages, 16, hkv, d)[table[:, 0].long(), 0].abs().repeat_interleave(hq // hkv, 1)
    bound = (2.0 ** -20 + 2.0 ** -23.8 + 2.0 ** -24) * size
    check_decode(out, None, ref, ref_lse, bound, None, dt)


def _by_definition(q, kc, ks, vc, vs, ql, kv, table, causal, window, bias=None):
    """fp64 attention, each row over the keys that it sees and no others (an
    infinite value times the weight of a key that is not seen is no term)."""
    page, pages = kc.shape[1], kc.shape[0]
    k, v = cache8.values(kc, ks), cache8.values(vc, vs)
    g = q.shape[1] // kc.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    row = 0
    for s, n in enumerate(kv):
        at = cache8.rows(table, s, 0, n, page, pages)
        for i in range(ql[s]):
            end = i + n - ql[s]
            lo = max(0, end - window + 1) if window else 0
            see = at[lo:end + 1 if causal else n]
            for h in range(q.shape[1]):
                x = (k[see, h // g] * q[row, h].double()).sum(-1) / math.sqrt(q.shape[2])
                if bias is not None:
                    x = x + bias[row, 0, lo:lo + len(see)].double()
                p = torch.softmax(x, 0)
                out[row, h] = (p[:, None] * v[see, h // g]).sum(0)
            row += 1
    return out


@pytest.mark.parametrize("kind,dt,d,block,page,ql,kv,causal,window,biased", [
    ("e4m3", BF16, 128, 16, 16, [1, 4, 2], [100, 203, 31], True, 0, False),
    ("e4m3", F16, 64, 32, 96, [4, 1, 3], [333, 640, 65], True, 50, False),
    ("int8", BF16, 128, 16, 64, [2, 4, 1], [2500, 70, 900], True, 70, False),
    ("int8", F16, 64, 64, 64, [1, 3], [700, 2900], False, 0, False),
    ("e4m3", BF16, 64, 16, 48, [3, 1, 2], [200, 77, 3000], True, 0, True),
    ("int8", F16, 128, 32, 32, [2, 4], [400, 64], True, 90, True),
])
def test_decode_infinite_value_scales(mt, kind, dt, d, block, page, ql, kv, causal, window, biased):
    """A caller's own value scale that is an infinity gives what the definition
    gives, an infinity or, where signs meet or a code or a weight is 0, a NaN; also
    in a block whose other keys the row does not see."""
    gen = torch.Generator().manual_seed(53)
    hkv, g = 2, 2
    table, pages = pages_for(kv, page, gen)
    kc, ks = random_cache(kind, pages, page, hkv, d, block, gen)
    vc, vs = random_cache(kind, pages, page, hkv, d, block, gen)
    ks *= 2.0 ** -4 if kind == "e4m3" else 2.0 ** -2             # (no weight of a seen key underflows)
    # half of the columns have one sign, so that infinities stay
    mag = vc.float().abs()
    mag[..., ::2] = mag[..., ::2].clamp(min=1)
    vc = torch.where(torch.arange(d) % 2 == 0, mag, vc.float()).to(vc.dtype)
    flat = vs.flatten(0, 1)
    for s, n in enumerate(kv):
        if s == 1:                                              # (a sequence without)
            continue
        first = max(0, n - ql[s] - window + 1) if window else 0
        # the last block, which the sequence fills in part, and the first that a row sees
        for key, x in ((n - 1, math.inf), (first, -math.inf if s == 2 else math.inf)):
            flat[int(cache8.rows(table, s, key, key + 1, page, pages)[0]) // block, 0] = x
    q = torch.randn(sum(ql), hkv * g, d, generator=gen).to(dt)
    cu = _offsets(ql)
    bias = None
    if biased:                      # (the first sequence's second row: weights of 0 among its infinite values)
        bias = torch.randn(sum(ql), 1, max(kv), generator=gen)
        bias[1, 0, kv[0] - 5:] = -math.inf
    ref = _by_definition(q, kc, ks, vc, vs, ql, kv, table, causal, window, bias)
    clean = torch.where(torch.isinf(vs), torch.ones_like(vs), vs)
    _, _, bound, _ = decode_reference(q, kc, ks, vc, clean, cu, kv, table, d ** -0.5, causal, window, bias)
    assert all(int(f(ref).sum()) >= d for f in (torch.isinf, torch.isnan, torch.isfinite))
    out = mt.paged_decode(q.cuda(), kc.cuda(), vc.cuda(), _int32(cu), cu_of(kv, "cuda"), table.cuda(), max(ql), max(kv),
                          causal=causal, window=window, attn_bias=None if bias is None else bias.cuda(), k_scale=ks.cuda(),
                          v_scale=vs.cuda()).cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(out[inf].double(), ref[inf]) and not bool(torch.isinf(out[~inf]).any())
    fin = torch.isfinite(ref)
    check_decode(out[fin], None, ref[fin], None, bound[fin], None, dt)


def test_decode_largest_value_scales(mt):
    """Value scales up to the largest float beside small codes: a weight of 1 times
    the scale is above bf16's largest value, the result is not."""
    gen = torch.Generator().manual_seed(54)
    kv, hkv, d = [1, 40], 2, 64
    table, pages = pages_for(kv, 16, gen)
    kc, ks = random_cache("e4m3", pages, 16, hkv, d, 16, gen)
    vc = (torch.randint(-3, 4, (pages, 16, hkv, d), generator=gen) * 2.0 ** -9).to(torch.float8_e4m3fn)
    vs = torch.full((pages, 1, hkv), torch.finfo(F32).max)
    vs[::2] = -torch.finfo(F32).max
    q = torch.randn(2, 4, d, generator=gen).to(BF16)
    out = mt.paged_decode(q.cuda(), kc.cuda(), vc.cuda(), cu_of([1, 1], "cuda"), cu_of(kv, "cuda"), table.cuda(), 1, 40,
                          k_scale=ks.cuda(), v_scale=vs.cuda())
    ref, ref_lse, bound, _ = decode_reference(q, kc, ks, vc, vs, [0, 1, 2], kv, table, d ** -0.5)
    check_decode(out, None, ref, ref_lse, bound, None, BF16)


def _next_to(x, gen):
    """fp32 values at x (fp64, exact), rounded, and up to one step to either side."""
    y = x.float()
    step = torch.randint(-1, 2, y.shape, generator=gen, dtype=torch.int32)
    return (y.view(torch.int32) + step).view(F32)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_write_next_to_ties_of_held_scales(mt, kind, dt):
    """Tokens into blocks that hold earlier ones at scales of the caller's own, any
    fp32 value: quotients less than an fp32 rounding from a tie, for new codes where
    the held scale stays and for the held ones where it grows."""
    g = torch.Generator().manual_seed(57)
    n, hkv, d, block = 24, 4, 64, 16
    kv, new = [16] * n, [8] * n
    table, pages = pages_for(kv, block, g)
    cache = []
    top = cache8.QMAX[CODES[kind]]
    for _ in range(2):
        codes, _ = random_cache(kind, pages, block, hkv, d, block, g)
        # scales m 2^e: e4m3 keeps those with 448 2^e above the rows' magnitudes and lets
        # the others grow, int8 compares them with the largest magnitude / 127
        m = _next_to(1.0 + torch.rand(pages, 1, hkv, generator=g, dtype=torch.float64), g)
        # ratios of a tie to a code: recoded, that code lies next to the tie
        tie = torch.randint(8, 16, m.shape, generator=g).double() + 0.5
        code = torch.randint(8, 16, m.shape, generator=g).double()
        r = tie / code
        r = torch.where(r < 1, 2 * r, r)
        m[::2] = _next_to(r, g)[::2]
        scale = torch.ldexp(m, torch.randint(-8, 3, m.shape, generator=g))
        if kind == "e4m3":
            codes = torch.where(torch.rand(codes.shape, generator=g) < 0.5, codes.float(),
                                torch.ldexp(code.unsqueeze(-1).float(), torch.randint(-6, 5, codes.shape, generator=g)))
            codes = codes.to(CODES[kind])
        cache += [codes, scale]
    cache = [cache[0], cache[2], cache[1], cache[3]]
    rows = []
    for x in (2, 3):
        sc = cache[x][table[:, 0].long(), 0].double()[:, None, :, None]       # [n, 1, hkv, 1]
        if kind == "e4m3":
            t = (torch.randint(8, 16, (n, 8, hkv, d), generator=g).double() + 0.5)
            t = torch.ldexp(t, torch.randint(-9, 5, t.shape, generator=g))
        else:
            t = torch.randint(0, 127, (n, 8, hkv, d), generator=g).double() + 0.5
        t *= torch.randint(0, 2, t.shape, generator=g) * 2 - 1
        t = t.clamp(-top, top)
        # sequences with every third head's magnitudes above what the scale holds
        t[::2, 0, ::3, 0] = top * 1.7
        x = t * sc
        rows.append((_next_to(x, g) if dt == F32 else x.to(dt)).reshape(8 * n, hkv, d))
    dev = _dev(cache)
    before = [c.clone() for c in cache[2:]]
    mt.paged_cache_write(rows[0].cuda(), rows[1].cuda(), *dev, cu_of(new, "cuda"), cu_of(kv, "cuda"), table.cuda())
    for x in (0, 1):
        cache8.write(cache[x], cache[2 + x], rows[x], _offsets(new), kv, table)
        used = table[:, 0].long()
        grew = cache[2 + x][used] > before[x][used]
        assert bool(grew.any()) and not bool(grew.all())
        assert torch.equal(dev[2 + x].cpu(), cache[2 + x])
        assert same_codes(dev[x], cache[x]), int((dev[x].cpu().view(torch.uint8) != cache[x].view(torch.uint8)).sum())
