"""The 8-bit paged K/V cache on the GPU where its arithmetic and its index code
are at their edges."""

import math

import pytest
import torch

from oracle import cache8
from tests.cache8_helpers import CODES, check_decode, decode_reference, pages_for
from tests.helpers import cu_of

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def mt():
    import mtlattn
    return mtlattn


def _offsets(lens, start=0):
    c = [start]
    for n in lens:
        c.append(c[-1] + n)
    return c


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
