"""The softmax weights of attention over trees of drafted tokens: how many of their
bits reach the results, which values that cancel show, the logarithm of their
sum, and infinite values in the context."""

import math

import pytest
import torch

from tests.tree_helpers import U, Case

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def mt():
    import mtlattn
    return mtlattn


def place(c, x, s, j):
    return x[int(c.table[s, j // c.page]), j % c.page]


# rows of a kv head: 8 .. 256, which every layout of the launch takes; lengths of one tile
# to many, cut into pieces or not
SHAPES = [(4, 2, 16, [2, 1], [40, 9]), (8, 2, 32, [16, 7], [300, 64]), (8, 1, 16, [12], [260]),
          (8, 2, 64, [40, 3], [190, 170]), (16, 2, 64, [33], [512])]


def cancelling(hq, hkv, d, page, ql, kl, dtype, seed):
    """Whole numbers as queries and keys, so that scores are exact in fp32; neighbouring
    keys of the context that differ in one element and have opposite values."""
    g = torch.Generator().manual_seed(seed)
    c = Case(ql, kl, hq, hkv, d, page, dtype, g)
    c.q = torch.randint(-2, 3, c.q.shape, generator=g).to(dtype)
    c.k = torch.randint(-2, 3, c.k.shape, generator=g).to(dtype)
    c.v = torch.randn(c.v.shape, generator=g).to(dtype)
    for s, n in enumerate(kl):
        for j in range(0, n - 1, 2):
            place(c, c.k, s, j + 1).copy_(place(c, c.k, s, j))
            place(c, c.k, s, j + 1)[:, j % d] += 1
            place(c, c.v, s, j + 1).copy_(-place(c, c.v, s, j))
    return c


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,page,ql,kl", SHAPES)
def test_weights_keep_their_bits(mt, dtype, d, hq, hkv, page, ql, kl):
    """A score times its factor and less the maximum: 8 U of the largest, and e^x of
    that error; exp2 2^-18 with its argument's rounding. A weight as the sum of two numbers of the
    type: half a step of half a step, (eps / 2)^2, in fp16 half a step of its smallest
    numbers too (2^-25, against a sum of at least 1). Sums over keys and merges, 2 U a key; then
    one rounding. (Weights rounded to the type once would be off by eps / 2.)"""
    print(f"\n[case] weights {dtype} D {d} heads {hq}/{hkv} {ql} of {kl}", flush=True)
    c = cancelling(hq, hkv, d, page, ql, kl, dtype, d + hq)
    o, l, size, far = c.reference()
    out, lse = c.run(mt)
    n, half = max(kl), torch.finfo(dtype).eps / 2
    delta = 8 * U * far
    rel = torch.expm1(2 * delta) + 2.0 ** -18 + 2 * half * half + 2 * n * U
    low = n * 2.0 ** -25 * float(c.v.abs().max()) if dtype == F16 else 0.0
    bound = rel[..., None] * size + low + half * o.abs() + 2.0 ** -25
    err = (out.double().cpu() - o).abs()
    assert bool((err <= bound).all()), (int((err > bound).sum()), float((err / bound).max()))
    # the logarithm is of the weights' own sum: no rounding to the type in it
    lb = delta + n * U + 2.0 ** -18 + 2.0 ** -22 * l.abs()
    err = (lse.double().cpu() - l).abs()
    assert bool((err <= lb).all()), float((err / lb).max())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,page,ql,kl", [(4, 2, 16, [5], [700]), (8, 2, 16, [30, 2], [900, 40]),
                                               (8, 1, 48, [40], [3000])])
def test_infinite_values_of_the_context(mt, dtype, d, hq, hkv, page, ql, kl):
    """Every row sees them: their columns are the infinity, or NaN where they contradict; all
    other values keep their bits."""
    g = torch.Generator().manual_seed(d + kl[0])
    c = Case(ql, kl, hq, hkv, d, page, dtype, g)
    clean, clean_lse = c.run(mt)
    v, last = c.v.clone(), kl[0] - ql[0] - 1
    place(c, v, 0, 3)[0, 5] = math.inf
    place(c, v, 0, 70)[0, 6] = -math.inf
    place(c, v, 0, last)[0, 7] = math.inf
    place(c, v, 0, 0)[0, 8] = math.inf
    place(c, v, 0, 333)[0, 8] = -math.inf
    place(c, v, 0, 200)[hkv - 1, 9] = math.nan
    place(c, v, 0, 201)[hkv - 1, d - 1] = -math.inf
    place(c, v, 0, 140)[0, 11] = math.inf
    place(c, v, 0, 140 + 64)[0, 11] = math.inf
    out, lse = c.run(mt, v=v)
    assert torch.equal(lse, clean_lse)
    group, want = hq // hkv, clean.clone()
    first, behind = want[:ql[0], :group], want[:ql[0], -group:]
    first[..., 5], first[..., 6], first[..., 7], first[..., 8], first[..., 11] = (
        math.inf, -math.inf, math.inf, math.nan, math.inf)
    behind[..., 9], behind[..., d - 1] = math.nan, -math.inf
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf),
                       want.nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf))
