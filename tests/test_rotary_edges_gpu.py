"""Edges of the position rotation on the GPU: norms without an epsilon, what is
refused, very many rows, and what stands around the rows of an append."""

import pytest
import torch

from oracle import rotary as oracle
from tests.rotary_helpers import backward_bound, check, forward_bound, frequencies

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mt():
    import mtlattn
    return mtlattn


# (heads that fill a wave's passes, that do not, and a head per pass; D whose lanes are
# all in use, and not; the kernel of any D last)
@pytest.mark.parametrize("hq,hkv,d,rot", [(32, 8, 128, 128), (28, 4, 128, 64), (6, 2, 128, 128), (16, 8, 64, 64),
                                          (5, 1, 64, 64), (3, 3, 80, 80), (12, 4, 96, 48), (4, 1, 256, 256),
                                          (7, 3, 16, 16), (6, 2, 88, 44)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("eps", [0.0, 1e-50])
def test_norms_without_an_epsilon(mt, eps, interleaved, hq, hkv, d, rot):
    """An epsilon of 0, or one that is 0 in fp32: finite for every row that is not all 0."""
    g = torch.Generator().manual_seed(hq * 1000 + d)
    dtype = BF16 if d != 64 else F32
    print(f"\n[case] eps {eps} heads {hq}/{hkv} D {d} R {rot}", flush=True)
    for m in (5, 700):
        x = [torch.randn(m, h, d, generator=g).to(dtype) for h in (hq, hkv)]
        w = [(1 + 0.2 * torch.randn(d, generator=g)) for _ in x]
        dy = [torch.randn(t.shape, generator=g).to(dtype) for t in x]
        pos, f = torch.randint(0, 4096, (m,), generator=g, dtype=torch.int32), frequencies(rot)
        leaves = [t.cuda().requires_grad_() for t in (*x, *w)]
        out = mt.rotary(leaves[0], leaves[1], pos.cuda(), f.cuda(), interleaved, q_weight=leaves[2], k_weight=leaves[3],
                        eps=eps)
        grads = torch.autograd.grad(out, leaves, [t.cuda() for t in dy])
        for i, h in enumerate((hq, hkv)):
            ref = oracle.forward(x[i], pos, f, interleaved, 1.0, w[i], eps)
            check(out[i], ref, forward_bound(x[i], ref, f, interleaved, 1.0, w[i], eps, dtype), "out")
            back = oracle.backward(dy[i], x[i], pos, f, interleaved, 1.0, w[i], eps)
            bounds = backward_bound(dy[i], x[i], back, f, interleaved, 1.0, w[i], eps, dtype, m * h)
            check(grads[i], back[0], bounds[0], "dx")
            check(grads[2 + i], back[1], bounds[1], "dw")


def test_more_rows_than_a_grid_has_threads(mt):
    """2^26 + 5 tokens of a head of 16 elements, a wave each: past the 2^32 threads of a grid.
    The same bits as in two calls, and the rows about the borders by the oracle."""
    m, d = (1 << 26) + 5, 16
    half = 40_000_000
    pos = torch.arange(m, dtype=torch.int32, device="cuda") % 5003
    f = frequencies(d)
    x = [torch.randn(m, 1, d, device="cuda", dtype=BF16, generator=torch.Generator("cuda").manual_seed(i)) for i in range(2)]
    out = mt.rotary(*x, pos, f.cuda())
    parts = [mt.rotary(*[t[a] for t in x], pos[a], f.cuda()) for a in (slice(0, half), slice(half, m))]
    for i in range(2):
        assert torch.equal(out[i][:half], parts[0][i]) and torch.equal(out[i][half:], parts[1][i])
    last = 4 * ((1 << 24) - 1)                      # the first row of the second launch
    rows = torch.tensor([0, 1, half, last - 1, last, last + 1, m - 1])
    xs = x[0][rows.cuda()].cpu()
    ref = oracle.forward(xs, pos.cpu()[rows], f)
    check(out[0][rows.cuda()], ref, forward_bound(xs, ref, f, False, 1.0, None, 0.0, BF16))
    # the same rows appended, from the last page to the first
    del out, parts
    page = 1 << 20
    pages = -(-m // page)
    caches = [torch.zeros(pages, page, 1, d, dtype=BF16, device="cuda") for _ in range(2)]
    cu = torch.tensor([0, m], dtype=torch.int32, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    mt.paged_cache_append(*x, *caches, cu, cu, table)
    for t, c in zip(x, caches):
        assert torch.equal(c.flip(0).flatten(0, 1)[:m], t)
        assert not c.flip(0).flatten(0, 1)[m:].any()
