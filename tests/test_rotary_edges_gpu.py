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
