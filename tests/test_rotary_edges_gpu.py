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


def test_positions_of_a_tree_count_from_the_sequence_s_beginning(mt):
    """Drafted tokens behind a context, their positions as documented (context length +
    depth): each sees its path as if that had been appended alone, token after token."""
    g = torch.Generator().manual_seed(21)
    hq, hkv, d, page = 4, 2, 64, 16
    contexts, parents = [21, 0, 40], [-1, 0, 0, 1, 2, -1]
    n = len(parents)
    paths = []
    for j, p in enumerate(parents):
        paths.append((paths[p] if p >= 0 else []) + [j])
    depth = torch.tensor([len(p) - 1 for p in paths] * len(contexts), dtype=torch.int32, device="cuda")
    mask = torch.zeros(n, n, dtype=torch.bool)
    for j, p in enumerate(paths):
        mask[j, p] = True
    f = frequencies(d).cuda()
    old = [[torch.randn(c, hkv, d, generator=g).to(BF16).cuda() for _ in range(2)] for c in contexts]
    q, k, v = [torch.randn(n * len(contexts), h, d, generator=g).to(BF16).cuda() for h in (hq, hkv, hkv)]

    def cu(lens):
        return torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0).int()

    def caches(b):
        table = torch.randperm(4 * b, generator=g).view(b, 4).to(torch.int32).cuda()
        return [torch.zeros(4 * b, page, hkv, d, dtype=BF16, device="cuda") for _ in range(2)] + [table]

    kc, vc, table = caches(len(contexts))
    mt.paged_cache_append(torch.cat([x[0] for x in old]), torch.cat([x[1] for x in old]), kc, vc, cu(contexts),
                          cu(contexts), table, inv_freq=f)
    cu_q, cu_kv = cu([n] * len(contexts)), cu([c + n for c in contexts])
    drafted = cu_q.diff()
    context = (cu_kv.diff() - drafted).repeat_interleave(drafted)
    qr = mt.paged_cache_append(k, v, kc, vc, cu_q, cu_kv, table, q=q, positions=context + depth, inv_freq=f)
    out = mt.paged_tree_decode(qr, kc, vc, cu_q, cu_kv, table, mask.repeat(len(contexts), 1).cuda(), n,
                               max(contexts) + n)
    for s, c in enumerate(contexts):
        for j, path in enumerate(paths):
            at = torch.tensor(path, device="cuda") + s * n
            one_k, one_v, one = caches(1)
            keys, values = torch.cat((old[s][0], k[at])), torch.cat((old[s][1], v[at]))
            m = [c + len(path)]
            rows = torch.zeros(m[0], hq, d, dtype=BF16, device="cuda")
            rows[-1] = q[s * n + j]
            turned = mt.paged_cache_append(keys, values, one_k, one_v, cu(m), cu(m), one, q=rows, inv_freq=f)
            assert torch.equal(turned[-1], qr[s * n + j])
            # the definition over the rotated rows, in 64 bits
            p = torch.arange(m[0])
            kk = one_k.flatten(0, 1)[one[0].cpu()[p // page].long() * page + p % page].double().cpu()
            vv = values.double().cpu()
            qq = turned[-1].double().cpu()
            for h in range(hq):
                w = torch.softmax((kk[:, h // 2] * qq[h]).sum(-1) / 8.0, 0)
                ref, size = (w[:, None] * vv[:, h // 2]).sum(0), (w[:, None] * vv[:, h // 2].abs()).sum(0)
                # scores: 72 U of sum |q k| / 8; two parts of a weight 2^-16, exp2 2^-18, sums 2 U a key; one rounding
                far = float((kk[:, h // 2].abs() * qq[h].abs()).sum(-1).max()) / 8.0
                rel = 2.02 * 72 * 2.0 ** -24 * far + 2.0 ** -18 + 2.0 ** -15 + 2 * m[0] * 2.0 ** -24
                err = (out[s * n + j, h].double().cpu() - ref).abs()
                assert bool((err <= rel * size + 2.0 ** -8 * ref.abs() + 2.0 ** -25).all()), (s, j, h)


@pytest.mark.parametrize("cu,cu_kv", [([-4, 7, 5, 30], [0, 9, 3, 2 ** 31 - 1]), ([0, 12, 3, 12], [0, 20, 21, 30]),
                                      ([9, 2, 2, 40], [5, 0, 17, 40]), ([-9, -3, -1, 6], [-7, 3, 4, 9])])
def test_bad_offsets_write_placed_rows_alone(mt, cu, cu_kv):
    """Offsets that are not rising, negative or past the rows: what changes in the cache are rows
    that a table names for one of its sequence's last tokens, each holding a new row."""
    g = torch.Generator().manual_seed(13)
    page, m = 16, 12
    q, k, v = [torch.randn(m, h, 64, generator=g).to(BF16) for h in (4, 2, 2)]
    caches = torch.full((2, 7, page, 2, 64), -77.0, dtype=BF16, device="cuda")
    table = torch.tensor([[0, 1], [2, 3], [4, 6]], dtype=torch.int32)
    kw = dict(q=q.cuda(), inv_freq=frequencies(64).cuda())
    out = mt.paged_cache_append(k.cuda(), v.cuda(), caches[0], caches[1],
                                *[torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu, cu_kv)], table.cuda(), **kw)
    assert bool(torch.isfinite(out.float()).all())
    at = caches.cpu().flatten(1, 2)
    changed = (at != -77.0).flatten(2).any(2)
    allowed = set()
    for s in range(3):
        a = min(max(cu[s], 0), m)
        n, length = max(min(cu[s + 1], m) - a, 0), max(cu_kv[s + 1] - cu_kv[s], 0)
        for pos in range(max(length - n, 0), length):
            if pos // page < 2:
                allowed.add(int(table[s, pos // page]) * page + pos % page)
            else:
                break
    for side in range(2):
        assert set(changed[side].nonzero()[:, 0].tolist()) <= allowed
    assert torch.equal(changed[0], changed[1]) and int(changed[0].sum()) <= m
    for row in changed[1].nonzero()[:, 0].tolist():
        assert bool((v.flatten(1) == at[1, row].flatten()).all(1).any())
