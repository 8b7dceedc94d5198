"""Attention of trees of drafted tokens over a paged cache on the GPU: against the
fp64 oracle within what its arithmetic allows, every layout of the launch, masks
that leave nothing, values that are not finite, streams and graphs, and a
speculative step of all paged operators together."""

import ctypes
import math

import pytest
import torch

from mtlattn_amd import capi
from oracle import rotary as rope
from tests.helpers import cu_of
from tests.rotary_helpers import frequencies
from tests.tree_helpers import Case, random_tree

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def mt():
    import mtlattn
    return mtlattn


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,page,ql,kl", [
    # up to 32 rows a kv head, 64, 128, more; single tokens, no context, ends inside tiles and pages
    (4, 2, 16, [3, 1, 8, 0, 5], [40, 1, 8, 17, 333]),
    (8, 1, 48, [1, 1, 4], [700, 65, 64]),
    (8, 2, 16, [16, 9, 1], [16, 200, 129]),
    (4, 4, 32, [64, 1, 33, 0, 50], [64, 300, 161, 9, 1000]),
    (8, 2, 64, [32, 17, 2], [32, 81, 5]),
    (6, 2, 128, [64, 3, 40], [64, 259, 1500]),
    (16, 2, 256, [64, 31], [70, 700]),
    (3, 3, 16, [130, 256], [131, 600]),
])
def test_trees(mt, dtype, d, hq, hkv, page, ql, kl):
    g = torch.Generator().manual_seed(hq * 100 + page + d)
    print(f"\n[case] tree {dtype} D {d} heads {hq}/{hkv} page {page} {ql} of {kl}", flush=True)
    c = Case(ql, kl, hq, hkv, d, page, dtype, g, behind=2)
    c.check(*c.run(mt))
    # any mask, more columns than tokens; rows that see nothing where there is no context
    c = Case(ql, kl, hq, hkv, d, page, dtype, g, cols=min(256, max(ql) + 7), masks="any")
    out, lse = c.run(mt)
    c.check(out, lse)
    again, lse2 = c.run(mt)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    # more tokens than columns: seen by none
    c = Case(ql, kl, hq, hkv, d, page, dtype, g, cols=max(1, max(ql) // 2))
    c.check(c.run(mt, lse=False)[0], None)


@pytest.mark.parametrize("n", [64, 65, 130, 300])
def test_many_sequences(mt, n):
    g = torch.Generator().manual_seed(n)
    ql = [(5 * i) % 7 for i in range(n)]
    kl = [max(q, (37 * i) % 90) for i, q in enumerate(ql)]
    kl[n // 2] = 900
    c = Case(ql, kl, 4, 2, 64, 16, BF16, g)
    c.check(*c.run(mt))


@pytest.mark.parametrize("hq,hkv,n", [(4, 1, 4), (8, 1, 8), (8, 1, 40)])
def test_long_contexts_are_cut(mt, hq, hkv, n):
    """One sequence over all workgroups, and two of very different lengths."""
    g = torch.Generator().manual_seed(n)
    for ql, kl in (([n], [9001]), ([n, 3], [5000, 70])):
        c = Case(ql, kl, hq, hkv, 128, 64, BF16, g)
        c.check(*c.run(mt))


def test_more_queries_than_tokens(mt):
    """Offsets that give a sequence fewer tokens than queries: nodes before the first
    token do not exist."""
    g = torch.Generator().manual_seed(3)
    c = Case([9, 5, 4], [4, 0, 7], 4, 2, 64, 16, BF16, g, masks="any")
    c.check(*c.run(mt))


def test_more_tokens_than_a_mask_has_columns(mt):
    """300 drafted tokens: those past the 256th column are seen by none."""
    g = torch.Generator().manual_seed(17)
    c = Case([300, 2], [333, 40], 4, 2, 64, 16, BF16, g, cols=256)
    c.check(*c.run(mt))


def test_rows_before_the_first_sequence(mt):
    """Offsets that begin past row 0: the rows before them are left as they were."""
    g = torch.Generator().manual_seed(18)
    c = Case([3, 0, 6], [3, 0, 120], 4, 2, 64, 16, BF16, g, behind=2)
    q = torch.cat((torch.full((2, 4, 64), math.nan).to(BF16), c.q))
    mask = torch.cat((torch.zeros(2, c.cols, dtype=torch.bool), c.mask))
    lse = torch.full((q.shape[0], 4), 7.0, device="cuda")
    out = mt.paged_tree_decode(q.cuda(), c.k.cuda(), c.v.cuda(), cu_of(c.ql, "cuda") + 2, cu_of(c.kl, "cuda") + 5,
                               c.table.cuda(), mask.cuda(), 6, 120, c.scale, lse)
    assert bool((lse[:2] == 7.0).all())
    c.check(out[2:], lse[2:])


def test_one_mask_for_all_tokens(mt):
    """A mask broadcast over the rows (a prefix mask)."""
    g = torch.Generator().manual_seed(19)
    c = Case([4, 4], [90, 4], 4, 2, 64, 16, F16, g)
    row = torch.tensor([[True, True, False, True]])
    c.mask = row.expand(8, 4)
    c.check(*c.run(mt, mask=row.cuda().expand(8, 4)))


def test_bounds_shape_the_launch_alone(mt):
    g = torch.Generator().manual_seed(4)
    c = Case([40, 3, 9], [900, 3, 77], 8, 2, 128, 16, BF16, g)
    for max_q, max_kv in ((1, 16), (12, 0), (200, 900), (40, 100), (1 << 20, 912)):
        c.check(*c.run(mt, max_q=max_q, max_kv=max_kv))


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales(mt, scale):
    g = torch.Generator().manual_seed(5)
    for ql, kl in (([4, 2], [90, 5]), ([40], [500])):
        c = Case(ql, kl, 8, 2, 64, 16, F16, g)
        c.scale = scale
        c.check(*c.run(mt))


def test_rising_scores(mt):
    """Scores that grow along the keys, tile after tile, by more than a type's range."""
    g = torch.Generator().manual_seed(6)
    for dtype in (BF16, F16):
        c = Case([5, 20], [700, 1200], 4, 2, 64, 16, dtype, g, poison=False)
        c.q[:] = 1.0
        for s, n in enumerate(c.kl):
            j = torch.arange(n)
            c.k.flatten(0, 1)[c.table[s, j // 16].long() * 16 + j % 16] = (j / 16.0).to(dtype)[:, None, None]
        c.check(*c.run(mt))


@pytest.mark.parametrize("ql", [[7], [16], [40]])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_not_finite_values_of_unseen_keys(mt, dtype, ql):
    """A drafted token's key or value that is infinite or NaN reaches the rows that see
    it and no other."""
    g = torch.Generator().manual_seed(ql[0])
    n, kl = ql[0], [ql[0] + 60]
    c = Case(ql, kl, 4, 1, 128, 16, dtype, g)
    clean = c.reference()

    def put(x, node, col, value):
        j = kl[0] - n + node
        x[int(c.table[0, j // 16]), j % 16, 0, col] = value

    k, v = c.k.clone(), c.v.clone()
    put(v, 1, 5, math.inf)
    put(v, 2, 5, -math.inf)
    put(v, 3, 9, math.nan)
    put(v, 0, 77, -math.inf)
    put(k, 5, 3, math.nan)
    out, lse = c.run(mt, k=k, v=v)
    out, lse = out.double().cpu(), lse.double().cpu()
    want = clean[0].clone()
    sees = c.mask[:, :, None, None]
    hit = torch.zeros(n, 4, 128, dtype=torch.bool)
    for i in range(n):
        if c.mask[i, 5]:
            hit[i] = True
            assert out[i].isnan().all() and lse[i].isnan().all()
            continue
        kinds = {5: [x for x, node in ((math.inf, 1), (-math.inf, 2)) if c.mask[i, node]],
                 9: [math.nan] if c.mask[i, 3] else [], 77: [-math.inf] if c.mask[i, 0] else []}
        for col, seen in kinds.items():
            if not seen:
                continue
            hit[i, :, col] = True
            x = out[i, :, col]
            if len(seen) > 1 or seen[0] != seen[0]:
                assert x.isnan().all()
            else:
                assert bool((x == seen[0]).all())
    assert bool(hit.any()) and bool((~hit).any()) and sees.any()
    assert bool(torch.isfinite(out[~hit]).all())
    keep = Case.__new__(Case)
    keep.__dict__.update(c.__dict__)
    out[hit] = want[hit]
    seen5 = c.mask[:, 5]
    lse[seen5] = clean[1][seen5]
    keep.check(out, torch.cat([lse]), clean)


def test_infinite_context_reaches_every_row(mt):
    g = torch.Generator().manual_seed(8)
    c = Case([6], [300], 4, 1, 64, 16, BF16, g)
    j = 100
    c.v[int(c.table[0, j // 16]), j % 16, 0, 3] = math.inf
    out, _ = c.run(mt)
    assert bool((out[:6, :, 3] == math.inf).all()) and bool(torch.isfinite(out[:6, :, 4:].float()).all())


def test_layouts(mt):
    """q as a slice of a projection, K and V side by side, masks with strides: the same
    bits as plain ones."""
    g = torch.Generator().manual_seed(9)
    c = Case([5, 17, 1], [50, 400, 1], 8, 2, 128, 16, BF16, g)
    out, lse = c.run(mt)
    wide = torch.zeros(c.q.shape[0], 12, 128, dtype=BF16, device="cuda")
    wide[:, 2:10] = c.q.cuda()
    both = torch.stack((c.k, c.v), 2).cuda()
    big = torch.zeros(c.q.shape[0], 40, dtype=torch.bool, device="cuda")
    big[:, 3:3 + c.cols] = c.mask.cuda()
    for kw in (dict(q=wide[:, 2:10]), dict(k=both[:, :, 0], v=both[:, :, 1]), dict(mask=big[:, 3:3 + c.cols]),
               dict(mask=c.mask.t().contiguous().cuda().t())):
        a, b = c.run(mt, **kw)
        assert torch.equal(a, out) and torch.equal(b, lse), kw.keys()
    # one row of q for all tokens
    a, _ = c.run(mt, q=c.q[:1].expand(c.q.shape))
    b, _ = c.run(mt, q=c.q[:1].expand(c.q.shape).contiguous())
    assert torch.equal(a, b)


def test_a_chain_is_causal_decode(mt):
    """A tree that is a chain: what paged_decode computes."""
    g = torch.Generator().manual_seed(10)
    c = Case([4, 1, 3], [700, 33, 3], 8, 2, 128, 16, BF16, g, cols=4)
    c.mask = torch.cat([torch.tril(torch.ones(n, 4)).bool() for n in c.ql])
    out, lse = c.run(mt)
    c.check(out, lse)
    lse2 = torch.empty_like(lse)
    ref = mt.paged_decode(c.q.cuda(), c.k.cuda(), c.v.cuda(), cu_of(c.ql, "cuda"), cu_of(c.kl, "cuda"), c.table.cuda(), 4,
                          700, causal=True, lse_out=lse2)
    c.check(ref, lse2)


def test_far_pages(mt):
    """A cache whose rows lie past 2^31 elements: appended to and attended."""
    g = torch.Generator().manual_seed(11)
    hkv, d, page = 8, 128, 64
    pages = (1 << 31) // (page * hkv * d) + 40
    caches = [torch.empty(pages, page, hkv, d, dtype=BF16, device="cuda") for _ in range(2)]
    c = Case([9, 20], [200, 150], 8, hkv, d, page, BF16, g, poison=False)
    small = c.table.clone()
    c.table = (pages - 1 - small).to(torch.int32)               # the far end
    c.table[0, 0] = 0
    m = sum(c.kl)
    k, v = [torch.randn(m, hkv, d, generator=g).to(BF16) for _ in range(2)]
    cu = cu_of(c.kl, "cuda")
    mt.paged_cache_append(k.cuda(), v.cuda(), *caches, cu, cu, c.table.cuda())
    out = mt.paged_tree_decode(c.q.cuda(), *caches, cu_of(c.ql, "cuda"), cu, c.table.cuda(), c.mask.cuda(), 20, 200)
    # the same through a small cache
    c.table, first = small, 0
    for s, n in enumerate(c.kl):
        j = torch.arange(n)
        at = c.table[s, j // page].long() * page + j % page
        c.k.flatten(0, 1)[at], c.v.flatten(0, 1)[at] = k[first:first + n], v[first:first + n]
        first += n
    c.check(out, None)
    assert torch.equal(out, c.run(mt)[0])


def test_the_longest_sequence(mt):
    """2^31 - 2^16 logical tokens, in two pages again and again: equal keys and values of
    +-1, whose sums stay exact, over work that passes 2^24 tiles."""
    n = 2 ** 31 - 2 ** 16
    k = torch.ones(3, 64, 1, 64, dtype=BF16, device="cuda")
    v = torch.where(torch.arange(64, device="cuda") % 3 == 0, 1.0, -1.0).to(BF16).expand(3, 64, 1, 64).contiguous()
    q = torch.ones(1, 1, 64, dtype=BF16, device="cuda")
    lse = torch.empty(1, 1, device="cuda")
    mask = torch.ones(1, 1, dtype=torch.bool, device="cuda")
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    ck = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    table = 1 + torch.arange(n // 64, dtype=torch.int32, device="cuda")[None] % 2
    out = mt.paged_tree_decode(q, k, v, cu, ck, table, mask, 1, n, 0.125, lse)
    assert torch.equal(out[0, 0], v[0, 0, 0])
    # (64 products of 0.125; the logarithm in fp32)
    assert abs(float(lse) - (8.0 + math.log(n))) <= 4 * 2.0 ** -23 * 32


def test_bad_pages_are_clamped(mt):
    """Pages and columns that do not exist read the nearest ones that do, as in
    paged_decode."""
    g = torch.Generator().manual_seed(12)
    c = Case([3, 6], [100, 90], 4, 2, 64, 16, BF16, g, poison=False)
    c.table[0, 2], c.table[1, 1] = -7, 10 ** 6
    c.check(*c.run(mt))
    c.table = c.table[:, :4].contiguous()                       # lengths past the table
    c.check(*c.run(mt, max_kv=64))


def test_refusals(mt):
    c = Case([3], [40], 4, 2, 64, 16, BF16, torch.Generator().manual_seed(13))
    q, k, v, mask = c.q.cuda(), c.k.cuda(), c.v.cuda(), c.mask.cuda()
    cu, ck, table = cu_of([3], "cuda"), cu_of([40], "cuda"), c.table.cuda()

    def call(q=q, k=k, v=v, cu=cu, table=table, mask=mask, max_q=3, max_kv=40, **kw):
        return mt.paged_tree_decode(q, k, v, cu, ck, table, mask, max_q, max_kv, **kw)

    call()
    for kw in (dict(q=q.float(), k=k.float(), v=v.float()), dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :32]),
               dict(k=k[:, :8], v=v[:, :8]), dict(k=k[:, :, :1]), dict(mask=mask.int()), dict(mask=mask[:2]),
               dict(mask=mask[:, :0]), dict(mask=mask.cpu()), dict(mask=torch.ones(3, 257, dtype=torch.bool, device="cuda")),
               dict(max_q=0), dict(max_kv=-1), dict(max_kv=10 ** 6), dict(scale=math.nan), dict(scale=math.inf),
               dict(table=table.long().cpu()), dict(cu=cu_of([3, 0], "cuda")), dict(lse_out=torch.empty(3, 3, device="cuda")),
               dict(lse_out=torch.empty(3, 4, device="cuda", dtype=torch.float64)),
               dict(q=torch.zeros(3 * 256 + 1, dtype=BF16, device="cuda")[1:].view(3, 4, 64))):
        with pytest.raises(RuntimeError, match="mtlattn|tree_decode"):
            call(**kw)
    assert call(q=q[:0], mask=mask[:0], cu=cu_of([0], "cuda")).shape == (0, 4, 64)


# ---- streams, graphs, and the operators together ----


def test_graph_and_shared_workspace(mt):
    """Two graphs over one workspace through the C entry, replayed in turn with new
    lengths, masks and rows, against eager calls."""
    g = torch.Generator().manual_seed(14)
    c = Case([8, 8, 8], [600, 90, 300], 8, 2, 128, 16, BF16, g, poison=False)
    c.cols = 8
    q, k, v, table = c.q.cuda(), c.k.cuda(), c.v.cuda(), c.table.cuda()
    mask, cu, ck = c.mask.cuda(), cu_of(c.ql, "cuda"), cu_of(c.kl, "cuda")
    p = capi.problem_for(q, k.flatten(0, 1), cu, ck, 8, c.scale)
    size = capi.lib().mtlattn_tree_decode_workspace_size(ctypes.byref(p), 600)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def call(out, lse):
        capi.call("mtlattn_tree_decode", p, q.data_ptr(), 1024, k.data_ptr(), 256, v.data_ptr(), 256, 16, k.shape[0],
                  table.data_ptr(), table.shape[1], 600, mask.data_ptr(), 8, 8, out.data_ptr(), lse.data_ptr(),
                  ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)

    def room():
        return torch.empty_like(q), torch.empty(24, 8, device="cuda")

    eager = room()
    call(*eager)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        outs, graph = room(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(*outs)
        graphs.append((graph, outs))
    for i in range(6):
        q.copy_(torch.randn(q.shape, generator=g).to(BF16))
        mask.copy_(torch.cat([random_tree(8, 8, g) for _ in range(3)]))
        ck.copy_(cu_of([600 - 90 * i, 90 - 3 * i, 8 + 50 * i]))
        graph, outs = graphs[i % 2]
        graph.replay()
        call(*eager)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1]), i


def test_two_streams(mt):
    g = torch.Generator().manual_seed(15)
    cases = [Case([8, 20], [900, 200], 8, 2, 128, 16, BF16, g), Case([3], [2000], 8, 2, 128, 16, BF16, g)]
    want = [c.run(mt) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(cases[i % 2].run(mt))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, want[i % 2][0]) and torch.equal(b, want[i % 2][1]), i


def test_speculative_steps(mt):
    """Two steps of a speculative server: the prompt appended and attended, a tree of
    drafted tokens appended at its depths and verified, the accepted path appended in
    its place, then a step of one token. Each result is what full attention over
    the accepted tokens gives."""
    g = torch.Generator().manual_seed(16)
    hq, hkv, d, page = 8, 2, 64, 16
    w = [(1 + 0.1 * torch.randn(d, generator=g)).to(BF16) for _ in range(2)]
    f = frequencies(d)
    prompts, tree_n = [37, 5], 9
    pages = 16
    table = torch.randperm(pages, generator=g).view(2, 8).to(torch.int32).cuda()
    caches = [torch.full((pages, page, hkv, d), math.nan, dtype=BF16, device="cuda") for _ in range(2)]
    wq, wk = [x.cuda() for x in w]

    def draw(n):
        return [torch.randn(n, h, d, generator=g).to(BF16) for h in (hq, hkv, hkv)]

    def append(rows, ql, kl, positions=None):
        q, k, v = [t.cuda() for t in rows]
        return mt.paged_cache_append(k, v, *caches, cu_of(ql, "cuda"), cu_of(kl, "cuda"), table, q=q,
                                     positions=positions, inv_freq=f.cuda(), q_weight=wq, k_weight=wk)

    # history: per sequence the rows (q, k, v) of its tokens, at positions 0, 1, ...
    rows = draw(sum(prompts))
    append(rows, prompts, prompts)
    history = [[t[:37] for t in rows], [t[37:] for t in rows]]
    trees = [random_tree(tree_n, tree_n, g) for _ in prompts]
    depth = torch.cat([t.sum(1) - 1 for t in trees])
    drafted = draw(2 * tree_n)
    ql, kl = [tree_n] * 2, [n + tree_n for n in prompts]
    first = torch.tensor(prompts).repeat_interleave(tree_n)
    q = append(drafted, ql, kl, positions=(first + depth).cuda())
    out = mt.paged_tree_decode(q, *caches, cu_of(ql, "cuda"), cu_of(kl, "cuda"), table, torch.cat(trees).cuda(), tree_n, max(kl))

    def full(q, k, v, scale=1.0 / math.sqrt(d)):
        """The last token of a history, from the definition: (result, bound's size)."""
        pos = torch.arange(k.shape[0])
        kr = rope.forward(k, pos, f, weight=w[1]).to(BF16).double()
        qr = rope.forward(q[-1:], pos[-1:], f, weight=w[0]).to(BF16).double()
        res = torch.empty(hq, d, dtype=torch.float64)
        for h in range(hq):
            p = torch.softmax((kr[:, h // 4] * qr[0, h]).sum(-1) * scale, 0)
            res[h] = (p[:, None] * v[:, h // 4].double()).sum(0)
        return res

    # rotated rows may differ by a step of bf16 (2^-7) where they lie next to a border: of a few
    # of D products each, |q k| scale <= 4; then P's and the result's rounding
    tol = 4 * 2.0 ** -7
    for s in range(2):
        for i in range(tree_n):
            path = trees[s][i].nonzero()[:, 0]
            mine = [torch.cat([a, b[s * tree_n + path]]) for a, b in zip(history[s], drafted)]
            err = (out[s * tree_n + i].double().cpu() - full(*mine)).abs().max()
            assert err <= tol, (s, i, float(err))
    # the longest path of each tree is accepted: its rows again, in their places
    best = [t[int(t.sum(1).argmax())].nonzero()[:, 0] for t in trees]
    ql = [len(b) for b in best]
    kl = [n + len(b) for n, b in zip(prompts, best)]
    take = torch.cat([b + s * tree_n for s, b in enumerate(best)])
    accepted = [t[take] for t in drafted]
    append(accepted, ql, kl)
    history = [[torch.cat([a, b[s * tree_n + best[s]]]) for a, b in zip(history[s], drafted)] for s in range(2)]
    # one more token each, through plain decode
    token = draw(2)
    kl = [n + 1 for n in kl]
    q = append(token, [1, 1], kl)
    out = mt.paged_decode(q, *caches, cu_of([1, 1], "cuda"), cu_of(kl, "cuda"), table, 1, max(kl), causal=True)
    for s in range(2):
        mine = [torch.cat([a, b[s:s + 1]]) for a, b in zip(history[s], token)]
        assert float((out[s].double().cpu() - full(*mine)).abs().max()) <= tol
