"""The position rotation with per-head norms on the GPU: against the fp64 oracle
within what its arithmetic and one rounding allow, its gradients, appended rows of
a paged cache, memory layouts, streams and graphs."""

import ctypes

import pytest
import torch

from mtlattn_amd import capi
from oracle import cache8
from oracle import rotary as oracle
from tests.helpers import cu_of
from tests.rotary_helpers import backward_bound, check, forward_bound, frequencies, half_step

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


@pytest.fixture(scope="module")
def mt():
    import mtlattn
    return mtlattn


def rows(m, hq, hkv, d, dtype, gen, packed=False):
    """(q, k, v) with a few large channels; packed: slices of one tensor's rows."""
    x = torch.randn(m, hq + 2 * hkv, d, generator=gen) * torch.exp(0.5 * torch.randn(d, generator=gen))
    x = x.to(dtype)
    if not packed:
        return [t.contiguous() for t in x.split([hq, hkv, hkv], 1)]
    return list(x.split([hq, hkv, hkv], 1))


def on_gpu(parts, packed):
    if not packed:
        return [t.cuda() for t in parts]
    x = torch.cat(parts, 1).cuda()
    return list(x.split([t.shape[1] for t in parts], 1))


def weights(d, dtype, gen):
    return [(1 + 0.2 * torch.randn(d, generator=gen)).to(dtype) for _ in range(2)]


# head dims and rotated parts of both kernels: multiples of 16, and others
SHAPES = [(128, 128), (64, 64), (80, 32), (256, 256), (128, 64), (16, 16), (96, 96), (192, 96),
          (96, 24), (88, 88), (80, 20), (33, 10), (1, 0), (2, 2), (255, 254), (64, 0), (128, 8)]


@pytest.mark.parametrize("d,rot", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_forward_and_gradients(mt, dtype, normed, interleaved, d, rot):
    g = torch.Generator().manual_seed(d * 1000 + rot)
    hq, hkv = (6, 3) if d != 128 else (8, 2)
    scale = 1.25 if rot != d else 1.0
    for m, packed in ((1, False), (67, True)):
        parts = rows(m, hq, hkv, d, dtype, g, packed)
        w = weights(d, dtype if m == 1 else F32, g) if normed else [None, None]
        pos = torch.randint(0, 1 << 17, (m,), generator=g, dtype=torch.int32)
        f = frequencies(rot)
        dys = [torch.randn(t.shape, generator=g).to(dtype) for t in parts[:2]]
        leaves = [t.detach().requires_grad_() for t in on_gpu(parts, packed)[:2]]
        wl = [x.cuda().requires_grad_() if normed else None for x in w]
        args = (pos.cuda(), f.cuda())
        kw = dict(interleaved=interleaved, scale=scale, q_weight=wl[0], k_weight=wl[1], eps=EPS)
        print(f"\n[case] rotary {dtype} D {d} R {rot} m {m} norm {normed} interleaved {interleaved}", flush=True)
        out = mt.rotary(leaves[0], leaves[1], *args, **kw)
        grads = torch.autograd.grad(out, leaves + (wl if normed else []), [t.cuda() for t in dys])
        with torch.no_grad():
            again = mt.rotary(leaves[0], leaves[1], *args, **kw)
        for i, name in enumerate(("q", "k")):
            assert torch.equal(out[i], again[i]) and out[i].dtype == dtype and out[i].is_contiguous()
            ref = oracle.forward(parts[i], pos, f, interleaved, scale, w[i], EPS)
            check(out[i], ref, forward_bound(parts[i], ref, f, interleaved, scale, w[i], EPS, dtype), name)
            back = oracle.backward(dys[i], parts[i], pos, f, interleaved, scale, w[i], EPS)
            dxb, dwb = backward_bound(dys[i], parts[i], back, f, interleaved, scale, w[i], EPS, dtype, m * hq)
            check(grads[i], back[0], dxb, "d" + name)
            if normed:
                assert grads[2 + i].dtype == w[i].dtype
                check(grads[2 + i], back[1], dwb, "d" + name + "_weight")


def test_many_rows(mt):
    """More tokens than one round of the backward's workgroups, the forward's two
    passes per wave."""
    g = torch.Generator().manual_seed(5)
    m, hq, hkv, d = 9001, 5, 1, 64
    parts = rows(m, hq, hkv, d, BF16, g)
    w = weights(d, F32, g)
    pos = torch.arange(m, dtype=torch.int32) * 97
    f = frequencies(d)
    leaves = [t.cuda().requires_grad_() for t in parts[:2]]
    wl = [x.cuda().requires_grad_() for x in w]
    dys = [torch.randn(t.shape, generator=g).to(BF16) for t in parts[:2]]
    out = mt.rotary(*leaves, pos.cuda(), f.cuda(), q_weight=wl[0], k_weight=wl[1])
    grads = torch.autograd.grad(out, leaves + wl, [t.cuda() for t in dys])
    for i in range(2):
        ref = oracle.forward(parts[i], pos, f, weight=w[i])
        check(out[i], ref, forward_bound(parts[i], ref, f, False, 1.0, w[i], EPS, BF16))
        back = oracle.backward(dys[i], parts[i], pos, f, weight=w[i])
        bounds = backward_bound(dys[i], parts[i], back, f, False, 1.0, w[i], EPS, BF16, m * hq // 64)
        check(grads[i], back[0], bounds[0])
        check(grads[2 + i], back[1], bounds[1])
    twice = torch.autograd.grad(mt.rotary(*leaves, pos.cuda(), f.cuda(), q_weight=wl[0], k_weight=wl[1]), leaves + wl,
                                [t.cuda() for t in dys])
    assert all(torch.equal(a, b) for a, b in zip(grads, twice))


@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 16), (1, 1, 256), (24, 8, 128), (7, 3, 64)])
@pytest.mark.parametrize("m", [3, 511, 512, 513, 1023, 1025])
def test_gradients_of_few_tokens(mt, m, hq, hkv, d):
    """Four, two or one of the backward's waves share a token's heads, which may be
    fewer than the waves."""
    g = torch.Generator().manual_seed(m + d)
    parts = rows(m, hq, hkv, d, BF16, g)[:2]
    w = weights(d, F32, g)
    pos, f = torch.randint(0, 4096, (m,), generator=g, dtype=torch.int32), frequencies(d)
    leaves = [t.cuda().requires_grad_() for t in (*parts, *w)]
    dys = [torch.randn(t.shape, generator=g).to(BF16) for t in parts]
    out = mt.rotary(*leaves[:2], pos.cuda(), f.cuda(), q_weight=leaves[2], k_weight=leaves[3])
    grads = torch.autograd.grad(out, leaves, [t.cuda() for t in dys])
    for i, h in enumerate((hq, hkv)):
        back = oracle.backward(dys[i], parts[i], pos, f, weight=w[i])
        bounds = backward_bound(dys[i], parts[i], back, f, False, 1.0, w[i], EPS, BF16, m * h)
        check(grads[i], back[0], bounds[0])
        check(grads[2 + i], back[1], bounds[1])


@pytest.mark.parametrize("d,rot", [(64, 64), (24, 12)])
def test_far_and_negative_positions(mt, d, rot):
    """Angles of up to 2^31 radians; their product in 64 bits is off by up to
    2^-52 of them, twice."""
    g = torch.Generator().manual_seed(6)
    pos = torch.tensor([0, -1, 1, 2 ** 20, 2 ** 24 + 1, -(2 ** 24) - 1, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32)
    q, k, _ = rows(len(pos), 2, 1, d, F32, g)
    f = frequencies(rot, 1e6)
    out = mt.rotary(q.cuda(), k.cuda(), pos.cuda(), f.cuda())
    for x, y in zip((q, k), out):
        ref = oracle.forward(x, pos, f)
        far = pos.double().abs()[:, None, None] * 2.0 ** -50 * oracle.size(x, f, False, 1.0)
        check(y, ref, forward_bound(x, ref, f, False, 1.0, None, EPS, F32) + far)


def test_64_bit_positions_and_grads_of_broadcasts(mt):
    g = torch.Generator().manual_seed(7)
    q, k, _ = rows(9, 4, 2, 64, F32, g)
    f = frequencies(64).cuda()
    pos = torch.arange(9)
    ql, kl = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    a, b = mt.rotary(ql, kl, pos.cuda(), f)
    (a.sum() + (b * 0.5).sum()).backward()                     # (gradients are expanded scalars)
    for x, l, s in ((q, ql, 1.0), (k, kl, 0.5)):
        ref = oracle.backward(torch.full(x.shape, s), x, pos, f.cpu())[0]
        check(l.grad, ref, backward_bound(torch.full(x.shape, s), x, (ref, None), f.cpu(), False, 1.0, None, EPS, F32, 0)[0])
    # one row for all tokens, one gradient for it
    one = q[:1].cuda().requires_grad_()
    a, b = mt.rotary(one.expand(9, 4, 64), kl.detach(), pos.cuda(), f)
    ref = oracle.forward(q[:1].expand(9, 4, 64), pos, f.cpu())
    check(a, ref, forward_bound(q[:1].expand(9, 4, 64), ref, f.cpu(), False, 1.0, None, EPS, F32))
    a.backward(torch.ones_like(a))
    assert one.grad.shape == (1, 4, 64)
    ref = oracle.backward(torch.ones(9, 4, 64), q, pos, f.cpu())[0].sum(0, keepdim=True)
    assert float((one.grad.cpu().double() - ref).abs().max()) < 9 * 2 * 20 * 2.0 ** -24


def test_one_output_alone(mt):
    """A loss of the queries only: the keys' gradients are 0."""
    g = torch.Generator().manual_seed(8)
    q, k, _ = rows(5, 4, 2, 64, BF16, g)
    w = [x.cuda().requires_grad_() for x in weights(64, BF16, g)]
    ql, kl = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    a, _ = mt.rotary(ql, kl, torch.arange(5).cuda(), frequencies(64).cuda(), q_weight=w[0], k_weight=w[1])
    a.float().square().sum().backward()
    assert bool((kl.grad == 0).all()) and bool((w[1].grad == 0).all())
    assert bool(torch.isfinite(ql.grad).all()) and float(ql.grad.abs().max()) > 0 and float(w[0].grad.abs().max()) > 0


def test_gradients_of_gradients_are_refused(mt):
    g = torch.Generator().manual_seed(18)
    q, k, _ = [t.cuda().requires_grad_() for t in rows(5, 4, 2, 64, F32, g)]
    a, b = mt.rotary(q, k, torch.arange(5).cuda(), frequencies(64).cuda())
    d, = torch.autograd.grad(a.square().sum() + b.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()


def test_rows_changed_before_the_backward_are_noticed(mt):
    """Without norms the backward does not need the rows; with them a changed row raises."""
    g = torch.Generator().manual_seed(19)
    q, k, _ = [t.cuda() for t in rows(5, 4, 2, 64, F32, g)]
    w = [x.cuda().requires_grad_() for x in weights(64, F32, g)]
    f, pos = frequencies(64).cuda(), torch.arange(5).cuda()
    a, _ = mt.rotary(q, k, pos, f, q_weight=w[0], k_weight=w[1])
    q.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        a.sum().backward()


def test_no_rows(mt):
    f = frequencies(64).cuda()
    q = torch.empty(0, 4, 64, dtype=BF16, device="cuda", requires_grad=True)
    k = torch.empty(0, 2, 64, dtype=BF16, device="cuda", requires_grad=True)
    w = [torch.ones(64, dtype=BF16, device="cuda", requires_grad=True) for _ in range(2)]
    a, b = mt.rotary(q, k, torch.empty(0, dtype=torch.int32, device="cuda"), f, q_weight=w[0], k_weight=w[1])
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)
    (a.sum() + b.sum()).backward()
    assert bool((w[0].grad == 0).all()) and bool((w[1].grad == 0).all())


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_what_is_not_finite_stays_in_its_pair(mt, bad, interleaved):
    """Without a norm a value reaches its pair alone, with one its head alone."""
    g = torch.Generator().manual_seed(9)
    d, rot = 80, 32
    q, k, _ = rows(6, 4, 2, d, BF16, g)
    f = frequencies(rot)
    pos = torch.arange(6, dtype=torch.int32) + 3
    a, b = oracle.pairs(d, rot, interleaved)
    q[2, 1, 40] = bad                                           # passes
    q[3, 0, a[5]] = bad                                         # turns, with its partner
    k[4, 1, b[0]] = bad
    for w in ([None, None], weights(d, BF16, g)):
        out = mt.rotary(q.cuda(), k.cuda(), pos.cuda(), f.cuda(), interleaved, 1.0, *[x if x is None else x.cuda() for x in w])
        lost = [torch.zeros(x.shape, dtype=torch.bool) for x in (q, k)]
        if w[0] is None:
            lost[0][2, 1, 40] = True
            lost[0][3, 0, [a[5], b[5]]] = True
            lost[1][4, 1, [a[0], b[0]]] = True
            assert out[0][2, 1, 40].isnan() if bad != bad else out[0][2, 1, 40] == bad
        else:
            lost[0][2, 1] = lost[0][3, 0] = lost[1][4, 1] = True
        for x, y, l, wt in zip((q, k), out, lost, w):
            x = x.masked_fill(l, 0.0) if wt is None else x.masked_fill(l.any(-1, keepdim=True), 1.0)
            ref = oracle.forward(x, pos, f, interleaved, 1.0, wt, EPS)
            bound = forward_bound(x, ref, f, interleaved, 1.0, wt, EPS, BF16)
            keep = ~l
            check(y.cpu()[keep], ref[keep], bound[keep])


def descriptor(q, k, pos, f, **kw):
    r = capi.Rotary(dtype={BF16: capi.DTYPE_BF16, F16: capi.DTYPE_F16, F32: capi.DTYPE_F32}[q.dtype],
                    num_heads_q=q.shape[1], num_heads_kv=k.shape[1], head_dim=q.shape[2], rotary_dim=2 * f.numel(),
                    scale=1.0, eps=EPS, total=q.shape[0], positions=pos.data_ptr(), inv_freq=f.data_ptr())
    for name, x in kw.items():
        setattr(r, name, x)
    return r


@pytest.mark.parametrize("d,shift", [(64, 0), (64, 1), (40, 0), (40, 3)])
def test_in_place_and_unaligned_rows(mt, d, shift):
    """Through the C entry: rows that begin anywhere, at any stride, turned where they lie;
    the gaps between them stay."""
    g = torch.Generator().manual_seed(10)
    m, hq, hkv, gap = 37, 4, 2, 5 if shift else 8
    q, k, _ = rows(m, hq, hkv, d, BF16, g)
    pos, f = torch.arange(m, dtype=torch.int32).cuda(), frequencies(d).cuda()
    want = mt.rotary(q.cuda(), k.cuda(), pos, f)
    stride = (hq + hkv) * d + gap
    buf = torch.full((shift + m * stride,), 7.0, dtype=BF16, device="cuda")
    both = buf[shift:].view(m, stride)
    both[:, :hq * d] = q.view(m, -1).cuda()
    both[:, hq * d:(hq + hkv) * d] = k.view(m, -1).cuda()
    at_q, at_k = both.data_ptr(), both.data_ptr() + 2 * hq * d
    capi.call("mtlattn_rotary_fwd", descriptor(q, k, pos, f), at_q, stride, at_k, stride, at_q, stride, at_k, stride,
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(both[:, :hq * d].reshape(m, hq, d), want[0])
    assert torch.equal(both[:, hq * d:(hq + hkv) * d].reshape(m, hkv, d), want[1])
    assert bool((both[:, (hq + hkv) * d:] == 7).all()) and bool((buf[:shift] == 7).all())


def test_attention_after_rotation_depends_on_distance_alone(mt):
    """Rotated queries and keys of prompts, through varlen attention and back to the
    rows: the same for positions that are all shifted."""
    g = torch.Generator().manual_seed(11)
    lens = [17, 1, 130]
    m = sum(lens)
    q, k, v = [t.cuda().requires_grad_() for t in rows(m, 4, 2, 64, F32, g)]
    cu, f = cu_of(lens, "cuda"), frequencies(64).cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    w = [x.cuda().requires_grad_() for x in weights(64, F32, g)]
    seen = []
    for shift in (0, 4096):
        a, b = mt.rotary(q, k, pos + shift, f, q_weight=w[0], k_weight=w[1])
        out = mt.varlen_attention(a, b, v, cu, cu, max(lens), causal=True)
        seen.append((out, *torch.autograd.grad(out.square().sum(), (q, k, v, *w))))
    # angles differ by roundings: about 20 U a score of size <= 64, through few sums
    for x, y in zip(*seen):
        x, y = x.detach(), y.detach()
        assert float((x - y).abs().max()) <= 2e-4 * float(x.abs().max())


# ---- appended rows ----


def pages_of(kv_lens, page, gen, spare=2):
    need = [-(-n // page) for n in kv_lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((len(kv_lens), max(need + [1])), -1, dtype=torch.int32)
    used = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[used:used + n]
        used += n
    return table, total


def check_append(mt, ql, kl, page, dtype, hq, hkv, d, rot, gen, normed=False, interleaved=False, given=False, behind=0,
                 table=None, pages=None, side_by_side=False, packed=True, with_q=True):
    if table is None:
        table, pages = pages_of(kl, page, gen)
    cu = cu_of(ql).tolist()
    m = cu[-1] + behind
    parts = rows(m, hq, hkv, d, dtype, gen, packed)
    w = weights(d, dtype, gen) if normed else [None, None]
    f = frequencies(rot)
    pos = torch.randint(-5, 1000, (m,), generator=gen, dtype=torch.int32) if given else None
    if side_by_side:
        both = torch.randn(pages, page, 2, hkv, d, generator=gen).to(dtype)
        caches, at = [both[:, :, 0], both[:, :, 1]], both.cuda()
        at = [at[:, :, 0], at[:, :, 1]]
    else:
        caches = [torch.randn(pages, page, hkv, d, generator=gen).to(dtype) for _ in range(2)]
        at = [c.cuda() for c in caches]
    q, k, v = on_gpu(parts, packed)
    with_q = with_q and (normed or rot > 0)
    out = mt.paged_cache_append(k, v, *at, cu_of(ql, "cuda"), cu_of(kl, "cuda"), table.cuda(), q=q if with_q else None,
                                positions=None if pos is None else pos.cuda(), inv_freq=f.cuda() if rot else None,
                                interleaved=interleaved, scale=1.5 if rot else 1.0,
                                q_weight=w[0].cuda() if normed and with_q else None,
                                k_weight=w[1].cuda() if normed else None)
    assert (out is None) == (not with_q)
    where = oracle.places(cu, kl, table, page, pages)
    where += [(-1, 0, -1)] * behind
    place = torch.tensor([p for _, p, _ in where], dtype=torch.int32) if pos is None else pos
    scale = 1.5 if rot else 1.0
    ref = [oracle.forward(x, place, f, interleaved, scale, wt, EPS) for x, wt in zip(parts[:2], w)]
    bounds = [forward_bound(x, r, f, interleaved, scale, wt, EPS, dtype) for x, r, wt in zip(parts[:2], ref, w)]
    keys, vals = caches[0].double().flatten(0, 1).clone(), caches[1].flatten(0, 1).clone()
    far = torch.zeros_like(keys)
    for i, (_, _, row) in enumerate(where):
        if row >= 0:
            keys[row], far[row], vals[row] = ref[1][i], bounds[1][i], parts[2][i]
    check(at[0].flatten(0, 1), keys, far, "k_cache")
    assert torch.equal(at[1].flatten(0, 1).cpu(), vals)
    if with_q:
        none = torch.tensor([s < 0 for s, _, _ in where], dtype=torch.bool)
        ref[0][none] = 0.0
        bounds[0][none] = 0.0
        check(out, ref[0], bounds[0], "q")


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("d,rot,interleaved,page,dtype", [
    (128, 128, False, 16, BF16), (64, 64, True, 48, F16), (80, 32, True, 1, BF16), (96, 24, False, 64, F16),
    (33, 32, False, 7, BF16), (256, 256, False, 32, BF16), (128, 64, True, 256, F16), (64, 0, False, 16, BF16)])
def test_append(mt, d, rot, interleaved, page, dtype, normed):
    g = torch.Generator().manual_seed(d + rot + page)
    # prompts, single tokens, chunks, nothing, more rows than tokens
    ql, kl = [5, 1, 0, 70, 1, 9], [5, 33, 12, 200, 1, 4]
    print(f"\n[case] append D {d} R {rot} page {page} norm {normed}", flush=True)
    check_append(mt, ql, kl, page, dtype, 6, 3, d, rot, g, normed, interleaved, behind=3)
    check_append(mt, ql, kl, page, dtype, 6, 3, d, rot, g, normed, interleaved, given=True, side_by_side=True, packed=False)
    check_append(mt, [1], [1], page, dtype, 4, 1, d, rot, g, normed, interleaved, with_q=False)


@pytest.mark.parametrize("n", [64, 65, 200, 4100])
def test_append_of_many_sequences(mt, n):
    g = torch.Generator().manual_seed(n)
    ql = [(i * 7) % 3 for i in range(n)]
    kl = [x + (i * 13) % 40 for i, x in enumerate(ql)]
    check_append(mt, ql, kl, 16, BF16, 2, 1, 16, 16, g, behind=2)


def test_append_drops_rows_without_a_page(mt):
    """Pages of -1, past the cache, and a table that is too short: those rows alone are
    not written, their queries are still turned."""
    g = torch.Generator().manual_seed(12)
    ql, kl = [20, 40, 3], [20, 90, 3]
    table, pages = pages_of(kl, 16, g, spare=1)
    table[0, 1] = -1
    table[1, 4] = pages + 5
    table[1, 3] = torch.iinfo(torch.int32).min
    check_append(mt, ql, kl, 16, BF16, 4, 2, 64, 64, g, table=table[:, :5], pages=pages)


def test_append_bad_offsets_stay_inside(mt):
    """Offsets that are not rising, negative or past the rows: nothing outside of the
    cache's placed rows is written, nothing read out of range."""
    g = torch.Generator().manual_seed(13)
    q, k, v = [t.cuda() for t in rows(12, 4, 2, 64, BF16, g)]
    cu = torch.tensor([-4, 7, 5, 30], dtype=torch.int32).cuda()
    cu_kv = torch.tensor([0, 9, 3, 2 ** 31 - 1], dtype=torch.int32).cuda()
    caches = torch.zeros(2, 5, 16, 2, 64, dtype=BF16, device="cuda")
    table = torch.tensor([[0, 1], [2, 3], [4, 4]], dtype=torch.int32).cuda()
    out = mt.paged_cache_append(k, v, caches[0], caches[1], cu, cu_kv, table, q=q, inv_freq=frequencies(64).cuda())
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out.float()).all()) and bool(torch.isfinite(caches.float()).all())


def test_append_rows_before_the_first_sequence(mt):
    """Offsets that begin past row 0: the rows before them belong to nobody."""
    g = torch.Generator().manual_seed(20)
    q, k, v = rows(9, 4, 2, 64, BF16, g)
    f = frequencies(64)
    cu, kl, page = [2, 5, 8], [10, 3], 16
    table = torch.tensor([[2], [0]], dtype=torch.int32)
    caches = torch.zeros(2, 3, page, 2, 64, dtype=BF16, device="cuda")
    out = mt.paged_cache_append(k.cuda(), v.cuda(), *caches, torch.tensor(cu).cuda(), torch.tensor([4, 14, 17]).cuda(),
                                table.cuda(), q=q.cuda(), inv_freq=f.cuda())
    pos = torch.tensor([0, 0, 7, 8, 9, 0, 1, 2, 0], dtype=torch.int32)
    ref = [oracle.forward(x, pos, f) for x in (q, k)]
    bounds = [forward_bound(x, r, f, False, 1.0, None, EPS, BF16) for x, r in zip((q, k), ref)]
    mine = torch.tensor([False] * 2 + [True] * 6 + [False])
    check(out[mine.cuda()], ref[0][mine], bounds[0][mine])
    assert bool((out[~mine.cuda()] == 0).all())
    flat = [c.flatten(0, 1).cpu() for c in caches]
    at = torch.tensor([2 * page + 7, 2 * page + 8, 2 * page + 9, 0, 1, 2])
    check(flat[0][at], ref[1][mine], bounds[1][mine])
    assert torch.equal(flat[1][at], v[mine])
    rest = torch.ones(3 * page, dtype=torch.bool)
    rest[at] = False
    assert all(bool((c[rest] == 0).all()) for c in flat)


def test_append_refusals(mt):
    k = torch.zeros(4, 2, 64, dtype=BF16, device="cuda")
    q = torch.zeros(4, 4, 64, dtype=BF16, device="cuda")
    caches = torch.zeros(2, 5, 16, 2, 64, dtype=BF16, device="cuda")
    cu = cu_of([4], "cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    f = frequencies(64).cuda()

    def call(k=k, v=k, kc=caches[0], vc=caches[1], cu=cu, table=table, **kw):
        return mt.paged_cache_append(k, v, kc, vc, cu, cu, table, **kw)

    call()
    with pytest.raises(RuntimeError, match="neither"):
        call(q=q)
    for kw in (dict(k=k.float(), v=k.float(), kc=caches[0].float(), vc=caches[1].float()), dict(kc=caches[0].half()),
               dict(vc=caches[0]), dict(table=table.expand(2, 2)), dict(table=table[:, :0]), dict(table=table[0]),
               dict(kc=caches[0, :, :, :1]), dict(kc=caches[0, :, :8], vc=caches[1, :, :8]), dict(kc=caches[0][..., ::2]),
               dict(inv_freq=f.half()), dict(inv_freq=torch.ones(33, device="cuda")), dict(inv_freq=f.cpu()),
               dict(inv_freq=f, positions=torch.arange(3).cuda()), dict(k_weight=torch.ones(63, device="cuda")),
               dict(k_weight=torch.ones(64, device="cuda", dtype=torch.float16)), dict(q=q[:3], inv_freq=f),
               dict(q=q, inv_freq=f, k_weight=torch.ones(64, device="cuda")), dict(k=caches[0, 0, :4], v=k)):
        with pytest.raises(RuntimeError, match="mtlattn|cache_append"):
            call(**kw)


def test_rotary_refusals(mt):
    q = torch.zeros(4, 4, 64, dtype=BF16, device="cuda")
    k, pos, f = q[:, :2].contiguous(), torch.arange(4).cuda(), frequencies(64).cuda()
    w = torch.ones(64, device="cuda")
    for a, kw in (((q, k[:3], pos, f), {}), ((q, k.half(), pos, f), {}), ((q, k, pos[:3], f), {}),
                  ((q, k, pos, torch.ones(33, device="cuda")), {}), ((q, k, pos, f.double()), {}),
                  ((q.cpu(), k, pos, f), {}), ((q, k, pos.cpu(), f), {}), ((q[..., ::2], k[..., :32], pos, f[:16]), {}),
                  ((q, k, pos, f), dict(q_weight=w)), ((q, k, pos, f), dict(q_weight=w, k_weight=w.half())),
                  ((q, k, pos, f), dict(q_weight=w[:63], k_weight=w)), ((q[0], k[0], pos, f), {}),
                  ((q.double(), k.double(), pos, f), {})):
        with pytest.raises(RuntimeError, match="mtlattn|rotary"):
            mt.rotary(*a, **kw)


# ---- streams and graphs ----


def test_graph_of_a_step(mt):
    """An append with rotated queries, captured once and replayed with new rows and
    offsets between eager calls, on its own stream."""
    g = torch.Generator().manual_seed(14)
    n, hq, hkv, d, page = 5, 8, 2, 128, 16
    table, pages = pages_of([64] * n, page, g)
    table = table.cuda()
    w = [x.cuda() for x in weights(d, BF16, g)]
    f = frequencies(d).cuda()
    caches = torch.zeros(2, pages, page, hkv, d, dtype=BF16, device="cuda")
    mirror = caches.clone()
    q, k, v = [t.cuda() for t in rows(n, hq, hkv, d, BF16, g)]
    cu, cu_kv = cu_of([1] * n, "cuda"), cu_of([1] * n, "cuda")

    def step(c):
        return mt.paged_cache_append(k, v, c[0], c[1], cu, cu_kv, table, q=q, inv_freq=f, q_weight=w[0], k_weight=w[1])

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(caches)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches)
    caches.zero_()
    mirror.zero_()
    for i in range(6):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        cu_kv.copy_(cu_of([1 + (7 * i + s) % 60 for s in range(n)]))
        graph.replay()
        want = step(mirror)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(caches, mirror), i


def test_graph_of_forward_and_backward(mt):
    """The C entries in one graph, replayed with new values; two graphs share the
    workspace, replayed in turn."""
    g = torch.Generator().manual_seed(15)
    m, hq, hkv, d = 50, 4, 2, 64
    q, k, _ = [t.cuda() for t in rows(m, hq, hkv, d, BF16, g)]
    w = [x.cuda() for x in weights(d, F32, g)]
    pos, f = torch.arange(m, dtype=torch.int32).cuda(), frequencies(d).cuda()
    dys = [torch.randn_like(q), torch.randn_like(k)]
    r = descriptor(q, k, pos, f, q_weight=w[0].data_ptr(), k_weight=w[1].data_ptr(), weight_dtype=capi.DTYPE_F32)
    size = capi.lib().mtlattn_rotary_bwd_workspace_size(ctypes.byref(r))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def both(outs):
        sh = torch.cuda.current_stream().cuda_stream
        capi.call("mtlattn_rotary_fwd", r, q.data_ptr(), hq * d, k.data_ptr(), hkv * d, outs[0].data_ptr(), hq * d,
                  outs[1].data_ptr(), hkv * d, sh)
        capi.call("mtlattn_rotary_bwd", r, q.data_ptr(), hq * d, k.data_ptr(), hkv * d, dys[0].data_ptr(), hq * d,
                  dys[1].data_ptr(), hkv * d, outs[2].data_ptr(), hq * d, outs[3].data_ptr(), hkv * d,
                  outs[4].data_ptr(), outs[5].data_ptr(), ws.data_ptr(), size, sh)

    def room():
        return [torch.empty_like(t) for t in (q, k, q, k, *w)]

    eager = room()
    both(eager)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        outs, graph = room(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            both(outs)
        graphs.append((graph, outs))
    for i in range(6):
        for t in (q, k, *dys):
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        graph, outs = graphs[i % 2]
        graph.replay()
        both(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i


def test_graph_of_a_training_step(mt):
    """The differentiable operation and its gradients captured together, replayed with
    new values."""
    g = torch.Generator().manual_seed(17)
    m, d = 70, 128
    data = [t.cuda() for t in (*rows(m, 4, 2, d, BF16, g)[:2], *weights(d, F32, g))]
    dys = [torch.randn_like(t) for t in data[:2]]
    pos, f = torch.arange(m, dtype=torch.int32).cuda(), frequencies(d).cuda()

    def step(q, k, wq, wk):
        out = mt.rotary(q, k, pos, f, q_weight=wq, k_weight=wk)
        return [t.detach() for t in (*out, *torch.autograd.grad(out, (q, k, wq, wk), dys))]

    leaves = [t.clone().requires_grad_() for t in data]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*leaves)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*leaves)
    for i in range(5):
        for t, leaf in zip(data, leaves):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
            leaf.data.copy_(t)
        for t in dys:
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        graph.replay()
        want = step(*[t.clone().requires_grad_() for t in data])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_two_streams(mt):
    g = torch.Generator().manual_seed(16)
    f = frequencies(64).cuda()
    sets = []
    for m in (300, 700):
        q, k, _ = [t.cuda() for t in rows(m, 4, 2, 64, BF16, g)]
        sets.append((q, k, torch.arange(m).cuda(), *[x.cuda() for x in weights(64, BF16, g)]))

    def both(q, k, pos, wq, wk):
        q, k, wq, wk = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        out = mt.rotary(q, k, pos, f, q_weight=wq, k_weight=wk)
        return (*out, *torch.autograd.grad(out, (q, k, wq, wk), (q.detach(), k.detach())))

    want = [both(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(both(*sets[i % 2]))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2])), i
