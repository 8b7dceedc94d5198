"""Inputs and bounds of the tests of attention over trees of drafted tokens."""

import math

import torch

from oracle import tree as oracle
from tests.helpers import cu_of

U = 2.0 ** -24


def random_tree(n, cols, gen):
    """Mask rows of a random tree: each token sees itself and its ancestors."""
    mask = torch.zeros(n, cols, dtype=torch.bool)
    for j in range(n):
        parent = int(torch.randint(max(-1, j - 6), j, (1,), generator=gen)) if j else -1
        if parent >= 0:
            mask[j] = mask[parent]
        if j < cols:
            mask[j, j] = True
    return mask


def tables(kv_lens, page, gen, spare=2):
    """(block table, number of pages): the sequences' pages scattered over a cache."""
    need = [-(-n // page) for n in kv_lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.zeros(len(kv_lens), max(need + [1]), dtype=torch.int32)
    used = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[used:used + n]
        used += n
    return table, total


class Case:
    """Drafted tokens ql over lengths kl (which count them), on the host."""

    def __init__(self, ql, kl, hq, hkv, d, page, dtype, gen, cols=0, masks="tree", behind=0, poison=True):
        self.ql, self.kl, self.dtype, self.page = ql, kl, dtype, page
        self.cols = cols or max(ql + [1])
        self.cu = cu_of(ql).tolist()
        self.table, pages = tables(kl, page, gen)
        m = self.cu[-1] + behind
        self.q = torch.randn(m, hq, d, generator=gen).to(dtype)
        self.k = torch.randn(pages, page, hkv, d, generator=gen).to(dtype)
        self.v = torch.randn(pages, page, hkv, d, generator=gen).to(dtype)
        if masks == "tree":
            self.mask = torch.cat([random_tree(n, self.cols, gen) for n in ql] +
                                  [torch.zeros(behind, self.cols, dtype=torch.bool)])
        else:                                           # anything, rows that see nothing among them
            self.mask = torch.rand(m, self.cols, generator=gen) < 0.5
            self.mask[::3] = False
        self.scale = 1.0 / math.sqrt(d)
        if poison:                                      # what no sequence owns must not come in
            own = torch.zeros(pages * page, dtype=torch.bool)
            for s, n in enumerate(kl):
                j = torch.arange(n)
                own[self.table[s, j // page].long() * page + j % page] = True
            for x in (self.k, self.v):
                x.flatten(0, 1)[~own] = math.nan

    def run(self, mt, q=None, k=None, v=None, mask=None, max_q=None, max_kv=None, lse=True):
        m, hq = self.q.shape[:2]
        out_lse = torch.full((m, hq), 7.0, device="cuda") if lse else None
        out = mt.paged_tree_decode((self.q if q is None else q).cuda(), (self.k if k is None else k).cuda(),
                                   (self.v if v is None else v).cuda(), cu_of(self.ql, "cuda"), cu_of(self.kl, "cuda"),
                                   self.table.cuda(), (self.mask if mask is None else mask).cuda(),
                                   max_q or max(self.ql + [1]), max(self.kl) if max_kv is None else max_kv, self.scale,
                                   out_lse)
        return out, out_lse

    def reference(self):
        return oracle.forward(self.q, self.k, self.v, self.cu, self.kl, self.table, self.mask, self.scale)

    def check(self, out, lse, ref=None):
        """Scores: sums of D exact products in fp32, off by (D + 8) U of sum |q k| scale,
        8 for the factor and the maximum's subtraction; a weight: e^(2 that) - 1, 2^-19 for exp2
        and its argument's rounding, and half a step of the type it is rounded to, once for itself and
        once for the row's sum (in fp16 also half a step of the smallest numbers: 2^-25 a
        key, against a sum of at least 1). Sums over keys in fp32, and their merges: 2 U a key. Then one
        rounding of the result."""
        o, l, size, far = ref or self.reference()
        n = max(self.kl)
        d = self.q.shape[2]
        half = torch.finfo(self.dtype).eps / 2
        delta = (d + 8) * U * far
        rel = torch.expm1(2 * delta) + 2.0 ** -18 + 2 * half + 2 * n * U
        # (the bound takes the largest |v| for the keys whose weights vanish)
        low = n * 2.0 ** -24 * float(torch.nan_to_num(self.v.double(), 0, 0, 0).abs().max()) if self.dtype == torch.float16 else 0.0
        bound = rel[..., None] * size + low + half * o.abs() + 2.0 ** -25
        m = self.cu[-1]
        out, lse = out.double().cpu()[:m], None if lse is None else lse.double().cpu()
        bad = ~((out - o[:m]).abs() <= bound[:m])
        assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, worst "
                               f"{float(((out - o[:m]).abs() / bound[:m])[bad].max()):.2f} of the bound, rows "
                               f"{sorted(set(bad.nonzero()[:, 0].tolist()))[:8]}")
        if lse is not None:
            assert bool((lse[m:] == 7.0).all())
            lse, l, delta = lse[:m], l[:m], delta[:m]
            fin = torch.isfinite(l)
            assert torch.equal(torch.isfinite(lse), fin) and bool((lse[~fin] == -math.inf).all())
            lb = delta + half + n * U + 2.0 ** -18 + 2.0 ** -22 * l.abs() + (n * 2.0 ** -25 if self.dtype == torch.float16 else 0)
            assert bool(((lse - l)[fin].abs() <= lb[fin]).all()), float(((lse - l)[fin].abs() - lb[fin]).max())
