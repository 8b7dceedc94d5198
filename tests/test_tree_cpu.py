"""Attention of drafted tokens' trees without a GPU: the refusals of the C entry, its
workspace, and the oracle against a loop over single scores."""

import ctypes
import math

import pytest
import torch

from mtlattn_amd import capi
from oracle import tree as oracle
from tests.tree_helpers import Case

# addresses that are never dereferenced: calls that end before a launch
Q, K, V, OUT, WS, MASK, TABLE, CU = (i << 40 for i in range(1, 9))


def call(q=Q, q_rs=512, k=K, k_rs=128, v=V, v_rs=128, page=16, pages=64, table=TABLE, bts=8, max_kv=100, mask=MASK,
         mask_rs=8, cols=8, out=OUT, ws=WS, size=1 << 40, **kw):
    p = capi.Problem(dtype=capi.DTYPE_BF16, num_seqs=2, total_q=16, total_kv=0, num_heads_q=8, num_heads_kv=2, head_dim=64,
                     max_seqlen_q=8, scale=0.1, cu_seqlens_q=CU, cu_seqlens_kv=CU)
    for name, x in kw.items():
        setattr(p, name, x)
    rc = capi.lib().mtlattn_tree_decode(ctypes.byref(p), q, q_rs, k, k_rs, v, v_rs, page, pages, table, bts, max_kv, mask,
                                        mask_rs, cols, out, None, ws, size, None)
    return rc, capi.lib().mtlattn_last_error()


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=capi.DTYPE_F32), capi.ERR_UNSUPPORTED), (dict(dtype=9), capi.ERR_INVALID),
    (dict(head_dim=80), capi.ERR_UNSUPPORTED), (dict(head_dim=0), capi.ERR_INVALID), (dict(num_heads_q=7), capi.ERR_INVALID),
    (dict(num_seqs=0), capi.ERR_INVALID), (dict(total_q=-1), capi.ERR_INVALID), (dict(max_seqlen_q=0), capi.ERR_INVALID),
    (dict(scale=math.nan), capi.ERR_INVALID), (dict(scale=-math.inf), capi.ERR_INVALID), (dict(page=8), capi.ERR_INVALID),
    (dict(page=24), capi.ERR_INVALID), (dict(pages=0), capi.ERR_INVALID), (dict(pages=1 << 27), capi.ERR_INVALID),
    (dict(bts=0), capi.ERR_INVALID), (dict(max_kv=-1), capi.ERR_INVALID), (dict(cols=0), capi.ERR_UNSUPPORTED),
    (dict(cols=257), capi.ERR_UNSUPPORTED), (dict(total_q=1 << 30), capi.ERR_UNSUPPORTED), (dict(q=None), capi.ERR_INVALID),
    (dict(k=None), capi.ERR_INVALID), (dict(v=None), capi.ERR_INVALID), (dict(out=None), capi.ERR_INVALID),
    (dict(table=None), capi.ERR_INVALID), (dict(mask=None), capi.ERR_INVALID), (dict(q_rs=504), capi.ERR_INVALID),
    (dict(k_rs=120), capi.ERR_INVALID), (dict(v_rs=0), capi.ERR_INVALID), (dict(mask_rs=-8), capi.ERR_INVALID),
    (dict(q=Q + 8), capi.ERR_UNSUPPORTED), (dict(k=K + 2), capi.ERR_UNSUPPORTED), (dict(v_rs=132), capi.ERR_UNSUPPORTED),
    (dict(out=OUT + 8), capi.ERR_UNSUPPORTED), (dict(k_rs=1 << 24), capi.ERR_UNSUPPORTED),
    (dict(ws=None), capi.ERR_WORKSPACE), (dict(size=100), capi.ERR_WORKSPACE), (dict(ws=WS + 8), capi.ERR_WORKSPACE),
    (dict(cu_seqlens_q=None), capi.ERR_INVALID)])
def test_refusals(kw, rc):
    got, text = call(**kw)
    assert got == rc and text


def test_no_queries():
    assert call(total_q=0, q=None, out=None, ws=None, size=0)[0] == capi.OK


def test_workspace():
    size = capi.lib().mtlattn_tree_decode_workspace_size
    p = capi.Problem(dtype=capi.DTYPE_BF16, num_seqs=1, total_q=8, num_heads_q=8, num_heads_kv=2, head_dim=128,
                     max_seqlen_q=8, scale=0.1, cu_seqlens_q=CU, cu_seqlens_kv=CU)
    assert 0 < size(ctypes.byref(p), 100) < 1 << 20               # a few tiles: a few pieces
    p.max_seqlen_q, p.num_seqs, p.total_q = 64, 64, 4096
    assert size(ctypes.byref(p), 1 << 20) < 80 << 20
    assert size(ctypes.byref(p), -1) == 0
    p.head_dim = 0
    assert size(ctypes.byref(p), 100) == 0


def test_oracle_against_single_scores():
    g = torch.Generator().manual_seed(1)
    c = Case([3, 2], [3, 7], 2, 1, 64, 16, torch.bfloat16, g, masks="any", poison=False)
    out, lse, _, _ = oracle.forward(c.q, c.k, c.v, c.cu, c.kl, c.table, c.mask, 0.3)
    for s, (n, kv) in enumerate(zip(c.ql, c.kl)):
        for i in range(n):
            row = c.cu[s] + i
            for h in range(2):
                total, acc = 0.0, torch.zeros(64, dtype=torch.float64)
                for j in range(kv):
                    if j >= kv - n and not c.mask[row, j - (kv - n)]:
                        continue
                    at = int(c.table[s, j // 16]), j % 16, 0
                    e = math.exp(0.3 * float((c.q[row, h].double() * c.k[at].double()).sum()))
                    total += e
                    acc += e * c.v[at].double()
                if total == 0.0:
                    assert lse[row, h] == -math.inf and bool((out[row, h] == 0).all())
                else:
                    assert math.isclose(float(lse[row, h]), math.log(total), rel_tol=1e-12, abs_tol=1e-12)
                    assert torch.allclose(out[row, h], acc / total, rtol=1e-12, atol=1e-14)
