"""fp64 CPU restatement of attention of drafted tokens' trees over a paged cache.
No counterpart in the reference. Test infrastructure only.
"""

import math

import torch

from . import cache8


def forward(q, k_cache, v_cache, cu_q, kv_lens, table, mask, scale):
    """(out, lse, size, far) in fp64: q [M, Hq, D] and the offsets on the host, caches
    [num_pages, page_size, Hkv, D]; size: the same sums with |v|, far: the largest
    |q| . |k| scale of a row: what errors are relative to.
    Keys that a row does not see take no part; rows of no sequence are 0."""
    pages, page, hkv, d = k_cache.shape
    hq = q.shape[1]
    g = hq // hkv
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    far = torch.zeros(q.shape[:2], dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    for s, kv in enumerate(kv_lens):
        n = cu_q[s + 1] - cu_q[s]
        if n == 0 or kv == 0:
            continue
        at = cache8.rows(table, s, 0, kv, page, pages)
        k = k_cache.flatten(0, 1)[at].double()
        v = v_cache.flatten(0, 1)[at].double()
        for i in range(n):
            see = torch.ones(kv, dtype=torch.bool)
            for j in range(max(0, kv - n), kv):
                node = j - (kv - n)
                see[j] = bool(mask[cu_q[s] + i, node]) if node < mask.shape[1] else False
            if not see.any():
                continue
            ks, vs = k[see], v[see]                                     # [m, hkv, d]
            row = cu_q[s] + i
            for h in range(hq):
                x = (ks[:, h // g] * q[row, h].double()).sum(-1) * scale
                lse[row, h] = torch.logsumexp(x, 0)
                p = torch.exp(x - lse[row, h])[:, None]
                out[row, h] = (p * vs[:, h // g]).sum(0)
                size[row, h] = (p * vs[:, h // g].abs()).sum(0)
                far[row, h] = (ks[:, h // g].abs() * q[row, h].double().abs()).sum(-1).max() * abs(scale)
    return out, lse, size, far
