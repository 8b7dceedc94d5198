"""Decodes over the 8-bit K/V cache, each for a layout of the work that no smaller
one takes: as many kv heads of a workgroup as it has waves, whole sequences or
pieces, and more sequences than the passes over the offsets take at once."""

import ctypes

import torch

from mtlattn_amd import capi

# name: kind, query dtype, hq, hkv, d, page, block, sequences, most queries, longest, window, bias,
#       (waves, kv heads of a workgroup, cut into pieces)
CASES = {
    "pieces, a wave a head, D = 128": ("e4m3", "bf16", 32, 8, 128, 64, 32, 48, 3, 2100, 0, None, (8, 8, True)),
    "pieces, a wave a head, D = 64": ("int8", "fp16", 32, 8, 64, 16, 16, 64, 1, 2100, 0, None, (8, 8, True)),
    "pieces, a wave a head, two head groups": ("int8", "bf16", 64, 8, 128, 48, 16, 20, 4, 3000, 0, None, (8, 8, True)),
    "pieces, a wave a head, window": ("e4m3", "fp16", 8, 8, 64, 32, 32, 67, 2, 6000, 2500, None, (8, 8, True)),
    "whole, a wave a head, D = 64": ("int8", "fp16", 16, 16, 64, 16, 16, 130, 2, 400, 0, None, (8, 8, False)),
    "whole, a wave a head, D = 128": ("e4m3", "bf16", 32, 16, 128, 64, 64, 130, 1, 300, 60, None, (8, 8, False)),
    "pieces, a wave a head, bias, D = 64": ("e4m3", "bf16", 8, 4, 64, 32, 16, 24, 2, 3000, 0, "head", (4, 4, True)),
    "pieces, a wave a head, bias, D = 128": ("int8", "fp16", 8, 4, 128, 64, 64, 24, 1, 3000, 0, "row", (4, 4, True)),
    "whole, a wave a head, bias": ("int8", "bf16", 16, 16, 64, 16, 16, 130, 1, 200, 0, "row", (4, 4, False)),
    "pieces, window, 203 sequences": ("int8", "fp16", 4, 2, 64, 64, 32, 203, 3, 5000, 2100, None, (8, 2, True)),
    "pieces, 450 sequences": ("e4m3", "bf16", 4, 2, 64, 16, 16, 450, 2, 2500, 0, None, (8, 2, True)),
    "pieces, 700 sequences, one head": ("int8", "fp16", 4, 1, 128, 32, 32, 700, 1, 2200, 0, None, (8, 1, True)),
}


def lengths(name):
    """(query lengths, kv lengths), ragged: one sequence of the longest, runs of 64 and
    more that have no keys or no queries where there are many."""
    _, _, _, _, _, _, _, n, most, longest, _, _, _ = CASES[name]
    g = torch.Generator().manual_seed(n + longest)
    kv = torch.randint(1, (longest if n < 100 else min(longest, 500)) + 1, (n,), generator=g).tolist()
    ql = torch.randint(1, most + 1, (n,), generator=g).tolist()
    for i in range(3, n, 7):
        kv[i] = 0
    for i in range(1, n, 11):
        ql[i] = 0
    if n > 200:
        kv[66:132] = [0] * 66
        ql[134:199] = [0] * 65
    if n > 400:
        kv[256:330] = [0] * 74
        ql[340:410] = [0] * 70
    for i, x in ((0, longest // 3), (n // 2, longest), (n - 1, longest - 37)):
        kv[i], ql[i] = x, most
    return ql, kv


def layout(name):
    """(waves, heads, cut) that the library says of the case."""
    _, dt, hq, hkv, d, _, _, n, most, longest, window, bias, _ = CASES[name]
    ql, kv = lengths(name)
    at = 0x1000                                     # (never dereferenced)
    p = capi.Problem(dtype=capi.DTYPE_BF16 if dt == "bf16" else capi.DTYPE_F16, num_seqs=n, total_q=sum(ql),
                     total_kv=sum(kv), num_heads_q=hq, num_heads_kv=hkv, head_dim=d, max_seqlen_q=most, scale=1.0,
                     causal=1, window=window, cu_seqlens_q=at, cu_seqlens_kv=at)
    if bias:
        p.bias, p.bias_kv_cols = at, longest
    got = [ctypes.c_int32() for _ in range(3)]
    capi.call("mtlattn_decode8_layout", ctypes.byref(p), longest, *[ctypes.byref(x) for x in got])
    return got[0].value, got[1].value, got[2].value > 0
