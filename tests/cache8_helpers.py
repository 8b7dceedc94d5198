"""Inputs and bounds of the tests of the 8-bit K/V cache."""

import math

import torch

import oracle
from oracle import cache8
from tests.helpers import cu_of

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def pages_for(kv_lens, page, gen, spare=2, width=0):
    """(block table [B, max_pages], number of pages): the sequences' pages
    scattered over a cache with some of them free."""
    need = [-(-n // page) for n in kv_lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.zeros((len(kv_lens), max(max(need), 1, width)), dtype=torch.int32)
    used = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[used:used + n]
        used += n
    return table, total


def random_cache(kind, pages, page, hkv, d, block, gen):
    """(codes, scale) of one side: codes over their whole range, scales from
    1/512 to 1/32 (powers of two in e4m3)."""
    dt = CODES[kind]
    top = cache8.QMAX[dt]
    x = (torch.randn(pages, page, hkv, d, generator=gen) * top / 4).clamp_(-top, top)
    codes = (x.round_() if kind == "int8" else x).to(dt)
    e = torch.randint(-9, -5, (pages, page // block, hkv), generator=gen).float()
    scale = torch.exp2(e)
    if kind == "int8":
        scale = scale * (0.5 + torch.rand(scale.shape, generator=gen))
    return codes, scale


def poison_free_rows(codes, kv_lens, table):
    """Rows that no sequence owns get NaN codes (e4m3) or the largest (int8):
    what an attention must not let in."""
    own = torch.zeros(codes.shape[0] * codes.shape[1], dtype=torch.bool)
    for s, kv in enumerate(kv_lens):
        own[cache8.rows(table, s, 0, kv, codes.shape[1], codes.shape[0])] = True
    raw = codes.view(torch.uint8).flatten(0, 1)
    raw[~own] = 0x7f


def same_codes(a, b):
    """Equal codes, the two NaN patterns of e4m3 taken as one."""
    x, y = a.cpu(), b.cpu()
    if x.dtype == torch.int8:
        return torch.equal(x, y)
    x, y = x.view(torch.uint8), y.view(torch.uint8)
    nan = ((x & 0x7f) == 0x7f) & ((y & 0x7f) == 0x7f)
    # (-0 and 0 are the same value)
    zero = ((x & 0x7f) == 0) & ((y & 0x7f) == 0)
    return bool(((x == y) | nan | zero).all())


def decode_reference(q, kcache, kscale, vcache, vscale, cu_q, kv_lens, table, scale, causal=False, window=0, bias=None):
    """(out, lse, bound) in fp64 of attention over the cache's values, and how
    far a kernel's out may be from it by its arithmetic, without the output's
    own rounding.

    Scores are sums of D exact products in fp32: off by at most
    (D + 8) 2^-24 sum |q k| scale, the 8 for the two multiplications, the bias
    and the maximum's subtraction in the exponent's base; a weight's relative
    error is e^delta - 1 with twice that (its own and the sum's), 2^-21 for exp2
    and its argument's rounding (|x| up to 2^6 at 2^-24 each). The weights enter
    the product with two bf16 parts: 2^-17 relative. Accumulating n keys in fp32 and merging
    splits: n 2^-24 of sum p |v|."""
    kv = cache8.values(kcache, kscale)
    vv = cache8.values(vcache, vscale)
    page, pages = kcache.shape[1], kcache.shape[0]
    at = torch.cat([cache8.rows(table, s, 0, n, page, pages) for s, n in enumerate(kv_lens)])
    k, v = kv[at], vv[at]
    cq, ck = cu_of([cu_q[i + 1] - cu_q[i] for i in range(len(cu_q) - 1)]), cu_of(kv_lens)
    args = (scale, causal, window, bias)
    out, lse = oracle.varlen_forward(q.double(), k, v, cq, ck, *args, dtype=torch.float64)
    size, _ = oracle.varlen_forward(q.double(), k, v.abs(), cq, ck, *args, dtype=torch.float64)
    d, g = q.shape[2], q.shape[1] // k.shape[1]
    delta = torch.zeros(q.shape[0], q.shape[1], dtype=torch.float64)
    k0 = 0
    for s, n in enumerate(kv_lens):
        if n:
            ka = k[k0:k0 + n].abs().repeat_interleave(g, 1).permute(1, 2, 0).contiguous()
            qa = q[cu_q[s]:cu_q[s + 1]].double().abs().transpose(0, 1).contiguous()
            delta[cu_q[s]:cu_q[s + 1]] = (torch.matmul(qa, ka).amax(-1).transpose(0, 1) if qa.shape[1] else 0.0)
        k0 += n
    delta = (d + 8) * 2.0 ** -24 * delta * scale
    n = max(list(kv_lens) + [1])
    rel = torch.expm1(2 * delta) + 2.0 ** -17 + 2.0 ** -17 + n * 2.0 ** -24
    return out, lse, rel.unsqueeze(-1) * size, delta + n * 2.0 ** -24 + 2.0 ** -20


def check_decode(out, lse, ref, ref_lse, bound, lse_bound, dtype):
    """Half a step of the output's type, and the arithmetic's bound. (An fp16
    value below its normal range is rounded to a step of 2^-24.)"""
    out = out.double().cpu()
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + bound + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    bad = ~((out - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((out - ref).abs().max()):.3e}"
    if lse is not None:
        lse = lse.double().cpu()
        fin = torch.isfinite(ref_lse)
        assert torch.equal(torch.isfinite(lse), fin)
        assert bool((lse[~fin] == -math.inf).all())
        # (the LSE itself is rounded to fp32)
        assert bool(((lse - ref_lse)[fin].abs() <= (lse_bound + 2.0 ** -23 * ref_lse.abs())[fin]).all())
