"""fp64 CPU restatement of the 8-bit paged K/V cache: rows written into it and
read back. No counterpart in the reference. Test infrastructure only.

One side (K or V) at a time: `codes` [num_pages, page_size, Hkv, D]
(float8_e4m3fn or int8), `scale` fp32 [num_pages, page_size / block, Hkv],
`table` [B, max_pages], offsets as lists.
"""

import math

import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def nearest_code(x, dtype):
    """The codes' values nearest to x (fp64), ties to even, saturating; NaN is
    NaN in e4m3 and 0 in int8."""
    x = x.clamp(-QMAX[dtype], QMAX[dtype])
    if dtype == torch.int8:
        return torch.where(torch.isnan(x), torch.zeros_like(x), x).round()
    # three bits after the leading one; 2^-9 is the smallest step
    e = torch.floor(torch.log2(torch.nan_to_num(x).abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def scale_for(amax, dtype):
    """fp32 scale of a block whose largest finite magnitude is amax."""
    amax = max(float(amax), 2.0 ** -92)
    if dtype == torch.int8:
        return float(torch.tensor(amax, dtype=torch.float32) * torch.tensor(1.0 / 127.0, dtype=torch.float32))
    k = math.ceil(math.log2(amax / 448.0))
    while 448.0 * 2.0 ** k < amax:
        k += 1
    while 448.0 * 2.0 ** (k - 1) >= amax:
        k -= 1
    return 2.0 ** k


def write(codes, scale, x, cu, kv_lens, table):
    """x [M, Hkv, D] written in place: token by token into its block's list,
    then block by block."""
    pages, page, hkv, _ = codes.shape
    block = page // scale.shape[1]
    dtype = codes.dtype
    for s, kv in enumerate(kv_lens):
        n = cu[s + 1] - cu[s]
        p0 = kv - n
        blocks = {}
        for i in range(n):
            pos = p0 + i
            if pos >= 0 and pos // page < table.shape[1] and 0 <= int(table[s, pos // page]) < pages:
                blocks.setdefault(pos // block, []).append((pos, cu[s] + i))
        for b, rows in blocks.items():
            pg, off = int(table[s, b * block // page]), b * block % page
            sub = off // block
            held = max(0, p0 - b * block)
            new = x[[r for _, r in rows]].double()
            at = [off + pos - b * block for pos, _ in rows]
            for h in range(hkv):
                mag = new[:, h].abs()
                mag = mag[torch.isfinite(mag)]
                need = scale_for(mag.max() if mag.numel() else 0.0, dtype)
                old = float(scale[pg, sub, h])
                now = max(old, need) if held else need
                if held and now > old:
                    c = codes[pg, off:off + held, h].double()
                    codes[pg, off:off + held, h] = nearest_code(c * old / now, dtype).to(torch.float32).to(dtype)
                codes[pg, at, h] = nearest_code(new[:, h] / now, dtype).to(torch.float32).to(dtype)
                scale[pg, sub, h] = now


def rows(table, s, lo, hi, page, pages):
    """Cache rows of tokens [lo, hi) of sequence s, columns and pages clamped."""
    j = torch.arange(lo, hi)
    col = (j // page).clamp(max=table.shape[1] - 1)
    return table[s, col].long().clamp(0, pages - 1) * page + j % page


def values(codes, scale):
    """fp64 values [num_pages * page_size, Hkv, D] of the whole cache."""
    block = codes.shape[1] // scale.shape[1]
    v = codes.double() * scale.double().repeat_interleave(block, 1).unsqueeze(-1)
    return v.flatten(0, 1)


def read(codes, scale, cu, kv_lens, table, total):
    """The last cu[s + 1] - cu[s] tokens of each sequence, fp64 [total, Hkv, D];
    rows of no sequence and of negative positions are 0."""
    v = values(codes, scale)
    out = torch.zeros((total, *codes.shape[2:]), dtype=torch.float64)
    for s, kv in enumerate(kv_lens):
        n = cu[s + 1] - cu[s]
        m = min(n, kv)
        out[cu[s + 1] - m:cu[s + 1]] = v[rows(table, s, kv - m, kv, codes.shape[1], codes.shape[0])]
    return out
