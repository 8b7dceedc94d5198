"""Operators on a paged K/V cache held in 8 bits: writing it, reading it back,
and decode attention over it.

The cache is [num_pages, page_size, Hkv, D] of codes (e4m3 or int8) with an
fp32 scale for each block of tokens and kv head, [num_pages, page_size / block,
Hkv]; a value is its code times its scale. Logical token j of sequence s lies
in page block_table[s, j // page_size]. Each case is a dict of plain values;
`run` computes it in elementary torch operations, or, where `own` is set, with
the library's kernels.
"""

import math
import random

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_QMAX = {"e4m3": 448.0, "int8": 127.0}
# the scale of a block is made for a largest magnitude of at least this
_AMAX_MIN = 2.0 ** -92

# kind: "write" (new rows into the cache, and what their blocks then hold),
# "read" (the cache's rows as fp16/bf16/fp32), "decode" (attention).
# kv lengths are drawn from lens_seed over [kv_lo, kv_hi] and count the new
# tokens (write) or the queries (decode): [q_lo, q_hi] of them per sequence, all
# tokens when q_hi is 0.
_BASE = {"kind": "decode", "cache": "e4m3", "dtype": "bf16", "n": 1, "q_lo": 0, "q_hi": 0, "kv_lo": 1, "kv_hi": 1,
         "lens_seed": 0, "hq": 32, "hkv": 8, "d": 128, "page": 64, "block": 64, "causal": True, "window": 0,
         "bias": "none"}


def _case(**kw):
    c = dict(_BASE)
    c.update(kw)
    return c


def listed():
    return [
        # one token of each sequence of a chat batch: the smallest write, every step of a server
        _case(name="write_step", kind="write", n=64, q_lo=1, q_hi=1, kv_lo=128, kv_hi=4096, lens_seed=1, page=16,
              block=16),
        # a few prompts at once, from empty sequences, in int8
        _case(name="write_prompts", kind="write", cache="int8", dtype="fp16", n=5, kv_lo=33, kv_hi=1900, lens_seed=2,
              d=64, hkv=16, page=64, block=32),
        # a long prompt's chunks for a batch: the largest write
        _case(name="write_chunks", kind="write", n=8, q_lo=8000, q_hi=8192, kv_lo=9000, kv_hi=40000, lens_seed=3,
              page=64, block=64),
        # the context of a few short sequences, before a prompt's next chunk
        _case(name="read_short", kind="read", cache="int8", n=3, kv_lo=33, kv_hi=700, lens_seed=4, page=16, block=16),
        # the contexts of a batch of long sequences
        _case(name="read_contexts", kind="read", dtype="fp16", n=8, kv_lo=2048, kv_hi=32768, lens_seed=5, page=128,
              block=128),
        # one user, a short context: the smallest decode, where latency counts
        _case(name="decode_one", n=1, q_lo=1, q_hi=1, kv_lo=700, kv_hi=700, page=16, block=16),
        # a chat batch, int8
        _case(name="decode_chat", cache="int8", n=16, q_lo=1, q_hi=1, kv_lo=128, kv_hi=2048, lens_seed=6),
        # one very long context
        _case(name="decode_document", n=1, q_lo=1, q_hi=1, kv_lo=131071, kv_hi=131071, cache="int8", dtype="fp16",
              page=256, block=128),
        # speculative tokens, ragged
        _case(name="decode_speculative", n=24, q_lo=1, q_hi=4, kv_lo=1024, kv_hi=8192, lens_seed=7, dtype="fp16",
              page=16, block=16),
        # sliding window, D = 64, without grouped heads
        _case(name="decode_window", cache="int8", n=32, q_lo=1, q_hi=1, kv_lo=512, kv_hi=16384, lens_seed=8, hq=16,
              hkv=16, d=64, window=2048, page=32, block=32),
        # a batch of long contexts: the largest stream
        _case(name="decode_long", n=64, q_lo=1, q_hi=1, kv_lo=8192, kv_hi=65536, hq=64, hkv=8, lens_seed=9),
        # the same in int8 with fewer sequences and heads
        _case(name="decode_long_int8", cache="int8", n=12, q_lo=1, q_hi=2, kv_lo=4096, kv_hi=65536, lens_seed=10,
              page=128, block=32),
    ]


def _loguniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "decode"])
    cache = rng.choice(["e4m3", "int8"])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    block = rng.choice([b for b in (16, 32, 64, 128, 256) if page % b == 0])
    seed = rng.randrange(1 << 20)
    if kind != "decode":
        d = rng.choice([64, 80, 96, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8, 16]) if d <= 128 else rng.choice([2, 4, 8])
        # (all tokens of all sequences, at most as many values as the largest listed write)
        n = _loguniform(rng, 1, 64)
        top = max(64, min(40000, (1 << 27) // (n * hkv * d)))
        lo = _loguniform(rng, 1, top)
        hi = _loguniform(rng, lo, top)
        c = _case(kind=kind, cache=cache, dtype=rng.choice(["bf16", "fp16", "fp32"]), n=n, kv_lo=lo, kv_hi=hi,
                  lens_seed=seed, hq=hkv, hkv=hkv, d=d, page=page, block=block)
        if rng.random() < 0.6:              # the last tokens alone
            c["q_hi"] = _loguniform(rng, 1, hi)
            c["q_lo"] = _loguniform(rng, 1, c["q_hi"])
        return c
    d = rng.choice([64, 128, 128])
    hq, hkv = rng.choice([(8, 8), (16, 16), (12, 4), (16, 2), (32, 8), (32, 4), (64, 8), (28, 4)])
    n = _loguniform(rng, 1, 64)
    top = max(256, min(131072, (1 << 30) // (n * hkv * d)))
    lo = _loguniform(rng, 17, top)
    hi = _loguniform(rng, lo, top)
    q_hi = rng.choice([1, 1, 1, 2, 4, 8, 16])
    bias = "alibi" if n * hi <= 65536 and rng.random() < 0.3 else "none"
    return _case(cache=cache, dtype=rng.choice(["bf16", "bf16", "fp16"]), n=n, q_lo=1, q_hi=q_hi, kv_lo=lo, kv_hi=hi,
                 lens_seed=seed, hq=hq, hkv=hkv, d=d, page=page, block=block, causal=rng.random() < 0.8,
                 window=rng.choice([0, 0, 0, _loguniform(rng, 32, 4096)]), bias=bias)


def _lens(case):
    """(lengths of the last tokens that the call is about, kv lengths)."""
    rng = random.Random(case["lens_seed"])
    kv = [rng.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["n"])]
    if case["q_hi"] == 0:
        return list(kv), kv
    return [min(x, rng.randint(case["q_lo"], case["q_hi"])) for x in kv], kv


def _tails(case):
    """Tokens of each sequence from the first block that a write touches."""
    ql, kl = _lens(case)
    return [b - (b - a) // case["block"] * case["block"] for a, b in zip(ql, kl)]


def _cu(lens, device):
    c = [0]
    for x in lens:
        c.append(c[-1] + x)
    return torch.tensor(c, dtype=torch.int32, device=device)


def _codes(case, g, shape):
    """Random codes of a cache, in pieces (the fp32 values take four times their room)."""
    out = torch.empty(shape, dtype=_CODES[case["cache"]], device="cuda")
    top = _QMAX[case["cache"]]
    step = max(1, (1 << 27) // (shape[1] * shape[2] * shape[3]))
    for i in range(0, shape[0], step):
        part = torch.randn((min(step, shape[0] - i), *shape[1:]), generator=g, device="cuda")
        part *= top / 4.0
        part = part.clamp_(-top, top)
        out[i:i + step] = (part.round_() if case["cache"] == "int8" else part).to(out.dtype)
    return out


def _scales(case, g, shape):
    """Scales of values of about unit size, larger in some blocks than in others."""
    spread = torch.randint(-1, 3, shape, generator=g, device="cuda").float()
    if case["cache"] == "e4m3":
        return torch.exp2(spread - 7.0)
    return torch.exp2(spread - 5.0) * (0.5 + torch.rand(shape, generator=g, device="cuda"))


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    ql, kl = _lens(case)
    hkv, d, page, block, n = case["hkv"], case["d"], case["page"], case["block"], case["n"]
    s = {"case": case, "total": sum(ql), "max_q": max(ql), "max_kv": max(kl), "cu_q": _cu(ql, dev),
         "cu_kv": _cu(kl, dev)}
    # a cache with some of its pages free, the sequences' pages scattered in it
    pages = [-(-x // page) for x in kl]
    total = sum(pages) + sum(pages) // 16 + 1
    for x in ("k", "v"):
        s[x + "_cache"] = _codes(case, g, (total, page, hkv, d))
        s[x + "_scale"] = _scales(case, g, (total, page // block, hkv))
    perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((n, max(pages)), dtype=torch.int32, device=dev)
    used = 0
    for i, p in enumerate(pages):
        table[i, :p] = perm[used:used + p]
        used += p
    s["table"] = table

    def rand(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if case["kind"] == "write":
        # a few channels of keys are much larger than the others
        gain = torch.exp(0.7 * rand(1, hkv, d))
        s["k"] = (rand(sum(ql), hkv, d) * gain).to(dt)
        s["v"] = rand(sum(ql), hkv, d).to(dt)
        tails = _tails(case)
        s["cu_tail"], s["total_tail"] = _cu(tails, dev), sum(tails)
    if case["kind"] == "decode":
        s["q"] = rand(sum(ql), case["hq"], d).to(dt)
        s["scale"] = 1.0 / math.sqrt(d)
        s["bias"] = None
        if case["bias"] == "alibi":         # a slope per head, on sequence-local positions
            slope = torch.exp2(-8.0 * torch.arange(1, case["hq"] + 1, device=dev) / case["hq"])
            rows = [torch.arange(b - a, b, device=dev) for a, b in zip(ql, kl)]
            far = (torch.cat(rows)[:, None] - torch.arange(max(kl), device=dev)[None, :]).clamp_(min=0).float()
            s["bias"] = -slope[None, :, None] * far[:, None, :]
    return s


def _places(s, cu, total):
    """(sequence, cache row) of the `total` last tokens that cu gives to the sequences."""
    page = s["case"]["page"]
    row = torch.arange(total, dtype=torch.int32, device=cu.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    kv = s["cu_kv"][1:] - s["cu_kv"][:-1]
    pos = ((kv + cu[:-1] - cu[1:])[seq] + row - cu[seq]).long()
    return seq, s["table"][seq, pos // page].long() * page + pos % page


def _value(s, x, rows):
    """The values [..., Hkv, D] in fp32 of cache rows."""
    c = s["case"]
    cache, scale = s[x + "_cache"], s[x + "_scale"]
    codes = cache.view(torch.uint8).flatten(0, 1)[rows].view(cache.dtype).float()
    return codes.mul_(scale.flatten(0, 1)[rows // c["block"]].unsqueeze(-1))


def _round_codes(x, case):
    """The codes nearest to x (64 bits: a quotient can lie next to a border)."""
    top = _QMAX[case["cache"]]
    x = x.clamp(-top, top)
    if case["cache"] == "int8":
        return x.nan_to_num(nan=0.0).round().to(torch.int8)
    return x.to(torch.float8_e4m3fn)


def _need(amax, case):
    """The scale that a block with this largest magnitude needs."""
    amax = amax.clamp(min=_AMAX_MIN)
    if case["cache"] == "int8":
        return amax / 127.0
    m, e = torch.frexp(amax)                # amax = m 2^e, 448 = 0.875 * 2^9
    return torch.ldexp(torch.ones_like(m), e - 9 + (m > 0.875))


def _plain_write(s):
    c = s["case"]
    block, hkv, d = c["block"], c["hkv"], c["d"]
    cu, kv = s["cu_q"], s["cu_kv"][1:] - s["cu_kv"][:-1]
    _, rows = _places(s, cu, s["total"])
    # the earlier tokens in the block of each sequence's first new one
    p0 = kv - (cu[1:] - cu[:-1])
    first = p0 // block * block
    i = torch.arange(block, device=cu.device)
    has = i[None, :] < (p0 - first)[:, None]
    # (a sequence without earlier tokens there takes any row, which is written back as it is)
    col = (first // c["page"]).clamp(max=s["table"].shape[1] - 1).long()
    start = s["table"].gather(1, col[:, None])[:, 0].long() * c["page"] + first % c["page"]
    held = (start[:, None] + i[None, :])[has]
    for x in ("k", "v"):
        cache, scale = s[x + "_cache"], s[x + "_scale"]
        flat = scale.view(-1, hkv)
        new = s[x].float()
        mag = new.abs().masked_fill(~torch.isfinite(new), 0.0).amax(-1)
        amax = torch.full_like(flat, -1.0)
        amax.scatter_reduce_(0, (rows // block)[:, None].expand(-1, hkv), mag, "amax")
        touched = amax >= 0
        need = _need(amax, c)
        kept = torch.zeros(flat.shape[0], dtype=torch.bool, device=cu.device)
        kept[held // block] = True
        now = torch.where(kept[:, None] & touched, torch.maximum(flat, need), torch.where(touched, need, flat))
        codes = cache.view(torch.uint8).view(-1, hkv, d)
        old = codes[held].view(cache.dtype).double() * flat[held // block].unsqueeze(-1)
        codes[held] = _round_codes(old / now[held // block].unsqueeze(-1), c).view(torch.uint8)
        codes[rows] = _round_codes(new.double() / now[rows // block].unsqueeze(-1), c).view(torch.uint8)
        flat.copy_(now)
    return s["k_scale"], s["v_scale"]


def _plain_read(s, cu, total):
    _, rows = _places(s, cu, total)
    dt = _DTYPES[s["case"]["dtype"]]
    return _value(s, "k", rows).to(dt), _value(s, "v", rows).to(dt)


def _plain_decode(s):
    c = s["case"]
    n, hq, hkv, d, page = c["n"], c["hq"], c["hkv"], c["d"], c["page"]
    g, L, Q = hq // hkv, s["max_kv"], s["max_q"]
    dev = s["q"].device
    ql, kl = s["cu_q"][1:] - s["cu_q"][:-1], s["cu_kv"][1:] - s["cu_kv"][:-1]
    j = torch.arange(L, device=dev)
    rows = s["table"][:, j // page].long() * page + j % page
    i = torch.arange(Q, device=dev)
    q = s["q"].float()[(s["cu_q"][:-1, None] + i).clamp(max=s["total"] - 1).long()]      # [n, Q, hq, d]
    q = q.view(n, Q, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * Q, d)
    S = torch.matmul(q, _value(s, "k", rows).permute(0, 2, 3, 1)).mul_(s["scale"]).view(n, hq, Q, L)
    if s["bias"] is not None:
        at = (s["cu_q"][:-1, None] + i).clamp(max=s["total"] - 1).long()
        S += s["bias"][at].transpose(1, 2)
    end = (i[None, :] + (kl - ql)[:, None])[:, :, None]                # last key that a causal query sees
    see = (j < kl[:, None, None]) & (i[None, :, None] < ql[:, None, None])
    if c["causal"]:
        see = see & (j <= end)
    if c["window"] > 0:
        see = see & (j > end - c["window"])
    S.masked_fill_(~see[:, None], float("-inf"))
    top = S.amax(-1, keepdim=True)
    P = S.sub_(top.masked_fill(top == float("-inf"), 0.0)).exp_()
    total = P.sum(-1, keepdim=True)
    P.div_(total.masked_fill(total == 0, 1.0))
    O = torch.matmul(P.view(n, hkv, g * Q, L), _value(s, "v", rows).transpose(1, 2))
    O = O.view(n, hq, Q, d).transpose(1, 2)
    row = torch.arange(s["total"], dtype=torch.int32, device=dev)
    seq = torch.searchsorted(s["cu_q"], row, right=True) - 1
    return O[seq, (row - s["cu_q"][seq]).long()].to(s["q"].dtype)


def run(state):
    s = state
    c = s["case"]
    if own:
        import mtlattn

        caches = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        dt = _DTYPES[c["dtype"]]
        if c["kind"] == "write":
            mtlattn.paged_cache_write(s["k"], s["v"], *caches, s["cu_q"], s["cu_kv"], s["table"])
            k, v = mtlattn.paged_cache_read(*caches, s["cu_tail"], s["cu_kv"], s["table"], s["total_tail"], dtype=dt)
            return k, v, s["k_scale"], s["v_scale"]
        if c["kind"] == "read":
            return mtlattn.paged_cache_read(*caches, s["cu_q"], s["cu_kv"], s["table"], s["total"], dtype=dt)
        return mtlattn.paged_decode(s["q"], s["k_cache"], s["v_cache"], s["cu_q"], s["cu_kv"], s["table"], s["max_q"],
                                    s["max_kv"], scale=s["scale"], causal=c["causal"], window=c["window"],
                                    attn_bias=s["bias"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if c["kind"] == "write":
        scales = _plain_write(s)
        return (*_plain_read(s, s["cu_tail"], s["total_tail"]), *scales)
    if c["kind"] == "read":
        return _plain_read(s, s["cu_q"], s["total"])
    return _plain_decode(s)


def work(case):
    ql, kl = _lens(case)
    hkv, d, block = case["hkv"], case["d"], case["block"]
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "write":
        # new rows in, their codes out, the codes of the blocks' earlier rows
        # in, the blocks' values out; the blocks' scales in and out
        held = sum(_tails(case)) - sum(ql)
        blocks = sum(-(-t // block) for t in _tails(case))
        return {"bytes": 2 * hkv * (d * (es * sum(ql) + sum(ql) + held + es * sum(_tails(case))) + 8 * blocks),
                "flops": 2 * 2 * hkv * d * sum(ql)}
    if case["kind"] == "read":
        blocks = sum(-(-b // block) - (b - a) // block for a, b in zip(ql, kl))
        return {"bytes": 2 * hkv * (d * (1 + es) * sum(ql) + 4 * blocks), "flops": 2 * hkv * d * sum(ql)}
    pairs = keys = blocks = 0
    for a, b in zip(ql, kl):
        lows = []
        for i in range(a):
            end = i + b - a
            hi = min(b, end + 1) if case["causal"] else b
            lo = max(0, end - case["window"] + 1) if case["window"] > 0 else 0
            pairs += max(0, hi - lo)
            lows.append(lo)
        lo = min(lows)
        keys += b - lo
        blocks += -(-b // block) - lo // block
    bias = 4 * case["hq"] * pairs if case["bias"] != "none" else 0
    return {"bytes": 2 * hkv * (d * keys + 4 * blocks) + 2 * es * sum(ql) * case["hq"] * d + bias,
            "flops": 4 * d * case["hq"] * pairs}


def _exact_values(s, x, i, lo, hi, cache=None, scale=None):
    """Tokens [lo, hi) of sequence i in 64 bits."""
    c = s["case"]
    cache = s[x + "_cache"] if cache is None else cache
    scale = s[x + "_scale"] if scale is None else scale
    j = torch.arange(lo, hi, device=s["table"].device)
    pg, off = s["table"][i, j // c["page"]].long(), j % c["page"]
    codes = cache.view(torch.uint8)[pg, off].view(cache.dtype) if cache.element_size() == 1 else cache[pg, off]
    return codes.to(torch.float64) * scale[pg, off // c["block"]].to(torch.float64)[:, :, None]


def _exact_write(s, ql, kl):
    """Block by block of a sequence, from the definition: all that the block
    then holds, on the scale of its largest magnitude."""
    c = s["case"]
    block, page, top = c["block"], c["page"], _QMAX[c["cache"]]
    found = []
    for x in ("k", "v"):
        scale = s[x + "_scale"].to(torch.float64)
        out, q0 = [], 0
        for i, (a, b) in enumerate(zip(ql, kl)):
            p0 = b - a
            lo = p0 // block * block
            new = s[x][q0:q0 + a].to(torch.float64)
            q0 += a
            rows = torch.cat([_exact_values(s, x, i, lo, p0), new])
            nb = -(-(b - lo) // block)
            pad = torch.zeros((nb * block - rows.shape[0], *rows.shape[1:]), dtype=torch.float64, device=rows.device)
            rows = torch.cat([rows, pad]).view(nb, block, c["hkv"], c["d"])
            fresh = rows.clone()
            fresh[0, :p0 - lo] = 0
            amax = fresh.abs().amax((1, 3)).clamp(min=_AMAX_MIN)
            if c["cache"] == "int8":
                need = (amax / top).float().double()
            else:
                need = torch.exp2(torch.ceil(torch.log2(amax / top)))
                need = torch.where(need * top < amax, need * 2, need)
                need = torch.where(need / 2 * top >= amax, need / 2, need)
            first = lo + block * torch.arange(nb, device=rows.device)
            pg, sub = s["table"][i, first // page].long(), first % page // block
            if p0 > lo:
                need[0] = torch.maximum(need[0], scale[pg[0], sub[0]])
            scale[pg, sub] = need
            unit = (rows / need[:, None, :, None]).clamp(-top, top)
            if c["cache"] == "int8":
                unit = unit.round()
            else:               # three bits after the leading one, 2^-9 the smallest step
                e = torch.floor(torch.log2(unit.abs().clamp(min=2.0 ** -6)))
                step = torch.exp2(e - 3)
                unit = torch.round(unit / step) * step
            out.append((unit * need[:, None, :, None]).flatten(0, 1)[:b - lo])
        found.append((torch.cat(out), scale))
    return found[0][0], found[1][0], found[0][1], found[1][1]


def exact(case, seed):
    s = prepare(case, seed)
    ql, kl = _lens(case)
    if case["kind"] == "write":
        return _exact_write(s, ql, kl)
    if case["kind"] == "read":
        return tuple(torch.cat([_exact_values(s, x, i, b - a, b) for i, (a, b) in enumerate(zip(ql, kl))])
                     for x in ("k", "v"))
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out, q0 = [], 0
    for i, (a, b) in enumerate(zip(ql, kl)):
        K, V = _exact_values(s, "k", i, 0, b), _exact_values(s, "v", i, 0, b)
        j = torch.arange(b, device=K.device)
        heads = []
        for h in range(hkv):
            Kt, Vh = K[:, h].t().contiguous(), V[:, h].contiguous()
            rows = []
            for m in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                S = torch.matmul(s["q"][q0:q0 + a, m].double(), Kt) / math.sqrt(d)
                if s["bias"] is not None:
                    S = S + s["bias"][q0:q0 + a, m, :b].double()
                end = torch.arange(b - a, b, device=K.device)[:, None]
                if case["causal"]:
                    S = S.masked_fill(j > end, float("-inf"))
                if case["window"] > 0:
                    S = S.masked_fill(j <= end - case["window"], float("-inf"))
                rows.append(torch.matmul(torch.softmax(S, -1), Vh))
            heads += rows
        out.append(torch.stack(heads, 1))
        q0 += a
    return torch.cat(out)
