"""Operators around the attention calls: the position rotation of queries and
keys with their per-head norms (forward, and with its gradients), appending
rotated keys and values to a paged cache in 16 bits, and attention of a tree of
drafted tokens over that cache.

Rows are packed [tokens, heads, D]; the cache is [num_pages, page_size, Hkv, D],
logical token j of sequence s in page block_table[s, j // page_size]. Each case
is a dict of plain values; `run` computes it in elementary torch operations, or,
where `own` is set, with the library's kernels.
"""

import math
import random

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6

# kind: "rotary" (q and k rows, m of them), "append" (new rows of n sequences
# into their cache), "tree" (drafted tokens of n sequences over their cache).
# rot: elements of a head that the rotation takes (0: none); norm: a per-head
# norm before it; train: with the gradients; packed: q, k and v are slices of one
# projection's rows. kv lengths are drawn from lens_seed over [kv_lo, kv_hi] and
# count the new tokens, [q_lo, q_hi] per sequence (all when q_hi is 0).
# positions: "cache" (a token's place in its sequence) or "given".
_BASE = {"kind": "rotary", "dtype": "bf16", "hq": 32, "hkv": 8, "d": 128, "rot": 128, "interleaved": False,
         "norm": False, "train": False, "packed": False, "base": 10000.0, "factor": 1.0, "scale": 1.0, "m": 0,
         "pos_hi": 4096, "n": 1, "q_lo": 0, "q_hi": 0, "kv_lo": 1, "kv_hi": 1, "lens_seed": 0, "page": 64,
         "positions": "cache"}


def _case(**kw):
    c = dict(_BASE)
    c.update(kw)
    return c


def listed():
    return [
        # one step of a small decode batch, slices of the fused projection: latency counts
        _case(name="rotary_step", m=16, packed=True, pos_hi=32768),
        # the prompts of a prefill, 8 x 4096 tokens
        _case(name="rotary_prompts", m=32768, packed=True),
        # a training step of a model that norms its queries and keys, with all gradients
        _case(name="rotary_train_norm", m=16384, norm=True, train=True),
        # a part of an odd head, neighbouring elements as pairs, fp32, forward and gradients
        _case(name="rotary_train_part", dtype="fp32", m=1999, hq=16, hkv=16, d=80, rot=32, interleaved=True, train=True),
        # one token of each sequence of a server's batch: the smallest append, every step
        _case(name="append_step", kind="append", n=64, q_lo=1, q_hi=1, kv_lo=128, kv_hi=4096, lens_seed=1, page=16,
              packed=True),
        # chunks of long prompts of a model with norms, positions scaled for a longer context
        _case(name="append_chunks", kind="append", n=8, q_lo=2000, q_hi=2048, kv_lo=2048, kv_hi=8192, lens_seed=2,
              norm=True, base=500000.0, factor=4.0, scale=1.1386),
        # ragged prompts of a model without rotation, fp16, D = 64, no grouped heads
        _case(name="append_plain", kind="append", dtype="fp16", n=5, kv_lo=33, kv_hi=1900, lens_seed=3, hq=16, hkv=16,
              d=64, rot=0, page=32),
        # one user's tree over a short context: the smallest tree, where latency counts
        _case(name="tree_one", kind="tree", n=1, q_lo=16, q_hi=16, kv_lo=700, kv_hi=700, page=16),
        # a chat batch with trees of ragged sizes
        _case(name="tree_chat", kind="tree", n=16, q_lo=8, q_hi=32, kv_lo=128, kv_hi=4096, lens_seed=4),
        # a large batch with a few drafted tokens each: the stream of the cache counts
        _case(name="tree_batch", kind="tree", n=64, q_lo=2, q_hi=8, kv_lo=1024, kv_hi=16384, lens_seed=5, page=128),
        # no grouped heads, D = 64, fp16, from one token to 64
        _case(name="tree_heads", kind="tree", dtype="fp16", n=12, q_lo=1, q_hi=64, kv_lo=512, kv_hi=16384, lens_seed=6,
              hq=16, hkv=16, d=64, page=32),
        # full trees over long contexts: the largest
        _case(name="tree_long", kind="tree", n=4, q_lo=64, q_hi=64, kv_lo=32768, kv_hi=98304, lens_seed=7, hq=64, hkv=8,
              page=64),
    ]


def _loguniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "tree", "tree"])
    seed = rng.randrange(1 << 20)
    hq, hkv = rng.choice([(8, 8), (16, 16), (12, 4), (16, 2), (32, 8), (32, 4), (64, 8), (28, 4), (5, 1)])
    if kind == "tree":
        d = rng.choice([64, 128, 128])
        q_hi = _loguniform(rng, 1, 128)
        n = _loguniform(rng, 1, 64)
        # (bounded by the largest listed case's keys and scores)
        top = max(256, min(98304, (1 << 28) // (n * hkv * d), (1 << 36) // (n * q_hi * hq * d)))
        lo = _loguniform(rng, 1, top)
        hi = _loguniform(rng, lo, top)
        return _case(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp16"]), n=n, q_lo=_loguniform(rng, 1, q_hi),
                     q_hi=q_hi, kv_lo=lo, kv_hi=hi, lens_seed=seed, hq=hq, hkv=hkv, d=d,
                     page=rng.choice([16, 32, 48, 64, 128, 256]))
    d = rng.choice([64, 80, 96, 128, 128, 256])
    rot = rng.choice([d, d, d // 2, d // 4])
    c = _case(kind=kind, hq=hq, hkv=hkv, d=d, rot=rot, interleaved=rng.random() < 0.4, norm=rng.random() < 0.5,
              packed=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0, 1000000.0]), lens_seed=seed)
    if rng.random() < 0.3:                  # a longer context than the one that was trained
        c["factor"] = rng.choice([2.0, 4.0, 32.0])
        c["scale"] = round(0.1 * math.log(c["factor"]) + 1.0, 4)
    if kind == "rotary":
        c["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c["m"] = _loguniform(rng, 1, max(1, (1 << 25) // ((hq + hkv) * d)))
        c["pos_hi"] = _loguniform(rng, 1, 1 << 20)
        c["train"] = rng.random() < 0.5
        return c
    c["dtype"] = rng.choice(["bf16", "fp16"])
    c["rot"] = rng.choice([rot, rot, rot, 0])
    c["page"] = rng.choice([16, 32, 48, 64, 128, 256])
    c["positions"] = rng.choice(["cache", "given"])
    n = c["n"] = _loguniform(rng, 1, 64)
    top = max(32, min(8192, (1 << 25) // (n * (hq + 2 * hkv) * d)))
    c["kv_lo"] = _loguniform(rng, 1, top)
    c["kv_hi"] = _loguniform(rng, c["kv_lo"], top)
    if rng.random() < 0.6:                  # the last tokens alone
        c["q_hi"] = _loguniform(rng, 1, c["kv_hi"])
        c["q_lo"] = _loguniform(rng, 1, c["q_hi"])
    return c


def _lens(case):
    """(lengths of the new tokens, kv lengths)."""
    rng = random.Random(case["lens_seed"])
    kv = [rng.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["n"])]
    if case["q_hi"] == 0:
        return list(kv), kv
    return [min(x, rng.randint(case["q_lo"], case["q_hi"])) for x in kv], kv


def _cu(lens, device):
    c = [0]
    for x in lens:
        c.append(c[-1] + x)
    return torch.tensor(c, dtype=torch.int32, device=device)


def _tree(rng, n):
    """Rows of a mask: each drafted token sees itself and its ancestors."""
    rows = []
    for j in range(n):
        parent = rng.randint(max(-1, j - 8), j - 1)
        rows.append((rows[parent] if parent >= 0 else 0) | 1 << j)
    return rows


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    hq, hkv, d, rot, n = case["hq"], case["hkv"], case["d"], case["rot"], case["n"]
    s = {"case": case}

    def rand(*shape):
        return torch.randn(shape, generator=g, device=dev)

    m = case["m"]
    if case["kind"] != "rotary":
        ql, kl = _lens(case)
        m = sum(ql)
        s.update(max_q=max(ql), max_kv=max(kl), cu_q=_cu(ql, dev), cu_kv=_cu(kl, dev))
        # a cache with some of its pages free, the sequences' pages scattered in it
        page = case["page"]
        pages = [-(-x // page) for x in kl]
        total = sum(pages) + sum(pages) // 16 + 1
        for x in ("k_cache", "v_cache"):
            s[x] = rand(total, page, hkv, d).to(dt)
        perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
        table = torch.zeros((n, max(pages)), dtype=torch.int32, device=dev)
        used = 0
        for i, p in enumerate(pages):
            table[i, :p] = perm[used:used + p]
            used += p
        s["table"] = table
    s["m"] = m
    if case["kind"] == "tree":
        s["q"] = rand(m, hq, d).to(dt)
        s["attn_scale"] = 1.0 / math.sqrt(d)
        s["lse"] = torch.empty(m, hq, dtype=torch.float32, device=dev)
        rng = random.Random(seed)
        rows = [r for x in ql for r in _tree(rng, x)]
        s["mask"] = torch.tensor([[r >> j & 1 for j in range(max(ql))] for r in rows], dtype=torch.bool, device=dev)
        return s
    # a few channels are much larger than the others
    if case["packed"]:
        s["rows"] = (rand(m, hq + 2 * hkv, d) * torch.exp(0.5 * rand(1, 1, d))).to(dt)
        s["q"], s["k"], s["v"] = s["rows"][:, :hq], s["rows"][:, hq:hq + hkv], s["rows"][:, hq + hkv:]
    else:
        for x, h in (("q", hq), ("k", hkv), ("v", hkv)):
            s[x] = (rand(m, h, d) * torch.exp(0.5 * rand(1, 1, d))).to(dt)
    s["q_weight"] = s["k_weight"] = s["inv_freq"] = s["positions"] = None
    if case["norm"]:
        s["q_weight"], s["k_weight"] = (1.0 + 0.2 * rand(d)).to(dt), (1.0 + 0.2 * rand(d)).to(dt)
    if rot:
        i = torch.arange(0, rot, 2, dtype=torch.float64)
        s["inv_freq"] = (case["base"] ** (-i / rot) / case["factor"]).float().to(dev)
        if case["kind"] == "rotary" or case["positions"] == "given":
            s["positions"] = torch.randint(0, case["pos_hi"], (m,), generator=g, device=dev, dtype=torch.int32)
    if case["train"]:
        s["dq"], s["dk"] = rand(m, hq, d).to(dt), rand(m, hkv, d).to(dt)
    return s


def _angles(s, positions):
    """cos and sin [m, 1, rot / 2] times the scale; the angles of far positions
    in 64 bits."""
    a = positions.double()[:, None, None] * s["inv_freq"].double()
    return (a.cos() * s["case"]["scale"]).float(), (a.sin() * s["case"]["scale"]).float()


def _halves(x, case):
    """The two elements of each pair [..., rot / 2], and the rest of the head."""
    r = case["rot"]
    if case["interleaved"]:
        return x[..., 0:r:2], x[..., 1:r:2], x[..., r:]
    return x[..., :r // 2], x[..., r // 2:r], x[..., r:]


def _joined(a, b, rest, case):
    pairs = torch.stack((a, b), dim=-1).flatten(-2) if case["interleaved"] else torch.cat((a, b), dim=-1)
    return torch.cat((pairs, rest), dim=-1)


def _plain_rotate(x, s, cos, sin, weight):
    """The normed and rotated rows of x in 32 bits, and what the norm divides by."""
    c = s["case"]
    x = x.float()
    inv = None
    if weight is not None:
        inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        x = x * inv * weight.float()
    if cos is not None:
        a, b, rest = _halves(x, c)
        x = _joined(a * cos - b * sin, b * cos + a * sin, rest, c)
    return x, inv


def _plain_gradients(dy, x, s, cos, sin, weight, inv):
    """The gradients of x and of the norm's weight."""
    c = s["case"]
    a, b, rest = _halves(dy.float(), c)
    g = _joined(a * cos + b * sin, b * cos - a * sin, rest, c)
    if weight is None:
        return g, None
    xh = x.float() * inv
    dw = (g * xh).sum((0, 1), dtype=torch.float64)
    g = g * weight.float()
    return inv * (g - xh * (g * xh).mean(-1, keepdim=True)), dw


def _plain_rotary(s):
    c = s["case"]
    dt = s["q"].dtype
    cos, sin = _angles(s, s["positions"])
    q, qi = _plain_rotate(s["q"], s, cos, sin, s["q_weight"])
    k, ki = _plain_rotate(s["k"], s, cos, sin, s["k_weight"])
    if not c["train"]:
        return q.to(dt), k.to(dt)
    dq, dqw = _plain_gradients(s["dq"], s["q"], s, cos, sin, s["q_weight"], qi)
    dk, dkw = _plain_gradients(s["dk"], s["k"], s, cos, sin, s["k_weight"], ki)
    out = (q.to(dt), k.to(dt), dq.to(dt), dk.to(dt))
    return (*out, dqw.to(dt), dkw.to(dt)) if c["norm"] else out


def _plain_append(s):
    c = s["case"]
    cu, kv = s["cu_q"], s["cu_kv"][1:] - s["cu_kv"][:-1]
    row = torch.arange(s["m"], dtype=torch.int32, device=cu.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    place = ((kv + cu[:-1] - cu[1:])[seq] + row - cu[seq]).long()
    cos = sin = None
    if c["rot"]:
        cos, sin = _angles(s, place if s["positions"] is None else s["positions"])
    at = s["table"][seq, place // c["page"]].long() * c["page"] + place % c["page"]
    k, _ = _plain_rotate(s["k"], s, cos, sin, s["k_weight"])
    s["k_cache"].flatten(0, 1)[at] = k.to(s["k"].dtype)
    s["v_cache"].flatten(0, 1)[at] = s["v"]
    if not c["rot"] and not c["norm"]:
        return s["k_cache"], s["v_cache"]
    q, _ = _plain_rotate(s["q"], s, cos, sin, s["q_weight"])
    return q.to(s["q"].dtype), s["k_cache"], s["v_cache"]


def _plain_tree(s):
    c = s["case"]
    n, hq, hkv, d, page = c["n"], c["hq"], c["hkv"], c["d"], c["page"]
    g, L, Q = hq // hkv, s["max_kv"], s["max_q"]
    dev = s["q"].device
    ql, kl = s["cu_q"][1:] - s["cu_q"][:-1], s["cu_kv"][1:] - s["cu_kv"][:-1]
    j = torch.arange(L, device=dev)
    rows = s["table"][:, j // page].long() * page + j % page
    i = torch.arange(Q, device=dev)
    at = (s["cu_q"][:-1, None] + i).clamp(max=s["m"] - 1).long()
    q = s["q"].float()[at].view(n, Q, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * Q, d)
    k = s["k_cache"].flatten(0, 1)[rows].float().permute(0, 2, 3, 1)
    S = torch.matmul(q, k).mul_(s["attn_scale"]).view(n, hq, Q, L)
    # keys before the tree, and those of the tree that the row's mask names
    node = j - (kl - ql)[:, None]                                      # [n, L]
    see = s["mask"][at].gather(2, node.clamp(0, Q - 1)[:, None].expand(n, Q, L))
    see = ((node < 0)[:, None] | see) & (j < kl[:, None])[:, None] & (i[None] < ql[:, None])[..., None]
    S.masked_fill_(~see[:, None], float("-inf"))
    top = S.amax(-1, keepdim=True)
    top = top.masked_fill_(top == float("-inf"), 0.0)
    P = S.sub_(top).exp_()
    total = P.sum(-1, keepdim=True)
    lse = (top + total.log())[..., 0].transpose(1, 2)                  # [n, Q, hq]
    O = torch.matmul(P.view(n, hkv, g * Q, L), s["v_cache"].flatten(0, 1)[rows].float().transpose(1, 2))
    O = O.view(n, hq, Q, d).div_(total.masked_fill(total == 0, 1.0)).transpose(1, 2)
    row = torch.arange(s["m"], dtype=torch.int32, device=dev)
    seq = torch.searchsorted(s["cu_q"], row, right=True) - 1
    local = (row - s["cu_q"][seq]).long()
    return O[seq, local].to(s["q"].dtype), lse[seq, local]


def run(state):
    s = state
    c = s["case"]
    if own:
        import mtlattn

        rot = dict(interleaved=c["interleaved"], scale=c["scale"], q_weight=s.get("q_weight"),
                   k_weight=s.get("k_weight"), eps=_EPS)
        if c["kind"] == "rotary":
            if not c["train"]:
                return mtlattn.rotary(s["q"], s["k"], s["positions"], s["inv_freq"], **rot)
            leaves = [s[x].detach().requires_grad_() for x in (("q", "k", "q_weight", "k_weight") if c["norm"] else
                                                               ("q", "k"))]
            if c["norm"]:
                rot.update(q_weight=leaves[2], k_weight=leaves[3])
            out = mtlattn.rotary(leaves[0], leaves[1], s["positions"], s["inv_freq"], **rot)
            return (*(x.detach() for x in out), *torch.autograd.grad(out, leaves, (s["dq"], s["dk"])))
        if c["kind"] == "append":
            turned = bool(c["rot"]) or c["norm"]
            q = mtlattn.paged_cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["cu_q"], s["cu_kv"],
                                           s["table"], q=s["q"] if turned else None, positions=s["positions"],
                                           inv_freq=s["inv_freq"], **rot)
            return (q, s["k_cache"], s["v_cache"]) if turned else (s["k_cache"], s["v_cache"])
        out = mtlattn.paged_tree_decode(s["q"], s["k_cache"], s["v_cache"], s["cu_q"], s["cu_kv"], s["table"],
                                        s["mask"], s["max_q"], s["max_kv"], scale=s["attn_scale"], lse_out=s["lse"])
        return out, s["lse"]
    if c["kind"] == "rotary":
        return _plain_rotary(s)
    return _plain_append(s) if c["kind"] == "append" else _plain_tree(s)


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    es = 4 if case["dtype"] == "fp32" else 2
    per = (3.0 if case["rot"] else 0.0) + (4.0 if case["norm"] else 0.0)
    if case["kind"] == "rotary":
        n = case["m"] * (hq + hkv) * d
        passes = 2 + (case["train"] and (3 if case["norm"] else 2))
        return {"bytes": float(n * es * passes + 4 * case["m"]), "flops": float(n * per * (3 if case["train"] else 1))}
    ql, kl = _lens(case)
    if case["kind"] == "append":
        turned = (hq if per else 0) + 2 * hkv
        return {"bytes": float(sum(ql) * turned * d * es * 2), "flops": float(sum(ql) * (hq + hkv) * d * per)}
    # (of the tree itself, each token's own key alone is counted)
    pairs = sum(a * (b - a + 1) for a, b in zip(ql, kl))
    return {"bytes": float(2 * sum(kl) * hkv * d * es + 2 * sum(ql) * hq * d * es + 4 * sum(ql) * hq),
            "flops": 4.0 * pairs * hq * d}


def _exact_rotate(x, s, positions, weight):
    """Rows of x from the definition: the norm, then each pair as a complex number
    times exp(i position frequency)."""
    c = s["case"]
    if weight is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["d"] + _EPS) * weight
    r = c["rot"]
    if not r:
        return x
    turn = torch.polar(torch.full((), c["scale"], dtype=torch.float64, device=x.device).expand(x.shape[0], 1, r // 2),
                       torch.outer(positions.double(), s["inv_freq"].double())[:, None])
    part = x[..., :r].unflatten(-1, (r // 2, 2) if c["interleaved"] else (2, r // 2))
    if not c["interleaved"]:
        part = part.transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
    if not c["interleaved"]:
        y = y.transpose(-1, -2)
    return torch.cat((y.reshape(*x.shape[:-1], r), x[..., r:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "rotary":
        names = ["q", "k"] + (["q_weight", "k_weight"] if c["norm"] else [])
        leaf = [s[x].double().requires_grad_(c["train"]) for x in names] + [None, None]
        out = (_exact_rotate(leaf[0], s, s["positions"], leaf[2]), _exact_rotate(leaf[1], s, s["positions"], leaf[3]))
        if not c["train"]:
            return out
        grads = torch.autograd.grad(out, leaf[:len(names)], (s["dq"].double(), s["dk"].double()))
        return (*(x.detach() for x in out), *grads)
    ql, kl = _lens(c)
    page = c["page"]
    places = [torch.arange(b, device="cuda") for b in kl]
    rows = [s["table"][i].long()[p // page] * page + p % page for i, p in enumerate(places)]
    if c["kind"] == "append":
        new = torch.cat([p[b - a:] for p, a, b in zip(places, ql, kl)])
        at = torch.cat([r[b - a:] for r, a, b in zip(rows, ql, kl)])
        pos = new if s["positions"] is None else s["positions"]
        qw, kw = (s["q_weight"].double(), s["k_weight"].double()) if c["norm"] else (None, None)
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        kc.view(-1, c["hkv"], c["d"])[at] = _exact_rotate(s["k"].double(), s, pos, kw)
        vc.view(-1, c["hkv"], c["d"])[at] = s["v"].double()
        if not c["rot"] and not c["norm"]:
            return kc, vc
        return _exact_rotate(s["q"].double(), s, pos, qw), kc, vc
    g = c["hq"] // c["hkv"]
    out, lse, first = [], [], 0
    for a, b, at in zip(ql, kl, rows):
        k = s["k_cache"].flatten(0, 1)[at].double().movedim(1, 0)       # [hkv, b, d]
        v = s["v_cache"].flatten(0, 1)[at].double().movedim(1, 0)
        q = s["q"][first:first + a].double().reshape(a, c["hkv"], g, c["d"])
        hide = torch.zeros(a, b, dtype=torch.bool, device="cuda")
        hide[:, b - a:] = ~s["mask"][first:first + a, :a]
        o, l = torch.empty_like(q), torch.empty(a, c["hkv"], g, dtype=torch.float64, device="cuda")
        for h in range(c["hkv"]):
            x = torch.matmul(q[:, h].reshape(a * g, c["d"]), k[h].t().contiguous()).mul_(s["attn_scale"])
            x.view(a, g, b).masked_fill_(hide[:, None], float("-inf"))
            z = torch.logsumexp(x, -1, keepdim=True)
            o[:, h] = torch.matmul(x.sub_(z).exp_(), v[h]).view(a, g, c["d"])
            l[:, h] = z.view(a, g)
        out.append(o.view(a, c["hq"], c["d"]))
        lse.append(l.view(a, c["hq"]))
        first += a
    return torch.cat(out), torch.cat(lse)
