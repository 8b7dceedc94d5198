"""fp64 CPU restatement of the position rotation with per-head norms, its
gradients, and rows appended to a 16-bit paged cache. No counterpart in the
reference. Test infrastructure only.
"""

import torch


def pairs(d, rot, interleaved):
    """Indexes (a, b) of the elements of each pair."""
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def turn(x, positions, inv_freq, interleaved, scale, back=False):
    """x [M, H, D] with its pairs turned by position * frequency (by the opposite
    angle with `back`) and scaled; one pair at a time."""
    x = x.double()
    y = x.clone()
    a, b = pairs(x.shape[2], 2 * len(inv_freq), interleaved)
    for i, f in enumerate(inv_freq.double().tolist()):
        t = positions.double() * f * (-1.0 if back else 1.0)
        c, s = (torch.cos(t) * scale)[:, None], (torch.sin(t) * scale)[:, None]
        y[..., a[i]] = x[..., a[i]] * c - x[..., b[i]] * s
        y[..., b[i]] = x[..., b[i]] * c + x[..., a[i]] * s
    return y


def norm(x, weight, eps):
    x = x.double()
    if weight is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()


def forward(x, positions, inv_freq, interleaved=False, scale=1.0, weight=None, eps=1e-6):
    return turn(norm(x, weight, eps), positions, inv_freq, interleaved, scale)


def backward(dy, x, positions, inv_freq, interleaved=False, scale=1.0, weight=None, eps=1e-6):
    """(dx, dweight): the transposed rotation, then the norm's derivative by its
    Jacobian, d xn_i / d x_j = r (delta_ij - xn_i xn_j / D)."""
    g = turn(dy, positions, inv_freq, interleaved, scale, back=True)
    if weight is None:
        return g, None
    x = x.double()
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    xn = x * r
    wg = g * weight.double()
    return r * (wg - xn * (xn * wg).sum(-1, keepdim=True) / x.shape[-1]), (g * xn).sum((0, 1))


def size(x, inv_freq, interleaved, scale):
    """scale (|a| + |b|) for the elements of a pair, |x| for those that pass: what
    errors of a rotation are relative to."""
    m = x.double().abs()
    out = m.clone()
    a, b = pairs(x.shape[2], 2 * len(inv_freq), interleaved)
    both = (m[..., a] + m[..., b]) * abs(scale)
    out[..., a] = both
    out[..., b] = both
    return out


def places(cu, kv_lens, table, page, pages):
    """For each row of the offsets: (sequence or -1, place in it, cache row or -1)."""
    out = []
    for row in range(cu[-1]):
        s = max(i for i in range(len(cu) - 1) if cu[i] <= row)
        if row >= cu[s + 1]:
            out.append((-1, 0, -1))
            continue
        pos = kv_lens[s] - (cu[s + 1] - row)
        at = -1
        if pos >= 0 and pos // page < table.shape[1] and 0 <= int(table[s, pos // page]) < pages:
            at = int(table[s, pos // page]) * page + pos % page
        out.append((s, pos, at))
    return out
