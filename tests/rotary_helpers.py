"""Inputs and bounds of the tests of the position rotation."""

import torch

from oracle import rotary as oracle

U = 2.0 ** -24          # half a step of fp32, relative


def half_step(ref, dtype):
    """Half a step of dtype at ref: what rounding once may be off by."""
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    return torch.finfo(dtype).eps / 2 * ref.abs() + least


def forward_bound(x, ref, inv_freq, interleaved, scale, weight, eps, dtype):
    """How far a rotated row may be from ref. cos and sin: 1 U for the argument's
    rounding, 3 for the series' evaluation, 1 for the scale; the two products and
    their sum: 3. The norm: a sum of D squares in fp32, at most 16 in a row and 8
    levels of sums of them (24 U, halved by the root), the root, the division and
    the two factors (4 U). All relative to scale (|a| + |b|)."""
    xh = oracle.norm(x, weight, eps)
    ulps = 8 + (16 if weight is not None else 0)
    return half_step(ref, dtype) + 1.01 * ulps * U * oracle.size(xh, inv_freq, interleaved, scale)


def backward_bound(dy, x, ref, inv_freq, interleaved, scale, weight, eps, dtype, sums):
    """The same for (dx, dw): G bounds |g| and carries 8 U of its rotation; r and
    xn: 16 U; the product w g xn's mean, a sum of D terms like the norm's: 24 + 3
    more; two products and a difference: 4. dw: a fp32 sum of terms of 8 + 17 U each
    with at most `sums` additions one after the other."""
    g = oracle.size(dy, inv_freq, interleaved, scale)
    if weight is None:
        return half_step(ref[0], dtype) + 1.01 * 8 * U * g, None
    xd, w = x.double(), weight.double().abs()
    r = 1.0 / torch.sqrt((xd * xd).mean(-1, keepdim=True) + eps)
    xn = (xd * r).abs()
    arith = 72 * U * r * (w * g + xn * (xn * w * g).mean(-1, keepdim=True))
    dw = (25 + sums) * U * (g * xn).sum((0, 1))
    return half_step(ref[0], dtype) + 1.01 * arith, half_step(ref[1], weight.dtype) + 1.01 * dw


def check(out, ref, bound, what=""):
    out = out.detach().double().cpu()
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    bad = ~((out - ref).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst "
                           f"{float((out - ref).abs().max()):.3e}, {float(((out - ref).abs() / bound).max()):.2f} of the bound")


def frequencies(rot, base=10000.0):
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    return (base ** (-i / max(rot, 1))).float()
