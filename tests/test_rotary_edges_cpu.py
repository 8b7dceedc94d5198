"""Edges of the position rotation without a GPU: refusals before a launch, and the
frequencies of long trained contexts."""

import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import mtlattn

from mtlattn_amd import capi
from tests.test_rotary_cpu import W, append, bwd, descriptor, fwd


@pytest.mark.parametrize("eps", [-1e-6, -math.inf, math.inf, math.nan])
@pytest.mark.parametrize("entry", [fwd, bwd, append])
def test_an_epsilon_that_is_no_number_from_0_on_is_refused(entry, eps):
    rc, text = entry(eps=eps, q_weight=W, k_weight=W, weight_dtype=capi.DTYPE_F32)
    assert rc == capi.ERR_INVALID and b"eps" in text
    size = capi.lib().mtlattn_rotary_bwd_workspace_size
    assert size(ctypes.byref(descriptor(eps=eps, q_weight=W, k_weight=W, weight_dtype=capi.DTYPE_F32))) == 0


def test_an_epsilon_without_norms_is_not_read():
    assert fwd(eps=math.nan, total=0)[0] == capi.OK


@pytest.mark.parametrize("dim,base,length,factor,ends,last", [
    # (pairs at which the blend begins and ends; how much slower the last pair turns)
    (64, 1e4, 65536, 4.0, (20, 33), 11 / 13), (128, 1e4, 131072, 4.0, (45, 70), 18 / 25),
    (128, 1e4, 65536, 32.0, (40, 65), 23 / 25), (128, 1e4, 4096, 16.0, (20, 46), 1.0),
    # every pair turns more than beta_fast times; pair 0 fewer than that
    (64, 100.0, 1 << 20, 8.0, (59, 84), 0.0), (64, 1e4, 100, 2.0, (0, 10), 1.0)])
def test_yarn_blends_over_the_turns_of_the_trained_length(dim, base, length, factor, ends, last):
    """Pair by pair, from the turns: pair i turns length / (2 pi base^(2 i / dim)) times, so
    that 32 and 1 turns lie at pairs dim ln(length / (2 pi turns)) / (2 ln base), of which
    the ends are rounded outward; they may lie past the last pair."""
    f, _ = mtlattn.rotary_frequencies(dim, base=base, scaling="yarn", factor=factor, original_length=length, device="cpu")
    for turns, end, up in ((32.0, ends[0], False), (1.0, ends[1], True)):
        # (the end is the first whole pair beyond: it turns more, or fewer, than that; the next one inside not)
        count = [length / (2 * math.pi * base ** (2 * i / dim)) for i in (end, end + (-1 if up else 1))]
        if up:
            assert count[0] <= turns < count[1]
        else:
            assert count[1] < turns and (count[0] >= turns or end == 0)
    for i in range(dim // 2):
        slow = min(max((i - ends[0]) / (ends[1] - ends[0]), 0.0), 1.0)
        want = base ** (-2 * i / dim) * ((1 - slow) + slow / factor)
        assert math.isclose(float(f[i]), want, rel_tol=1e-7), (i, slow)
    assert math.isclose(min(max((dim // 2 - 1 - ends[0]) / (ends[1] - ends[0]), 0.0), 1.0), last)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.complex64])
def test_positions_that_are_no_integers_are_refused(dtype):
    """Positions divided by a factor would lose their fractions: the factor belongs to the
    frequencies."""
    x, f = torch.zeros(3, 2, 8), torch.ones(4)
    pos, cu = torch.arange(3).to(dtype) / 2, torch.tensor([0, 3], dtype=torch.int32)
    for train in (False, True):
        with pytest.raises(ValueError, match="mtlattn: positions must be integers"):
            mtlattn.rotary(x.detach().requires_grad_(train), x, pos, f)
    cache = torch.zeros(2, 16, 2, 8)
    with pytest.raises(ValueError, match="mtlattn: positions must be integers"):
        mtlattn.paged_cache_append(x, x, cache, cache, cu, cu, torch.zeros(1, 2, dtype=torch.int32), positions=pos,
                                   inv_freq=f)


def test_tangents_of_forward_mode_are_refused():
    """In q, k or a weight, with and without gradients of the other mode."""
    f, pos = torch.ones(4), torch.arange(3)
    for which in range(4):
        for train in (False, True):
            x = [torch.randn(3, 2, 8), torch.randn(3, 1, 8), torch.randn(8), torch.randn(8)]
            x = [t.requires_grad_(train) for t in x]
            with forward_ad.dual_level():
                x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
                with pytest.raises(NotImplementedError, match="mtlattn: .*tangents"):
                    mtlattn.rotary(x[0], x[1], pos, f, q_weight=x[2], k_weight=x[3])
