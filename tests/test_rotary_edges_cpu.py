"""Edges of the position rotation without a GPU: refusals before a launch, and the
frequencies of long trained contexts."""

import ctypes
import math

import pytest

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
