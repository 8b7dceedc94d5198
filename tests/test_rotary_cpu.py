"""The position rotation without a GPU: its frequencies, the oracle's gradients
against differences, and every refusal of the C entries."""

import ctypes
import math

import pytest
import torch

import mtlattn
from mtlattn_amd import capi
from oracle import rotary as oracle
from tests.rotary_helpers import frequencies


def test_frequencies_as_trained():
    f, scale = mtlattn.rotary_frequencies(64, base=500000.0, device="cpu")
    ref = [500000.0 ** (-2 * i / 64) for i in range(32)]
    assert scale == 1.0 and f.dtype == torch.float32
    assert torch.equal(f, torch.tensor(ref, dtype=torch.float64).float())


def test_frequencies_linear():
    f, scale = mtlattn.rotary_frequencies(64, scaling="linear", factor=8.0, device="cpu")
    plain, _ = mtlattn.rotary_frequencies(64, device="cpu")
    assert scale == 1.0 and torch.allclose(f * 8, plain, rtol=1e-6, atol=0)


def test_frequencies_ntk_keeps_the_fastest_and_slows_the_slowest():
    f, _ = mtlattn.rotary_frequencies(128, scaling="ntk", factor=4.0, device="cpu")
    plain, _ = mtlattn.rotary_frequencies(128, device="cpu")
    assert f[0] == plain[0] == 1.0
    assert math.isclose(float(plain[-1] / f[-1]), 4.0, rel_tol=1e-6)
    assert bool((f <= plain).all())


def test_frequencies_yarn_blends_by_turns():
    f, scale = mtlattn.rotary_frequencies(128, scaling="yarn", factor=16.0, original_length=4096, device="cpu")
    plain, _ = mtlattn.rotary_frequencies(128, device="cpu")
    assert math.isclose(scale, 0.1 * math.log(16.0) + 1.0)
    turns = 4096 * plain.double() / (2 * math.pi)
    # (a pair's index is rounded outward: one pair more on either side of the blend)
    assert torch.equal(f[turns > 32 * 1.2], plain[turns > 32 * 1.2])
    slow = turns < 1 / 1.2
    assert torch.allclose(f[slow] * 16, plain[slow], rtol=1e-6, atol=0) and bool(slow.any())
    ratio = plain / f
    assert bool((ratio[1:] >= ratio[:-1] * (1 - 1e-6)).all())
    assert mtlattn.rotary_frequencies(128, scaling="yarn", factor=1.0, device="cpu")[1] == 1.0


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=7), dict(dim=-2), dict(dim=64, base=0.0), dict(dim=64, factor=0.0),
                                dict(dim=64, scaling="other"), dict(dim=2, scaling="ntk", factor=2.0),
                                dict(dim=64, scaling="yarn", beta_fast=1.0, beta_slow=2.0),
                                dict(dim=64, scaling="yarn", original_length=0)])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError, match="mtlattn"):
        mtlattn.rotary_frequencies(device="cpu", **kw)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed", [False, True])
def test_oracle_gradients_against_differences(interleaved, normed):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 2, 10, generator=g, dtype=torch.float64)
    dy = torch.randn(3, 2, 10, generator=g, dtype=torch.float64)
    w = torch.rand(10, generator=g, dtype=torch.float64) + 0.5 if normed else None
    args = (torch.tensor([0, 5, 1000]), frequencies(6), interleaved, 1.25)
    dx, dw = oracle.backward(dy, x, *args, weight=w)
    h = 1e-5

    def loss(x, w):
        return float((oracle.forward(x, *args, weight=w) * dy).sum())

    # (central differences: h^2 times a third derivative of order 10, and 1e-15 / h)
    for at in [(0, 0, 0), (0, 1, 9), (1, 0, 3), (2, 1, 5), (2, 0, 7)]:
        e = torch.zeros_like(x)
        e[at] = h
        assert abs((loss(x + e, w) - loss(x - e, w)) / (2 * h) - float(dx[at])) < 1e-8
    for i in range(10 if normed else 0):
        e = torch.zeros_like(w)
        e[i] = h
        assert abs((loss(x, w + e) - loss(x, w - e)) / (2 * h) - float(dw[i])) < 1e-8


# ---- refusals: addresses that are never dereferenced, calls that end before a launch ----

Q, K, V, QO, KO, POS, FREQ, W = (i << 40 for i in range(1, 9))
KC, VC, TABLE, CU = (i << 40 for i in range(16, 20))


def descriptor(**kw):
    r = capi.Rotary(dtype=capi.DTYPE_BF16, num_heads_q=8, num_heads_kv=2, head_dim=64, rotary_dim=64, interleaved=0,
                    scale=1.0, eps=1e-6, total=100, positions=POS, inv_freq=FREQ)
    for name, x in kw.items():
        setattr(r, name, x)
    return r


def fwd(q=Q, q_rs=512, k=K, k_rs=128, qo=QO, qo_rs=512, ko=KO, ko_rs=128, **kw):
    rc = capi.lib().mtlattn_rotary_fwd(ctypes.byref(descriptor(**kw)), q, q_rs, k, k_rs, qo, qo_rs, ko, ko_rs, None)
    return rc, capi.lib().mtlattn_last_error()


def bwd(q=Q, k=K, g=(1 << 45), h=(1 << 46), dq=QO, dk=KO, dqw=None, dkw=None, ws=1 << 47, size=1 << 30, rs=512, **kw):
    rc = capi.lib().mtlattn_rotary_bwd(ctypes.byref(descriptor(**kw)), q, rs, k, 128, g, 512, h, 128, dq, 512, dk, 128,
                                       dqw, dkw, ws, size, None)
    return rc, capi.lib().mtlattn_last_error()


def append(q=Q, q_rs=512, qo=QO, qo_rs=512, k=K, k_rs=128, v=V, v_rs=128, kc=KC, kc_rs=128, vc=VC, vc_rs=128, page=16,
           pages=64, table=TABLE, bts=8, n=2, cu=CU, cu_kv=CU, **kw):
    rc = capi.lib().mtlattn_cache_append(ctypes.byref(descriptor(**kw)), q, q_rs, qo, qo_rs, k, k_rs, v, v_rs, kc, kc_rs,
                                         vc, vc_rs, page, pages, table, bts, n, cu, cu_kv, None)
    return rc, capi.lib().mtlattn_last_error()


DESCRIPTORS = [dict(dtype=7), dict(total=-1), dict(total=1 << 31), dict(head_dim=0), dict(head_dim=257, rotary_dim=0),
               dict(num_heads_kv=0), dict(num_heads_q=-1), dict(num_heads_q=1 << 20), dict(rotary_dim=3),
               dict(rotary_dim=-2), dict(rotary_dim=66), dict(inv_freq=None),
               dict(q_weight=W, k_weight=W, weight_dtype=capi.DTYPE_F16), dict(q_weight=W), dict(k_weight=W)]


@pytest.mark.parametrize("kw", DESCRIPTORS)
@pytest.mark.parametrize("entry", [fwd, bwd, append])
def test_descriptors_are_refused(entry, kw):
    rc, text = entry(**kw)
    assert rc == capi.ERR_INVALID and text


@pytest.mark.parametrize("kw", [
    dict(num_heads_q=0), dict(positions=None), dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(q_rs=511),
    dict(k_rs=0), dict(qo_rs=-512), dict(ko_rs=127), dict(q_rs=1 << 31), dict(q=Q + 1), dict(ko=KO + 1),
    dict(qo=K), dict(ko=Q), dict(qo=Q + 2), dict(qo=Q, qo_rs=1024), dict(qo=KO), dict(ko=QO + 100 * 1024 - 2),
    dict(qo=Q + 64), dict(dtype=capi.DTYPE_F32, q=Q + 2)])
def test_forward_refuses(kw):
    rc, text = fwd(**kw)
    assert rc == capi.ERR_INVALID and text


@pytest.mark.parametrize("kw,rc", [
    (dict(num_heads_q=0), capi.ERR_INVALID), (dict(positions=None), capi.ERR_INVALID), (dict(g=None), capi.ERR_INVALID),
    (dict(dq=None), capi.ERR_INVALID), (dict(dqw=W), capi.ERR_INVALID), (dict(dkw=W), capi.ERR_INVALID),
    (dict(dq=1 << 45), capi.ERR_INVALID), (dict(dk=1 << 46), capi.ERR_INVALID), (dict(dq=KO), capi.ERR_INVALID),
    (dict(q_weight=W, k_weight=W, q=None), capi.ERR_INVALID), (dict(q_weight=W, k_weight=W, dq=Q), capi.ERR_INVALID),
    (dict(q_weight=W, k_weight=W, rs=511), capi.ERR_INVALID),
    (dict(q_weight=W, k_weight=W, ws=None), capi.ERR_WORKSPACE), (dict(q_weight=W, k_weight=W, size=100), capi.ERR_WORKSPACE),
    (dict(q_weight=W, k_weight=W, ws=(1 << 47) + 2), capi.ERR_WORKSPACE)])
def test_backward_refuses(kw, rc):
    got, text = bwd(**kw)
    assert got == rc and text


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(num_heads_q=0), dict(rotary_dim=0), dict(page=0), dict(pages=0), dict(pages=1 << 27), dict(bts=0),
    dict(n=0), dict(cu=None), dict(cu_kv=None), dict(table=None), dict(kc=None), dict(vc=None), dict(k=None), dict(v=None),
    dict(qo=None), dict(k_rs=127), dict(v_rs=1), dict(kc_rs=100), dict(vc_rs=0), dict(kc=KC + 1), dict(k=K + 1),
    # memory that is shared
    dict(vc=KC), dict(vc=KC + 256), dict(k=KC), dict(v=VC + 1024), dict(qo=KC), dict(qo=K), dict(qo=V), dict(q=VC),
    dict(qo=Q + 1024), dict(qo=Q, qo_rs=1024), dict(kc=Q), dict(kc_rs=256, vc_rs=256, vc=KC + 128)])
def test_append_refuses(kw):
    rc, text = append(**kw)
    assert rc == capi.ERR_INVALID and text


def test_append_is_for_16_bits():
    rc, text = append(dtype=capi.DTYPE_F32)
    assert rc == capi.ERR_UNSUPPORTED and b"half" in text


def test_empty_calls_touch_nothing():
    assert fwd(total=0, q=None, k=None, qo=None, ko=None, positions=None, inv_freq=None)[0] == capi.OK
    assert bwd(total=0, q=None, k=None, g=None, h=None, dq=None, dk=None, ws=None, size=0)[0] == capi.OK
    assert append(total=0, q=None, qo=None, k=None, v=None, kc=None, vc=None, table=None)[0] == capi.OK


def test_workspace_is_for_norms():
    size = capi.lib().mtlattn_rotary_bwd_workspace_size
    assert size(ctypes.byref(descriptor())) == 0
    assert size(ctypes.byref(descriptor(head_dim=0))) == 0
    n = size(ctypes.byref(descriptor(q_weight=W, k_weight=W, weight_dtype=capi.DTYPE_F32, total=1 << 20)))
    assert 0 < n <= 1 << 24


def test_python_refuses():
    q, k = torch.zeros(3, 2, 8), torch.zeros(3, 1, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        mtlattn.rotary(q, k, torch.arange(3), torch.ones(4))
    with pytest.raises(NotImplementedError, match="inv_freq"):
        mtlattn.rotary(q, k, torch.arange(3), torch.ones(4, requires_grad=True))
    with pytest.raises(ValueError, match="together"):
        mtlattn.rotary(q.requires_grad_(), k, torch.arange(3), torch.ones(4), q_weight=torch.ones(8))
    with pytest.raises(RuntimeError, match="GPU"):
        mtlattn.paged_cache_append(k, k, torch.zeros(2, 16, 1, 8), torch.zeros(2, 16, 1, 8), torch.tensor([0, 3]),
                                   torch.tensor([0, 3]), torch.zeros(1, 2, dtype=torch.int32))
