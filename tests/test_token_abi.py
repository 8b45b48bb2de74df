"""Argument checks of the operators over tokens and choices, without a GPU: every refusal comes before any device work."""
import ctypes

import pytest
import torch

FAKE = ctypes.c_void_p(0x1000)      # never dereferenced: every call below fails validation first
BIG = 1 << 32
OK, TOO_LARGE, BAD, WORKSPACE = 0, 2, 3, 4


@pytest.fixture(scope="module")
def lib():
    from snntc_amd import _lib
    return _lib.load()


def test_embed_argument_errors(lib):
    f = lambda tok=FAKE, tb=8, tab=FAKE, ty=0, z=FAKE, n=4, v=5, d=6: lib.snntc_embed_forward(tok, tb, tab, ty, z, n, v, d, 1.0, 0, None)
    assert f(n=-1) == f(v=-1) == f(d=-1) == BAD
    assert f(tb=2) == f(ty=3) == f(ty=-1) == BAD
    assert f(tok=None) == f(tab=None) == f(z=None) == BAD
    assert f(v=0) == BAD and b"empty table" in lib.snntc_last_error()
    assert f(n=BIG) == f(v=BIG) == f(d=BIG) == TOO_LARGE
    assert f(n=0) == f(d=0) == f(n=0, v=0) == f(n=0, tok=None, tab=None, z=None) == OK
    g = lambda gr=FAKE, tok=FAKE, tab=FAKE, out=FAKE, n=400, v=5, d=6, enc=0, ws=FAKE, have=1 << 20: lib.snntc_embed_backward(
        gr, tok, 8, tab, 0, out, n, v, d, 1.0, enc, ws, have, None)
    assert g(gr=None) == g(tok=None) == g(out=None) == g(tab=None, enc=1) == g(n=-1) == g(v=0) == BAD
    assert g(n=BIG) == TOO_LARGE
    assert g(ws=None) == g(ws=ctypes.c_void_p(0x1010)) == g(have=8) == WORKSPACE
    assert g(n=0, v=0) == g(d=0) == OK
    need = ctypes.c_size_t()
    assert lib.snntc_embed_backward_workspace_bytes(1000, 50, 8, ctypes.byref(need)) == OK and need.value >= 8000
    assert lib.snntc_embed_backward_workspace_bytes(1000, 50, 8, None) == BAD
    assert lib.snntc_embed_backward_workspace_bytes(-1, 50, 8, ctypes.byref(need)) == BAD


def test_gated_argument_errors(lib):
    need = ctypes.c_size_t()
    assert lib.snntc_gated_scan_workspace_bytes(2, 1 << 16, 64, ctypes.byref(need)) == OK
    f = lambda x=FAKE, g=FAKE, ty=0, y=FAKE, fin=FAKE, b=2, t=3, d=4, ws=FAKE, have=1 << 30: lib.snntc_gated_scan_forward(
        x, g, ty, None, None, y, fin, b, t, d, ws, have, None)
    assert f(x=None) == f(g=None) == f(y=None) == f(ty=7) == f(b=-1) == f(t=-1) == f(d=-1) == BAD
    assert f(b=BIG) == f(t=BIG) == f(d=BIG) == TOO_LARGE
    assert f(b=0) == f(d=0) == f(t=0, fin=None) == OK
    g = lambda x=FAKE, y=FAKE, dx=FAKE, dg=FAKE, ds=FAKE, t=3: lib.snntc_gated_scan_backward(
        FAKE, FAKE, x, FAKE, 0, y, None, None, dx, dg, ds, 2, t, 4, FAKE, 1 << 30, None)
    assert g(x=None) == g(y=None) == BAD
    assert g(dx=None, dg=None, ds=None) == g(ds=None, t=0) == OK
    s = lambda x=FAKE, ga=FAKE, ty=0, out=FAKE, n=4: lib.snntc_gated_step(x, ga, ty, None, out, n, None)
    assert s(x=None) == s(ga=None) == s(ty=3) == s(out=None) == s(n=-1) == BAD
    assert s(n=0) == OK and s(n=BIG) == TOO_LARGE


def test_choice_argument_errors(lib):
    need = ctypes.c_size_t()
    assert lib.snntc_choice_workspace_bytes(100, 10, ctypes.byref(need)) == OK and need.value == 0
    assert lib.snntc_choice_workspace_bytes(100, 200000, ctypes.byref(need)) == OK and need.value >= 100 * 25 * 8
    assert lib.snntc_choice_workspace_bytes(100, 10, None) == BAD
    assert lib.snntc_preference_workspace_bytes(10, 5, 10, ctypes.byref(need)) == OK and need.value >= 1600
    assert lib.snntc_preference_workspace_bytes(10, 5, 10, None) == lib.snntc_preference_workspace_bytes(-1, 5, 10, ctypes.byref(need)) == BAD
    f = lambda t=FAKE, ty=0, k=FAKE, lp=FAKE, r=4, j=70000, ws=FAKE, have=1 << 20: lib.snntc_time_logp(
        t, ty, k, None, lp, None, r, j, ws, have, None)
    assert f(t=None) == f(k=None) == f(lp=None) == f(ty=9) == f(r=-1) == f(j=-1) == f(j=0) == BAD
    assert f(r=1 << 24) == f(j=BIG) == TOO_LARGE
    assert f(ws=None) == f(have=16) == WORKSPACE
    assert f(r=0) == f(r=0, j=0) == OK
    p = lambda old=FAKE, adv=FAKE, lo=0.2, hi=0.2, kl=0.0, loss=FAKE, r=4, ws=FAKE: lib.snntc_policy_loss(
        FAKE, 0, FAKE, old, adv, None, None, lo, hi, kl, loss, None, None, None, None, r, 70000, ws, 1 << 20, None)
    assert p(old=None) == p(adv=None) == p(loss=None) == BAD
    nan, inf = float("nan"), float("inf")
    assert p(lo=-0.1) == p(lo=1.5) == p(hi=-0.1) == p(lo=nan) == p(hi=nan) == p(kl=nan) == p(kl=inf) == BAD
    assert p(ws=None) == WORKSPACE and p(r=0) == OK
    q = lambda ref=FAKE, beta=0.1, sm=0.0, pl=FAKE, sl=FAKE, P=2, T=3, J=5, t=FAKE, ws=FAKE: lib.snntc_preference_loss(
        t, 0, FAKE, ref, None, beta, sm, pl, sl, None, None, None, P, T, J, ws, 1 << 20, None)
    assert q(ref=None) == q(pl=None) == q(sl=None) == q(t=None) == q(P=-1) == q(T=-1) == q(J=0) == BAD
    assert q(beta=inf) == q(beta=nan) == q(sm=-0.1) == q(sm=1.1) == q(sm=nan) == BAD
    assert q(P=1 << 20, T=1 << 10) == q(P=BIG, T=0) == q(P=1 << 24, T=0) == TOO_LARGE
    assert q(ws=None) == WORKSPACE and q(P=0) == OK
    b = lambda t=FAKE, s=FAKE, c=FAKE, d=FAKE: lib.snntc_time_logp_backward(t, 0, FAKE, s, c, None, d, 4, 5, None)
    odd = ctypes.c_void_p(0x1004)
    assert b(s=odd) == BAD and b"aligned" in lib.snntc_last_error()
    assert lib.snntc_time_logp(FAKE, 0, FAKE, None, FAKE, odd, 4, 5, None, 0, None) == BAD
    assert b(t=None) == b(s=None) == b(c=None) == b(d=None) == BAD
    assert lib.snntc_loss_total(FAKE, None, None, 3, None) == lib.snntc_loss_total(None, None, FAKE, 3, None) == BAD
    assert lib.snntc_loss_total(FAKE, None, FAKE, -1, None) == BAD


def test_host_tensors_and_wrong_types_are_refused():
    import snntc_amd as snn
    x, k = torch.rand(2, 3, 4), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(snn.SnntcLibraryError, match="no CPU fallback"):
        snn.embed_tokens(k, torch.rand(5, 4))
    with pytest.raises(snn.SnntcLibraryError, match="no CPU fallback"):
        snn.gated_scan(x, x)
    with pytest.raises(snn.SnntcLibraryError, match="no CPU fallback"):
        snn.gated_step(x, x)
    with pytest.raises(snn.SnntcLibraryError, match="no CPU fallback"):
        snn.time_logp(x, k)
    with pytest.raises(snn.SnntcLibraryError, match="no CPU fallback"):
        snn.policy_loss(x, k, x[..., 0], x[..., 0])
    with pytest.raises(snn.SnntcLibraryError, match="no CPU fallback"):
        snn.preference_loss(x, k, x[:, 0, 0])
    with pytest.raises(TypeError, match="tokens must be a torch.Tensor"):
        snn.embed_tokens([1, 2], torch.rand(5, 4))
    with pytest.raises(ValueError, match="weight shape"):
        snn.SNN_embedding(4, 3, weight=[[1.0, 2.0]])
    with pytest.raises(ValueError, match="weight shape"):
        snn.SNN_recurrence(4, weight=[[1.0, 2.0]])


def test_layers_over_tokens_in_a_spec():
    import numpy as np
    import snntc_amd as snn
    from snntc_amd import networks
    spec = [("embed", 20, 8), ("recur", 8), ("steps",), ("dense", 8, 5)]
    assert networks.layer_weight_shapes(spec) == [(20, 8), (8, 8), (8, 5)]
    net = networks.build(spec, rng=np.random.default_rng(0))
    assert [type(m) for m in net] == [snn.SNN_embedding, snn.SNN_recurrence, snn.SNN_steps, snn.SNN_dense]
    assert [tuple(w.shape) for w in net.weights()] == [(20, 8), (9, 8), (9, 5)]
    assert net[2](torch.zeros(2, 3, 8)).shape == (6, 8)
