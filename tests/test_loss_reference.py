"""The 64-bit references of the training losses: their gradients against central differences of their losses, and
the library's entry points on a context that did not come up (CPU)."""
import ctypes

import numpy as np
import pytest

import loss_reference as ref


def differences(f, x, eps=1e-5):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        a, b = x.copy(), x.copy()
        a[i] += eps
        b[i] -= eps
        g[i] = (f(a) - f(b)) / (2 * eps)
    return g


def test_vocab_xent_gradient_is_that_of_its_loss():
    r = np.random.default_rng(1)
    X, W = r.normal(size=(5, 4)), r.normal(size=(7, 4))
    ts, dl = np.array([3, -1, 0, 3, 9]), r.normal(size=5)
    dx, dw = ref.vocab_xent_grad(X, W, ts, dl)
    f = lambda x, w: float((ref.vocab_xent(x, w, ts)[0] * dl).sum())
    assert np.allclose(dx, differences(lambda x: f(x, W), X), atol=1e-8)
    assert np.allclose(dw, differences(lambda w: f(X, w), W), atol=1e-8)
    assert np.all(dx[1] == 0) and np.all(dx[4] == 0)


def test_topk_distill_gradient_is_that_of_its_loss():
    r = np.random.default_rng(2)
    S, T, dl = r.normal(size=(4, 9)) * 2, r.normal(size=(4, 5)) * 2, r.normal(size=4)
    iss = np.array([[0, 3, 8, 2, 1], [4, 4, -1, 9, 4], [-1, -1, 12, -3, -1], [5, 6, 7, 8, 0]])
    T[3, 2] = -np.inf
    for tau in (1.0, 2.5):
        g, _ = ref.topk_distill_grad(S, iss, T, tau, dl)
        assert np.allclose(g, differences(lambda s: float((ref.topk_distill(s, iss, T, tau)[0] * dl).sum()), S), atol=1e-8)
        assert np.all(g[2] == 0) and ref.topk_distill(S, iss, T, tau)[0][2] == 0


def test_router_balance_gradient_is_that_of_its_loss():
    r = np.random.default_rng(3)
    R, keep = r.normal(size=(6, 5)), np.array([True, True, False, True, True, True])
    iss = r.integers(-1, 6, size=(6, 2))
    g, _ = ref.router_balance_grad(R, keep, iss, 0.7)
    assert np.allclose(g, differences(lambda x: 0.7 * ref.router_balance(x, keep, iss)[0], R), atol=1e-8)
    assert np.all(g[2] == 0)


def test_balanced_routing_has_loss_one():
    n, e = 12, 4
    R, keep = np.zeros((n, e)), np.ones(n, bool)
    iss = (np.arange(n * 2) % e).reshape(n, 2)
    assert ref.router_balance(R, keep, iss)[0] == pytest.approx(1.0, abs=1e-12)


@pytest.mark.parametrize("name,arrays", [
    ("vocab_xent_f16", 3), ("vocab_xent_grad_f16", 6), ("router_balance_f32", 3), ("router_balance_f16", 3),
    ("router_balance_grad_f32", 5), ("router_balance_grad_f16", 5)])
def test_entry_points_refuse_a_context_that_did_not_come_up(name, arrays):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    import futhark_b200 as fb
    L = fb.load()
    cfg = L.futhark_context_config_new()
    ctx = L.futhark_context_new(cfg)
    fb._take_string(L.futhark_context_get_error(ctx))
    out = ctypes.c_void_p()
    assert getattr(L, "futhark_entry_" + name)(ctx, ctypes.byref(out), *[None] * arrays) == 1
    assert "failed to initialise" in fb._take_string(L.futhark_context_get_error(ctx))
    L.futhark_context_free(ctx)
    L.futhark_context_config_free(cfg)
