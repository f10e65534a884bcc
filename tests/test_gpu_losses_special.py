"""The training losses where operands are not finite, and called from several threads."""
import threading

import numpy as np
import pytest

import futhark_b200 as fb
import loss_reference as ref
from test_gpu_losses import distill_inputs, half, router_inputs, within, xent_inputs

pytestmark = pytest.mark.gpu


def same(got, want):
    return all(np.array_equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("n,v,d", [(40, 300, 64), (300, 900, 72), (150, 700, 2500)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_vocab_xent_rows_that_are_not_finite(ctx, n, v, d, bad):
    X, W, ts, dl = xent_inputs(n, v, d, 5)
    ts[:10] = 1
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    clean = (loss, lse) + fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    X[7, 3] = bad
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    assert not np.isfinite(loss[7]) and not np.isfinite(lse[7])
    dx, dw = fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    others = np.arange(n) != 7
    assert same((loss[others], lse[others], dx[others]), (clean[0][others], clean[1][others], clean[2][others]))
    assert np.isnan(half(dx)[7]).all() and np.isnan(half(dw)).all()


@pytest.mark.parametrize("n", [30, 300])
def test_vocab_xent_words_ruled_out_by_their_weights(ctx, n):
    X, W, ts, dl = xent_inputs(n, 500, 64, 6)
    X[:, 0] = 1
    W[:, 0] = 0
    out = np.arange(0, 500, 7)
    ts[np.isin(ts, out)] = 1
    ts[3] = 14
    kept = np.setdiff1d(np.arange(500), out)
    Wc = W[kept]
    W[out] = 0
    W[out, 0] = -np.inf
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    tc = np.where(ts < 0, -1, np.searchsorted(kept, np.maximum(ts, 0))).astype(np.int32)
    tc[3] = -1
    want, wantl = ref.vocab_xent(X, Wc, tc)
    err = ref.vocab_xent_error(X, Wc, tc)
    within(lse, wantl, err, "lse")
    assert np.isposinf(loss[3])
    rest = np.arange(n) != 3
    within(loss[rest], want[rest], 2 * err[rest], "loss")
    dl[3] = 0
    dx, dw = fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    wx, ww = ref.vocab_xent_grad(X, Wc, tc, dl)
    ex, ew = ref.vocab_xent_grad_error(X, Wc, tc, dl)
    within(half(dx)[rest, 1:], wx[rest, 1:], ex[rest, 1:], "dX")        # column 0 is 0 times an infinity
    within(half(dw)[kept], ww, ew, "dW")
    assert not half(dw)[out].any()


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("tau", [1.5, 0.001])
@pytest.mark.parametrize("n,v,k", [(12, 700, 6), (300, 5003, 40)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_topk_distill_rows_that_are_not_finite(ctx, t, tau, n, v, k, bad):
    S, iss, T, dl = distill_inputs(t, n, v, k, 4)
    iss[3] = iss[8] = np.arange(k)
    iss[5] = -1
    loss, lse = fb.topk_distill(ctx, t, tau, S, iss, T)
    clean = (loss, lse, fb.topk_distill_grad(ctx, t, tau, S, iss, T, lse, dl))
    S[3, v - 2] = S[5, 9] = bad                            # row 5 has no word
    T[8, 1] = bad                                          # of the teacher
    loss, lse = fb.topk_distill(ctx, t, tau, S, iss, T)
    g = fb.topk_distill_grad(ctx, t, tau, S, iss, T, lse, dl)
    rest = ~np.isin(np.arange(n), [3, 5, 8])
    assert same((loss[rest], lse[rest], g[rest]), (x[rest] for x in clean))
    g = half(g) if t == "f16" else g
    assert not np.isfinite(loss[3]) and not np.isfinite(lse[3]) and np.isnan(g[3]).all()
    assert loss[5] == 0 and not g[5].any()
    assert np.isnan(loss[8]) and np.isfinite(lse[8]) and np.isnan(g[8, :k]).all() and np.isfinite(g[8, k:]).all()


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("n,e,k", [(30, 8, 2), (3000, 100, 4), (20000, 256, 8)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_router_balance_rows_that_are_not_finite(ctx, t, n, e, k, bad):
    R, keep, iss = router_inputs(t, n, e, k, 7)
    keep[4] = True
    one = np.ones(1, np.float32)
    loss, counts, norm = fb.router_balance(ctx, t, R, keep, iss)
    clean = fb.router_balance_grad(ctx, t, R, keep, counts, norm, one)
    R[4, e - 1] = bad
    got = fb.router_balance(ctx, t, R, keep, iss)
    assert not np.isfinite(got[0]).any() and same(got[1:], (counts, norm))
    g = fb.router_balance_grad(ctx, t, R, keep, counts, norm, one)
    rest = np.arange(n) != 4
    assert np.array_equal(g[rest], clean[rest]) and np.isnan((half(g) if t == "f16" else g)[4]).all()


@pytest.mark.parametrize("own", [False, True])
def test_losses_from_several_threads(ctx, own):
    """Calls of one context take turns; contexts of their own run side by side."""
    xent = xent_inputs(200, 900, 72, 1)
    distill = distill_inputs("f16", 40, 3000, 6, 2)
    router = router_inputs("f32", 500, 20, 3, 3)

    def step(c):
        l = fb.vocab_xent_f16(c, *xent[:3])
        s = fb.topk_distill(c, "f16", 2.0, *distill[:3])
        r = fb.router_balance(c, "f32", *router)
        return (*l, *fb.vocab_xent_grad_f16(c, *xent[:3], *l, xent[3]), *s, fb.topk_distill_grad(c, "f16", 2.0, *distill[:3], s[1], distill[3]),
                *r, fb.router_balance_grad(c, "f32", *router[:2], *r[1:], np.ones(1, np.float32)))

    want = step(ctx)
    wrong = []

    def work():
        try:
            c = fb.Context() if own else ctx
            for _ in range(20):
                if not same(step(c), want):
                    wrong.append("results differ")
            if own:
                c.close()
        except Exception as e:                             # noqa: BLE001 (shown below)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
