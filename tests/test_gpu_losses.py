"""The training losses and their gradients through the C ABI against their definitions in 64 bits."""
import numpy as np
import pytest

import futhark_b200 as fb
import loss_reference as ref

pytestmark = pytest.mark.gpu


def half(bits):
    return np.asarray(bits).view(np.float16).astype(np.float64)


def within(got, want, err, what):
    got = np.asarray(got, np.float64)
    bad = ~(np.abs(got - want) <= err)
    assert not bad.any(), "%s: %d of %d off, worst %.3g of what is allowed, first at %s: %r for %r" % (
        what, bad.sum(), bad.size, float((np.abs(got - want) / err)[bad].max()), np.argwhere(bad)[0].tolist(), got[bad][0], want[bad][0])


# ---- cross entropy over a vocabulary --------------------------------------------------------------------------
def xent_inputs(n, v, d, seed, scale=2.0):
    r = np.random.default_rng(seed)
    X = r.normal(size=(n, d)).astype(np.float16)
    W = (r.normal(size=(v, d)) * scale / max(1, d) ** 0.5).astype(np.float16)
    ts = r.integers(0, max(1, v), n).astype(np.int32)
    ts[r.random(n) < 0.1] = -1
    dl = ((r.random(n) + 0.5) * 1024 / max(1, n)).astype(np.float32)
    return X, W, ts, dl


def check_xent(ctx, X, W, ts, dl):
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    want, wantl = ref.vocab_xent(X, W, ts)
    err = ref.vocab_xent_error(X, W, ts)
    within(lse, wantl, err, "lse")
    within(loss, want, 2 * err, "loss")
    dx, dw = fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    wx, ww = ref.vocab_xent_grad(X, W, ts, dl)
    ex, ew = ref.vocab_xent_grad_error(X, W, ts, dl)
    within(half(dx), wx, ex, "dX")
    within(half(dw), ww, ew, "dW")
    assert np.all(dx[(ts < 0) | (ts >= len(W))] & 0x7fff == 0)


@pytest.mark.parametrize("n,v,d", [
    (1, 256, 64), (256, 256, 64), (1, 1, 1), (2, 3, 5), (1, 1000, 64), (31, 257, 8), (129, 255, 72), (128, 513, 136), (257, 1000, 100),
    (300, 700, 129), (5, 4097, 64), (1000, 300, 512), (64, 3001, 1000), (7, 20001, 64), (700, 1234, 63),
    (128, 300, 2048), (40, 600, 2056), (300, 1000, 4100), (1, 40000, 2500), (130, 2100, 2112)])
def test_vocab_xent_and_gradient(ctx, n, v, d):
    check_xent(ctx, *xent_inputs(n, v, d, n * 7 + v + d))


def test_vocab_xent_many_row_and_column_tiles(ctx):
    # more row tiles than share the columns' operand (16), and a ragged last one
    check_xent(ctx, *xent_inputs(4500, 1500, 96, 5))


def test_vocab_xent_in_pieces_of_the_vocabulary(ctx):
    # more logits than 2^29: the vocabulary is worked off in two pieces, the second one shorter
    n, v, d = 33000, 16500, 8
    X, W, ts, dl = xent_inputs(n, v, d, 6)
    rows = np.random.default_rng(7).permutation(n)[:400]          # dW sums over all rows: all but these weigh nothing
    dl[np.delete(np.arange(n), rows)] = 0
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    dx, dw = fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    X, ts, dl = X[rows], ts[rows], dl[rows]
    want, wantl = ref.vocab_xent(X, W, ts)
    err = ref.vocab_xent_error(X, W, ts)
    within(lse[rows], wantl, err, "lse")
    within(loss[rows], want, 2 * err, "loss")
    wx, ww = ref.vocab_xent_grad(X, W, ts, dl)
    ex, ew = ref.vocab_xent_grad_error(X, W, ts, dl)
    within(half(dx)[rows], wx, ex, "dX")
    within(half(dw), ww, ew, "dW")
    assert not half(np.delete(dx, rows, axis=0)).any()


@pytest.mark.parametrize("scale", [0.0, 30.0, 200.0])
def test_vocab_xent_flat_and_peaked(ctx, scale):
    # all logits equal; logits of which one is nearly all of the sum, with the target on it in every other row
    X, W, ts, dl = xent_inputs(150, 400, 64, 11, scale)
    ts[::2] = ref.vocab_xent(X, W, ts)[1].shape and (X.astype(np.float64) @ W.astype(np.float64).T).argmax(axis=1)[::2]
    check_xent(ctx, X, W, ts, dl)


def test_vocab_xent_weights_of_very_different_size(ctx):
    X, W, ts, dl = xent_inputs(200, 300, 64, 12)
    dl *= np.float32(2.0) ** np.random.default_rng(1).integers(-12, 3, 200).astype(np.float32)
    dl[::7] *= -1
    dl[5] = 0
    check_xent(ctx, X, W, ts, dl)


def test_vocab_xent_tokens_without_a_target(ctx):
    X, W, ts, dl = xent_inputs(100, 300, 64, 13)
    ts[:] = [-1, 300, -2**31, 2**31 - 1] * 25
    X[3], X[4], dl[5], dl[6] = np.nan, np.inf, np.nan, np.inf      # of tokens that do not count
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    assert np.all(loss == 0)
    dx, dw = fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    assert np.all(half(dx) == 0) and np.all(half(dw) == 0)
    # among others
    X, W, ts, dl = xent_inputs(300, 300, 64, 14)
    ts[10:20] = -1
    clean = X.copy()
    X[10:15], X[15:20] = np.nan, np.inf
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    got = fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    loss, lse = fb.vocab_xent_f16(ctx, clean, W, ts)
    want = fb.vocab_xent_grad_f16(ctx, clean, W, ts, loss, lse, dl)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_vocab_xent_nan_and_infinity_stay(ctx):
    X, W, ts, dl = xent_inputs(40, 300, 64, 15)
    ts[:] = 1
    X[7] = np.nan
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    assert np.isnan(loss[7]) and np.isnan(lse[7]) and np.isfinite(np.delete(loss, 7)).all()
    dx, dw = fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    assert np.isnan(half(dx)[7]).all() and np.isfinite(np.delete(half(dx), 7, axis=0)).all() and np.isnan(half(dw)).all()


@pytest.mark.parametrize("n,v,d", [
    (2, 70000, 8), (17, 9000, 40), (18, 9000, 40), (19, 9000, 40), (18, 1, 8), (18, 66000, 8), (36, 30000, 16), (37, 30000, 16), (129, 4000, 24),
    (576, 1020, 16), (577, 1020, 16), (576, 2060, 16), (10, 18688, 64), (10, 18689, 64), (200, 18432, 64), (200, 18433, 64), (5000, 100, 16),
    (8192, 100, 16), (8192, 300, 16), (300, 9000, 264), (100, 2000, 2050)])
def test_vocab_xent_small_calls(ctx, n, v, d):
    # small calls make the losses in the last CTA of the contraction, the rows' weights beside G and both products side by side
    check_xent(ctx, *xent_inputs(n, v, d, n + v))


@pytest.mark.parametrize("n,v,d", [(0, 5, 8), (5, 0, 8), (5, 7, 0), (0, 0, 0)])
def test_vocab_xent_of_nothing(ctx, n, v, d):
    X, W, ts, dl = xent_inputs(n, v, d, 1)
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    if v == 0:
        assert np.all(loss == 0) and np.all(lse == -np.inf)
    else:
        ok = (ts >= 0) & (ts < v)
        assert np.allclose(lse, np.log(v)) and np.allclose(loss, np.where(ok, np.log(v), 0))
    dx, dw = fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    assert dx.shape == (n, d) and dw.shape == (v, d) and not dx.any() and not dw.any()


def test_vocab_xent_operands_at_any_address(ctx):
    X, W, ts, dl = xent_inputs(70, 300, 64, 16)
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    dx, dw = fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
    bx = ctx.new("f16_1d", np.concatenate([np.zeros(3, np.uint16), X.view(np.uint16).ravel()]))
    bw = ctx.new("f16_1d", np.concatenate([np.zeros(1, np.uint16), W.view(np.uint16).ravel()]))
    x, w = ctx.new_raw("f16_2d", bx.raw + 6, 70, 64), ctx.new_raw("f16_2d", bw.raw + 2, 300, 64)
    t, g = ctx.new("i32_1d", ts), ctx.new("f32_1d", dl)
    l, s = ctx.entry_vocab_xent_f16(x, w, t)
    assert np.array_equal(l.values(), loss) and np.array_equal(s.values(), lse)
    gx, gw = ctx.entry_vocab_xent_grad_f16(x, w, t, l, s, g)
    assert np.array_equal(gx.values(), dx) and np.array_equal(gw.values(), dw)
    for a in (gx, gw, l, s, t, g, x, w, bx, bw):
        a.free()


def test_vocab_xent_is_the_same_every_time(ctx):
    X, W, ts, dl = xent_inputs(500, 5000, 256, 17)
    first = None
    for _ in range(3):
        loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
        now = (loss, lse) + fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)
        first = first or now
        assert all(np.array_equal(a, b) for a, b in zip(first, now))


# ---- distillation -----------------------------------------------------------------------------------------------
def distill_inputs(t, n, v, k, seed, scale=3.0):
    r = np.random.default_rng(seed)
    S = (r.normal(size=(n, v)) * scale).astype(np.float16 if t == "f16" else np.float32)
    iss = r.integers(0, max(1, v), (n, k)).astype(np.int32)
    iss[r.random((n, k)) < 0.1] = -1
    T = np.sort(r.normal(size=(n, k)) * 2 + 5, axis=1)[:, ::-1].astype(np.float32)
    dl = (r.random(n) + 0.5).astype(np.float32) * (64 if t == "f16" else 1)
    return S, iss, T, dl


def check_distill(ctx, t, tau, S, iss, T, dl):
    loss, lse = fb.topk_distill(ctx, t, tau, S, iss, T)
    want, wantl, mag = ref.topk_distill(S, iss, T, tau)
    big = np.abs(S.astype(np.float64)).max(axis=1, initial=0) / tau
    # exponents are products with an f32 constant: 2^-23 of their size; exp2, sums and the teacher's softmax 2^-20
    err = 2.0 ** -22 * big + 2.0 ** -20
    within(lse, wantl, err + 2.0 ** -23 * np.abs(wantl), "lse")
    within(loss, want, 2 * tau * tau * err + 2.0 ** -19 * mag, "loss")
    g = fb.topk_distill_grad(ctx, t, tau, S, iss, T, lse, dl)
    wg, mag = ref.topk_distill_grad(S, iss, T, tau, dl)
    got = half(g) if t == "f16" else g
    out = ref.H * np.abs(wg) + ref.HMIN if t == "f16" else 0
    within(got, wg, mag * (4 * err + 2.0 ** -20)[:, None] + out + 1e-37, "dS")


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("n,v,k,tau", [
    (1, 1, 1, 1.0), (3, 5, 2, 2.0), (17, 64, 8, 1.0), (9, 1001, 33, 0.5), (5, 8191, 64, 2.0), (4, 16385, 7, 4.0), (3, 50003, 128, 1.5),
    (300, 257, 20, 3.0), (2, 70000, 1024, 1.0), (6, 70, 1024, 2.0), (20, 1500, 300, 1.0), (600, 3000, 9, 1.0), (1300, 4100, 5, 2.0)])
def test_topk_distill_and_gradient(ctx, t, n, v, k, tau):
    check_distill(ctx, t, tau, *distill_inputs(t, n, v, k, n + v + k))


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_topk_distill_rows_of_every_kind(ctx, t):
    S, iss, T, dl = distill_inputs(t, 8, 4099, 6, 3)
    iss[0] = [7, 7, 7, 7, 7, 7]                        # one word six times
    iss[1] = [-1, 4099, -5, 2**31 - 1, -2**31, -1]     # none
    T[2] = -np.inf                                     # none either
    T[3, 2:] = -np.inf
    iss[4] = [0, 4098, 0, 4098, 1, 4097]               # both ends, twice
    S[5, 100:] = -np.inf                               # a student that rules words out
    iss[5] = [0, 1, 99, 5, 6, -1]
    S[6] = 0                                           # flat
    T[7] = [60000, 0, 0, -60000, 1, 2]                 # all of the weight on one word
    iss[5, 5], T[5, 5] = 4099, np.nan                  # padding that holds anything
    S[3, 50:] = np.finfo(S.dtype).min                  # words ruled out by the type's lowest value, in the student
    iss[3] = [3, 4, 5, 6, 7, 8]
    T[0, 4:] = np.finfo(np.float32).min                # and in the teacher
    S[7, iss[7, 3]] = -np.inf if iss[7, 3] not in (iss[7, 0], iss[7, 4], iss[7, 5]) else 0
    check_distill_special(ctx, t, 1.5, S, iss, T, dl)


def check_distill_special(ctx, t, tau, S, iss, T, dl):
    loss, lse = fb.topk_distill(ctx, t, tau, S, iss, T)
    want, wantl, mag = ref.topk_distill(S, iss, T, tau)
    within(lse, wantl, np.full(len(S), 1e-5), "lse")
    within(loss, want, 1e-5 * (1 + mag), "loss")
    g = fb.topk_distill_grad(ctx, t, tau, S, iss, T, lse, dl)
    wg, mag = ref.topk_distill_grad(S, iss, T, tau, dl)
    got = half(g) if t == "f16" else np.asarray(g, np.float64)
    within(got, wg, 1e-5 * mag + (ref.H * np.abs(wg) + ref.HMIN if t == "f16" else 1e-37), "dS")
    assert loss[1] == 0 and loss[2] == 0 and not got[1].any() and not got[2].any()


def test_topk_distill_of_lowest_values_only(ctx):
    """A teacher that gives every word the lowest value prefers none; a student's row of them has a finite lse (in f32, whose
    steps there are far larger than the logarithm of the number of words)."""
    S, iss, T, dl = distill_inputs("f32", 3, 300, 4, 8)
    iss[:] = [1, 2, 3, 4]
    T[:] = np.finfo(np.float32).min
    S[1] = np.finfo(np.float32).min
    loss, lse = fb.topk_distill(ctx, "f32", 1.0, S, iss, T)
    assert np.isfinite(loss[[0, 2]]).all() and np.isfinite(lse).all() and lse[1] == np.finfo(np.float32).min
    g = fb.topk_distill_grad(ctx, "f32", 1.0, S, iss, T, lse, dl)
    want, mag = ref.topk_distill_grad(S, iss, T, 1.0, dl)
    assert np.isfinite(g).all()
    within(g[[0, 2]], want[[0, 2]], 1e-5 * mag[[0, 2]] + 1e-37, "dS")


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("shift", [1, 2, 3, 5])
def test_topk_distill_rows_at_any_address(ctx, t, shift):
    S, iss, T, dl = distill_inputs(t, 5, 2111, 9, shift)
    loss, lse = fb.topk_distill(ctx, t, 2.0, S, iss, T)
    want = fb.topk_distill_grad(ctx, t, 2.0, S, iss, T, lse, dl)
    raw = fb._bits(S).ravel()
    base = ctx.new(t + "_1d", np.concatenate([np.zeros(shift, raw.dtype), raw]))
    s = ctx.new_raw(t + "_2d", base.raw + shift * raw.itemsize, 5, 2111)
    i, q, d = ctx.new("i32_2d", iss), ctx.new("f32_2d", T), ctx.new("f32_1d", dl)
    l, e = ctx.entry_topk_distill(t, 2.0, s, i, q)
    g = ctx.entry_topk_distill_grad(t, 2.0, s, i, q, e, d)
    # groups start elsewhere, so sums associate differently
    assert np.allclose(l.values(), loss, rtol=1e-5, atol=1e-5) and np.allclose(e.values(), lse, rtol=1e-6)
    if t == "f32":
        assert np.allclose(g.values(), want, rtol=1e-5, atol=1e-9)
    else:
        assert np.allclose(half(g.values()), half(want), rtol=2.0 ** -9, atol=2.0 ** -24)
    for a in (g, l, e, i, q, d, s, base):
        a.free()


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("n,v,k", [
    (16, 3000, 40), (17, 3000, 40), (16, 3000, 256), (16, 3000, 257), (1, 261888, 9), (1, 263000, 9), (3, 300000, 200), (592, 5000, 33), (600, 9000, 256)])
def test_topk_distill_of_few_rows(ctx, t, n, v, k):
    # few rows, words and runs are finished by the kernels that read the logits: both sides of each limit
    S, iss, T, dl = distill_inputs(t, n, v, k, n + v + k)
    iss[:, k // 2:] = iss[:, :k - k // 2][:, ::-1]                # every word twice, most of them far apart
    if n > 2:
        iss[1] = -1
    check_distill(ctx, t, 1.7, S, iss, T, dl)


@pytest.mark.parametrize("n,v,k", [(0, 5, 2), (4, 0, 2), (4, 5, 0)])
def test_topk_distill_of_nothing(ctx, n, v, k):
    S, iss, T, dl = distill_inputs("f32", n, v, k, 1)
    loss, lse = fb.topk_distill(ctx, "f32", 1.0, S, iss, T)
    assert np.all(loss == 0) and (v > 0 or np.all(lse == -np.inf))
    g = fb.topk_distill_grad(ctx, "f32", 1.0, S, iss, T, lse, dl)
    assert g.shape == (n, v) and not g.any()


# ---- router balance -----------------------------------------------------------------------------------------------
def router_inputs(t, n, e, k, seed):
    r = np.random.default_rng(seed)
    R = (r.normal(size=(n, e)) * 1.5 + r.normal(size=e)).astype(np.float16 if t == "f16" else np.float32)
    iss = np.argsort(-R.astype(np.float64), axis=1, kind="stable")[:, :k].astype(np.int32)
    iss[r.random((n, k)) < 0.05] = -1
    return R, r.random(n) > 0.1, np.ascontiguousarray(iss)


def check_router(ctx, t, R, keep, iss, dl):
    loss, counts, norm = fb.router_balance(ctx, t, R, keep, iss)
    wl, wc, wn, _ = ref.router_balance(R, keep, iss)
    assert np.array_equal(counts, wc)
    # rounded once from 64 bits; sums of positive terms, each within 2^-20 of its size (exponents up to 2^5)
    assert loss.shape == norm.shape == (1,)
    assert abs(float(norm[0]) - wn) <= ref.F * wn and abs(float(loss[0]) - wl) <= 2.0 ** -19 * wl
    g = fb.router_balance_grad(ctx, t, R, keep, counts, norm, np.array([dl], np.float32))
    wg, mag = ref.router_balance_grad(R, keep, iss, float(np.float32(dl)))
    got = half(g) if t == "f16" else g
    within(got, wg, 2.0 ** -19 * mag + (ref.H * np.abs(wg) + ref.HMIN if t == "f16" else 1e-37), "dR")


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("n,e,k", [
    (1, 1, 1), (1, 2, 1), (5, 3, 2), (16, 8, 2), (100, 31, 4), (333, 32, 4), (333, 33, 6), (1000, 60, 4), (777, 64, 8), (500, 100, 3),
    (2000, 256, 8), (300, 300, 16), (100, 513, 8), (64, 1024, 32), (20000, 5, 5), (9000, 160, 6), (70001, 8, 2), (30011, 100, 12), (20003, 256, 40)])
def test_router_balance_and_gradient(ctx, t, n, e, k):
    check_router(ctx, t, *router_inputs(t, n, e, k, n + e + k), 100.0 if t == "f16" else 0.01)


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_router_balance_rows_of_every_kind(ctx, t):
    R, keep, iss = router_inputs(t, 40, 20, 3, 9)
    R[keep.nonzero()[0][0]] = -np.inf                  # every expert ruled out: no probability at all
    R[5, 3:] = -np.inf
    R[6] = np.finfo(R.dtype).min                       # ruled out by the type's lowest value: all alike
    R[7, 1:] = np.finfo(R.dtype).min
    out = (~keep).nonzero()[0]
    R[out], iss[out] = np.nan, 1                       # padding does not count, whatever it holds
    iss[8] = [4, 4, 4]
    iss[9] = [-1, 20, 2**31 - 1]
    check_router(ctx, t, R, keep, iss, 3.0)


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("n,e,shift", [(3000, 64, 1), (3000, 64, 2), (700, 63, 3), (2500, 256, 4), (999, 1000, 1), (4001, 12, 2)])
def test_router_balance_rows_at_any_address(ctx, t, n, e, shift):
    R, keep, iss = router_inputs(t, n, e, min(4, e), n + e)
    loss, counts, norm = fb.router_balance(ctx, t, R, keep, iss)
    want = fb.router_balance_grad(ctx, t, R, keep, counts, norm, np.ones(1, np.float32))
    raw = fb._bits(R).ravel()
    base = ctx.new(t + "_1d", np.concatenate([np.zeros(shift, raw.dtype), raw]))
    r = ctx.new_raw(t + "_2d", base.raw + shift * raw.itemsize, n, e)
    k, i, d = ctx.new("bool_1d", keep), ctx.new("i32_2d", iss), ctx.new("f32_1d", np.ones(1, np.float32))
    l, c, m = ctx.entry_router_balance(t, r, k, i)
    g = ctx.entry_router_balance_grad(t, r, k, c, m, d)
    assert np.array_equal(c.values(), counts) and np.array_equal(m.values(), norm)
    assert np.allclose(l.values(), loss, rtol=1e-6)
    # rows are shared out differently among lanes: sums associate differently
    if t == "f32":
        assert np.allclose(g.values(), want, rtol=1e-5, atol=1e-6 * np.abs(want).max())
    else:
        assert np.allclose(half(g.values()), half(want), rtol=2.0 ** -9, atol=2.0 ** -24)
    for a in (g, l, c, m, d, i, k, r, base):
        a.free()


@pytest.mark.parametrize("keep,expert", [(False, 0), (True, -1)])
def test_router_balance_with_nothing_to_count(ctx, keep, expert):
    R, _, iss = router_inputs("f32", 30, 7, 2, 4)
    iss[:] = expert
    loss, counts, norm = fb.router_balance(ctx, "f32", R, np.full(30, keep), iss)
    assert loss[0] == 0 and norm[0] == 0 and not counts.any()
    g = fb.router_balance_grad(ctx, "f32", R, np.full(30, keep), counts, norm, np.ones(1, np.float32))
    assert not g.any()


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("e", [1, 3, 8, 60, 64, 255, 256, 1000, 1024])
def test_router_balance_partial_results_joined_either_way(ctx, t, e):
    # by the last CTA where there are few of them, by a kernel of their own where there are many
    for n in (1, 33, 1500, 9000):
        check_router(ctx, t, *router_inputs(t, n, e, min(3, e), n + e), 0.7)


@pytest.mark.parametrize("n,e,k", [(0, 4, 2), (4, 0, 2), (4, 4, 0)])
def test_router_balance_of_nothing(ctx, n, e, k):
    R, keep, iss = np.zeros((n, e), np.float32), np.ones(n, bool), np.zeros((n, k), np.int32)
    loss, counts, norm = fb.router_balance(ctx, "f32", R, keep, iss)
    assert loss[0] == 0 and norm[0] == 0 and counts.shape == (e,) and not counts.any()
    assert fb.router_balance_grad(ctx, "f32", R, keep, counts, norm, np.ones(1, np.float32)).shape == (n, e)


def test_router_balance_nearly_equal_counts(ctx):
    # every token goes everywhere but for a few drops: the gradient is what is left of a difference
    R, keep, _ = router_inputs("f32", 5000, 16, 16, 21)
    iss = np.tile(np.arange(16, dtype=np.int32), (5000, 1))
    iss[::1000, 3] = -1
    loss, counts, norm = fb.router_balance(ctx, "f32", R, keep, iss)
    g = fb.router_balance_grad(ctx, "f32", R, keep, counts, norm, np.ones(1, np.float32))
    want, _ = ref.router_balance_grad(R, keep, iss, 1.0)
    assert np.linalg.norm(g - want) <= 2.0 ** -18 * np.linalg.norm(want)


# ---- together, refusals, streams -------------------------------------------------------------------------------------
def test_a_step_with_all_three_losses(ctx):
    """A training step's sum of losses, every gradient taken: results stay on the device between the calls, blocks are reused."""
    n, v, d, e, k = 96, 1000, 64, 8, 2
    X, W, ts, dl = xent_inputs(n, v, d, 31)
    S, si, T, ddl = distill_inputs("f16", n, v, 5, 32)
    R, keep, ri = router_inputs("f32", n, e, k, 33)
    want = None
    for _ in range(3):
        arrs = [ctx.new(t, a) for t, a in (("f16_2d", X.view(np.uint16)), ("f16_2d", W.view(np.uint16)), ("i32_1d", ts), ("f32_1d", dl),
                                           ("f16_2d", S.view(np.uint16)), ("i32_2d", si), ("f32_2d", T), ("f32_1d", ddl),
                                           ("f32_2d", R), ("bool_1d", keep), ("i32_2d", ri), ("f32_1d", np.full(1, 0.01, np.float32)))]
        x, w, t, g, s, i, q, sg, r, kp, ex, rg = arrs
        out = ctx.entry_vocab_xent_f16(x, w, t)
        out += ctx.entry_topk_distill("f16", 2.0, s, i, q)
        out += ctx.entry_router_balance("f32", r, kp, ex)
        out += ctx.entry_vocab_xent_grad_f16(x, w, t, out[0], out[1], g)
        out += (ctx.entry_topk_distill_grad("f16", 2.0, s, i, q, out[3], sg), ctx.entry_router_balance_grad("f32", r, kp, out[5], out[6], rg))
        vals = [a.values_into(np.empty(a.shape, fb.ARRAY_TYPES[a.tname][0])) for a in out]
        for a in arrs + list(out):
            a.free()
        ctx.sync()
        want = want or vals
        assert all(np.array_equal(a, b) for a, b in zip(want, vals))
    within(want[0], ref.vocab_xent(X, W, ts)[0], 2 * ref.vocab_xent_error(X, W, ts), "loss")
    assert np.array_equal(want[5], ref.router_balance(R, keep, ri)[1])


def sampled(n, rows, seed):
    import torch
    return torch.randint(0, n, (rows,), generator=torch.Generator().manual_seed(seed)).cuda()


def borrowed(ctx, t):
    import torch
    name = {torch.float16: "f16", torch.float32: "f32", torch.int32: "i32", torch.bool: "bool"}[t.dtype]
    return ctx.new_raw("%s_%dd" % (name, t.dim()), t.data_ptr(), *t.shape)


def tensor(a):
    import torch
    t = torch.as_tensor(a, device="cuda")
    return t.view(torch.float16) if t.dtype == torch.uint16 else t


def test_topk_distill_beyond_32_bit_offsets(ctx):
    """More than 2^32 logits: rows at both ends and between against 64 bits."""
    import torch
    n, v, k = 33000, 131100, 6
    g = torch.Generator(device="cuda").manual_seed(3)
    S = torch.empty(n, v, dtype=torch.float16, device="cuda")
    for a in range(0, n, 1000):
        S[a:a + 1000] = torch.randn(min(1000, n - a), v, device="cuda", generator=g).mul_(3)
    iss = torch.randint(0, v, (n, k), device="cuda", generator=g).int()
    T = torch.randn(n, k, device="cuda", generator=g)
    dl = torch.full((n,), 64.0, device="cuda")
    torch.cuda.synchronize()
    ins = [borrowed(ctx, x) for x in (S, iss, T, dl)]
    loss, lse = ctx.entry_topk_distill("f16", 2.0, *ins[:3])
    grad = ctx.entry_topk_distill_grad("f16", 2.0, *ins[:3], lse, ins[3])
    ctx.sync()
    at = torch.cat([torch.tensor([0, 1, 16383, 16384, 32767, 32768, n - 2, n - 1]).cuda(), sampled(n, 30, 1)])
    Sn, In, Tn, Dn = (x[at].cpu().numpy() for x in (S, iss, T, dl))
    want, wantl, mag = ref.topk_distill(Sn, In, Tn, 2.0)
    within(tensor(lse)[at].cpu().numpy(), wantl, 1e-5, "lse")
    within(tensor(loss)[at].cpu().numpy(), want, 1e-5 * (1 + mag), "loss")
    wg, mag = ref.topk_distill_grad(Sn, In, Tn, 2.0, Dn)
    within(tensor(grad)[at].cpu().numpy(), wg, 1e-5 * mag + ref.H * np.abs(wg) + ref.HMIN, "dS")
    for a in [loss, lse, grad] + ins:
        a.free()
    ctx.clear_caches()


@pytest.mark.parametrize("n,v,d", [(9, 600000, 4096), (600000, 250, 4096)])
def test_vocab_xent_beyond_32_bit_offsets(ctx, n, v, d):
    """More than 2^31 weights, or hidden values: rows at both ends and between against 64 bits."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(4)

    def half(rows, scale):
        t = torch.empty(rows, d, dtype=torch.float16, device="cuda")
        for a in range(0, rows, 20000):
            t[a:a + 20000] = torch.randn(min(20000, rows - a), d, device="cuda", generator=gen).mul_(scale)
        return t

    X, W = half(n, 1.0), half(v, 2 / d ** 0.5)
    ts = torch.randint(0, v, (n,), device="cuda", generator=gen).int()
    ts[-1] = v - 1
    few = sampled(n, 8, 2) if n > 100 else torch.arange(n).cuda()
    few = torch.unique(torch.cat([few, torch.tensor([0, n - 1]).cuda()]))
    dl = torch.zeros(n, device="cuda")
    dl[few] = 64.0                                     # dW sums over all rows: all but these weigh nothing
    torch.cuda.synchronize()
    ins = [borrowed(ctx, x) for x in (X, W, ts, dl)]
    loss, lse = ctx.entry_vocab_xent_f16(*ins[:3])
    gx, gw = ctx.entry_vocab_xent_grad_f16(*ins[:3], loss, lse, ins[3])
    ctx.sync()
    x = X[few].double()
    z = torch.cat([x @ W[a:a + 20000].double().T for a in range(0, v, 20000)], dim=1)
    want = torch.logsumexp(z, dim=1)
    p = torch.softmax(z, dim=1)
    p[torch.arange(len(few)), ts[few].long()] -= 1
    p *= 64
    top = float(torch.cat([x.abs() @ W[a:a + 20000].abs().double().T for a in range(0, v, 20000)], dim=1).max())
    err = 2 * (d / 16 + 2) * 2.0 ** -23 * top + 2.0 ** -20 * (1 + top)
    within(tensor(lse)[few].cpu().numpy(), want.cpu().numpy(), err, "lse")
    rows = torch.unique(torch.cat([torch.tensor([0, v // 2, v - 1]).cuda(), sampled(v, 40, 5), ts[few].long()]))
    wx = sum(p[:, a:a + 20000] @ W[a:a + 20000].double() for a in range(0, v, 20000)).cpu().numpy()
    ax = sum(p[:, a:a + 20000].abs() @ W[a:a + 20000].abs().double() for a in range(0, v, 20000)).cpu().numpy()
    rel = 2 * ref.H + 4 * err + (n + v) / 16 * 2.0 ** -22        # roundings of G and of the result, the loss's error, the sums
    within(tensor(gx)[few].cpu().numpy(), wx, rel * ax + ref.HMIN, "dX")
    ww, aw = (p[:, rows].T @ x).cpu().numpy(), (p[:, rows].abs().T @ x.abs()).cpu().numpy()
    within(tensor(gw)[rows].cpu().numpy(), ww, 2 * rel * aw + 64 * ref.HMIN, "dW")
    for a in [loss, lse, gx, gw] + ins:
        a.free()
    ctx.clear_caches()


def test_losses_between_other_reductions(ctx):
    # they share the context's scratch words, each of which is 0 again when a kernel ends
    S, iss, T, dl = distill_inputs("f16", 3, 2000, 5, 1)
    X, W, ts, dls = xent_inputs(4, 900, 24, 2)
    R, keep, ie = router_inputs("f32", 50, 12, 2, 3)
    xs = np.arange(50000, dtype=np.int32)
    first = None
    for _ in range(3):
        out = [*fb.topk_distill(ctx, "f16", 2.0, S, iss, T), *fb.vocab_xent_f16(ctx, X, W, ts), *fb.router_balance(ctx, "f32", R, keep, ie)]
        assert fb.reduce_i32(ctx, xs) == xs.sum()
        dot = fb.dotprod_f32(ctx, xs.astype(np.float32), np.full(len(xs), 2.0 ** -10, np.float32))
        assert abs(dot - xs.sum() / 1024) <= len(xs) * 2.0 ** -24 * xs.sum() / 1024       # positive terms, whatever their order
        first = first or out
        for a, b in zip(first, out):
            assert np.array_equal(np.asarray(a), np.asarray(b))


def test_two_contexts_at_once(ctx):
    X, W, ts, dl = xent_inputs(600, 3000, 128, 41)
    want = fb.vocab_xent_f16(ctx, X, W, ts)
    with fb.Context() as other:
        a = [[c.new("f16_2d", X.view(np.uint16)), c.new("f16_2d", W.view(np.uint16)), c.new("i32_1d", ts)] for c in (ctx, other)]
        g = [c.new("f32_1d", dl) for c in (ctx, other)]
        outs = [(lambda o: o + c.entry_vocab_xent_grad_f16(*b, *o, d))(c.entry_vocab_xent_f16(*b)) for _ in range(4) for c, b, d in zip((ctx, other), a, g)]
        want += fb.vocab_xent_grad_f16(ctx, X, W, ts, *want, dl)
        for o in outs:
            assert all(np.array_equal(x.values(), y) for x, y in zip(o, want))
            for x in o:
                x.free()
        g[0].free(); g[1].free()
        for b in a:
            for x in b:
                x.free()


def refused(ctx, call, text):
    with pytest.raises(fb.FutharkError) as e:
        call()
    assert text in str(e.value)


def test_captured_calls_are_refused(ctx):
    import torch
    X, W, ts, dl = xent_inputs(4, 100, 16, 1)
    S, iss, T, dls = distill_inputs("f32", 3, 50, 4, 2)
    R, keep, ie = router_inputs("f16", 9, 8, 2, 3)
    x, w, t = ctx.new("f16_2d", X.view(np.uint16)), ctx.new("f16_2d", W.view(np.uint16)), ctx.new("i32_1d", ts)
    l, d = ctx.new("f32_1d", dl), ctx.new("f32_1d", dls)
    s, i, q = ctx.new("f32_2d", S), ctx.new("i32_2d", iss), ctx.new("f32_2d", T)
    r, k, j = ctx.new("f16_2d", R.view(np.uint16)), ctx.new("bool_1d", keep), ctx.new("i32_2d", ie)
    c, one = ctx.new("i32_1d", np.zeros(8, np.int32)), ctx.new("f32_1d", np.ones(1, np.float32))
    ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(torch.cuda.ExternalStream(ctx.stream)):
        graph.capture_begin(capture_error_mode="relaxed")
        try:
            for call in (lambda: ctx.entry_vocab_xent_f16(x, w, t), lambda: ctx.entry_vocab_xent_grad_f16(x, w, t, l, l, l),
                         lambda: ctx.entry_topk_distill("f32", 1.0, s, i, q), lambda: ctx.entry_topk_distill_grad("f32", 1.0, s, i, q, d, d),
                         lambda: ctx.entry_router_balance("f16", r, k, j), lambda: ctx.entry_router_balance_grad("f16", r, k, c, one, one)):
                refused(ctx, call, "cannot be captured")
        finally:
            graph.capture_end()
    for a in (x, w, t, l, d, s, i, q, r, k, j, c, one):
        a.free()
    check_xent(ctx, X, W, ts, dl)


def test_refusals(ctx):
    X, W, ts, dl = xent_inputs(4, 6, 8, 1)
    f = np.zeros(4, np.float32)
    sizes = "invalid sizes"
    refused(ctx, lambda: fb.vocab_xent_f16(ctx, X, W[:, :7], ts), sizes)
    refused(ctx, lambda: fb.vocab_xent_f16(ctx, X, W, ts[:3]), sizes)
    for at in range(3):
        args = [f, f, f]
        args[at] = f[:3]
        refused(ctx, lambda: fb.vocab_xent_grad_f16(ctx, X, W, ts, *args), sizes)
    S, iss, T, dl = distill_inputs("f32", 4, 9, 2, 1)
    refused(ctx, lambda: fb.topk_distill(ctx, "f32", 1.0, S, iss[:3], T), sizes)
    refused(ctx, lambda: fb.topk_distill(ctx, "f32", 1.0, S, iss, T[:, :1]), sizes)
    refused(ctx, lambda: fb.topk_distill_grad(ctx, "f32", 1.0, S, iss, T, f[:3], f), sizes)
    refused(ctx, lambda: fb.topk_distill_grad(ctx, "f32", 1.0, S, iss, T, f, f[:3]), sizes)
    for tau in (0.0, -1.0, float("nan"), float("inf"), 1e-30):
        refused(ctx, lambda: fb.topk_distill(ctx, "f32", tau, S, iss, T), "temperature")
        refused(ctx, lambda: fb.topk_distill_grad(ctx, "f32", tau, S, iss, T, f, f), "temperature")
    wide = np.zeros((4, 1025), np.int32)
    refused(ctx, lambda: fb.topk_distill(ctx, "f32", 1.0, S, wide, wide.astype(np.float32)), "1024")
    R, keep, ri = router_inputs("f32", 4, 3, 2, 1)
    one = np.ones(1, np.float32)
    refused(ctx, lambda: fb.router_balance(ctx, "f32", R, keep[:3], ri), sizes)
    refused(ctx, lambda: fb.router_balance(ctx, "f32", R, keep, ri[:3]), sizes)
    refused(ctx, lambda: fb.router_balance(ctx, "f32", np.zeros((4, 1025), np.float32), keep, ri), "1024")
    refused(ctx, lambda: fb.router_balance_grad(ctx, "f32", R, keep, np.zeros(2, np.int32), one, one), sizes)
    refused(ctx, lambda: fb.router_balance_grad(ctx, "f32", R, keep, np.zeros(3, np.int32), one, f), sizes)
    # and the context goes on
    assert fb.vocab_xent_f16(ctx, X, W, ts)[0].shape == (4,)


@pytest.mark.parametrize("rec,types", [(fb.LOSSES, ("f32_1d", "f32_1d")), (fb.GRADS_F16, ("f16_2d", "f16_2d")), (fb.BALANCE, ("f32_1d", "i32_1d", "f32_1d"))])
def test_records_share_their_fields(ctx, rec, types):
    import ctypes
    data = [np.arange(6, dtype=fb.ARRAY_TYPES[t][0]).reshape((2, 3) if t.endswith("2d") else 6) + i for i, t in enumerate(types)]
    arrs = [ctx.new(t, x) for t, x in zip(types, data)]
    obj = ctypes.c_void_p()
    assert getattr(ctx.lib, "futhark_new_" + rec)(ctx.ptr, ctypes.byref(obj), *[a.ptr for a in arrs]) == 0
    for a in arrs:
        a.free()
    for i, (t, want) in enumerate(zip(types, data)):
        p = ctypes.c_void_p()
        assert getattr(ctx.lib, "futhark_project_%s_%d" % (rec, i))(ctx.ptr, ctypes.byref(p), obj) == 0
        got = fb.Array(ctx, t, p.value)
        assert np.array_equal(got.values(), want)
        got.free()
    assert getattr(ctx.lib, "futhark_free_" + rec)(ctx.ptr, obj) == 0


def test_server_session_through_all_losses(tmp_path):
    """The server front-end: values of the new types from a file, every loss with its gradient, fields of the records stored."""
    from futhark_b200 import build
    from test_cli import ServerProc
    X, W, ts, dl = xent_inputs(20, 60, 16, 51)
    S, si, T, ddl = distill_inputs("f16", 20, 50, 3, 52)
    R, keep, ri = router_inputs("f32", 20, 6, 2, 53)
    values = [("x", "f16", X.view(np.uint16)), ("w", "f16", W.view(np.uint16)), ("t", "i32", ts), ("g", "f32", dl),
              ("s", "f16", S.view(np.uint16)), ("i", "i32", si), ("q", "f32", T), ("sg", "f32", ddl), ("tau", "f32", np.float32(2)),
              ("r", "f32", R), ("k", "bool", keep), ("e", "i32", ri), ("rg", "f32", np.ones(1, np.float32))]
    f = tmp_path / "in.dat"
    f.write_bytes(b"\n".join(fb.value_to_bytes(v, t, True) for _, t, v in values))
    srv = ServerProc(build.SERVER_BIN)
    srv.ok("restore %s %s" % (f, " ".join("%s %s%s" % (n, "[]" * np.ndim(v), t) for n, t, v in values)))
    srv.ok("call vocab_xent_f16 a x w t")
    for i in range(2):
        srv.ok("project a%d a %d" % (i, i))
    srv.ok("call vocab_xent_grad_f16 b x w t a0 a1 g")
    srv.ok("project b0 b 0")
    srv.ok("call topk_distill_f16 c tau s i q")
    srv.ok("project c1 c 1")
    srv.ok("call topk_distill_grad_f16 d tau s i q c1 sg")
    srv.ok("call router_balance_f32 h r k e")
    for i in range(3):
        srv.ok("project h%d h %d" % (i, i))
    srv.ok("call router_balance_grad_f32 m r k h1 h2 rg")
    assert srv.ok('fields "([]f32, []i32, []f32)"') == ["0 []f32", "1 []i32", "2 []f32"]
    o = tmp_path / "out.dat"
    srv.ok("store %s a0 b0 d h1 m" % o)
    srv.close()
    raw, got = o.read_bytes(), []
    for t, rank in (("f32", 1), ("f16", 2), ("f16", 2), ("i32", 1), ("f32", 2)):
        v, used = fb.value_from_bytes(raw, t, rank)
        got.append(v)
        raw = raw[used:]
    within(got[0], ref.vocab_xent(X, W, ts)[0], 2 * ref.vocab_xent_error(X, W, ts), "loss")
    within(half(got[1]), ref.vocab_xent_grad(X, W, ts, dl)[0], ref.vocab_xent_grad_error(X, W, ts, dl)[0], "dX")
    wg, mag = ref.topk_distill_grad(S, si, T, 2.0, ddl)
    within(half(got[2]), wg, 1e-5 * mag + ref.H * np.abs(wg) + ref.HMIN, "dS")
    assert np.array_equal(got[3], ref.router_balance(R, keep, ri)[1])
    wg, mag = ref.router_balance_grad(R, keep, ri, 1.0)
    within(got[4], wg, 2.0 ** -19 * mag + 1e-37, "dR")
