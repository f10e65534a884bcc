"""The training losses where weights, temperatures and logits are of very different sizes, against their definitions in 64 bits."""
import numpy as np
import pytest

import futhark_b200 as fb
import loss_reference as ref
from test_gpu_losses import distill_inputs, half, within, xent_inputs

pytestmark = pytest.mark.gpu


# one CTA per tile, pairs; the rows' weights beside G or by a kernel; X small enough for whoever needs its largest product, or not
@pytest.mark.parametrize("n,v,d", [(40, 300, 64), (300, 500, 64), (300, 500, 400), (5000, 200, 64), (90, 700, 1001), (2, 100, 2500)])
@pytest.mark.parametrize("ratio", [1e-4, 1e-5, 1e-6, 1e-7])
def test_vocab_xent_word_of_a_token_of_small_weight(ctx, n, v, d, ratio):
    """A word that no other token gives any probability to: its row of dW is what the one token adds.

    G is -2^13 exactly there.  X_ij w_i is rounded to binary16 with the largest product of all below 2^15, so by 2^-11 of
    itself or by 2^(E-39); the result by 2^-11 or 2^-25.  w is off by 2 err + 2^-20, exponents and sums by less than 2^-14.
    The other tokens' probabilities of the word are e^-64 of a usual one: less than 2^-80 of anything here."""
    X, W, ts, dl = xent_inputs(n, v, d, n + d)
    light, word = n // 3, v // 2
    ts[ts == word] = 0
    ts[light] = word
    X[:, 0], W[:, 0] = -8, 0
    X[light, 0] = 0
    W[word], W[word, 0] = 0, 8
    dl[:] = 1024
    dl[light] = np.float32(1024 * ratio)
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    dw = half(fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)[1])
    want = ref.vocab_xent_grad(X, W, ts, dl)[1][word]
    err = ref.vocab_xent_error(X[light:light + 1], W, ts[light:light + 1])[0]
    q = -np.expm1(-ref.vocab_xent(X, W, ts)[0])
    top = (np.abs(X.astype(np.float64)) * (np.where(ts < 0, 0, q * dl))[:, None]).max()
    assert q[light] > 0.5 and 0 <= np.log2(top) < 15
    rel = 2 * ref.H + 2 * (2 * err + 2.0 ** -20) + 2.0 ** -14
    within(dw[word], want, rel * np.abs(want) + ref.HMIN + 2.0 ** (np.floor(np.log2(top)) - 39), "dW of the word")


@pytest.mark.parametrize("scale", [2.0 ** -24, 1.0, 2.0 ** 100])
def test_vocab_xent_operands_of_any_size(ctx, scale):
    """Rows of zeros beside weights of any size, hidden states that are nearly all subnormal, weights whose products leave f32's range."""
    X, W, ts, dl = xent_inputs(60, 200, 72, 3)
    dl *= np.float32(scale)
    X[::3] = 0
    dl[::3] = 3e38
    X[1::3] = np.float16(2.0 ** -24) * np.sign(X[1::3])
    W = (W * np.float16(0.01)).astype(np.float16)
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    dw = half(fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)[1])
    with np.errstate(over="ignore"):
        want = ref.vocab_xent_grad(X, W, ts, dl)[1]
        ew = ref.vocab_xent_grad_error(X, W, ts, np.where(np.arange(60) % 3 == 0, 0, dl).astype(np.float32))[1]
    big = np.abs(want) > 65504                             # rounds to an infinity: both do, or the value is near the border
    within(dw[~big], want[~big], ew[~big], "dW")
    assert np.isinf(dw[np.abs(want) > 65600]).all() and not np.isnan(dw).any()


# either side of the temperature below which the gradient takes statistics of its own, and both ends of what is accepted
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("tau", [2.0 ** -60, 1e-9, 4e-5, 2.0 ** -6 * 0.999, 2.0 ** -6, 0.05, 100.0, 2.0 ** 60])
@pytest.mark.parametrize("n,v,k", [(3, 300, 5), (17, 5001, 40), (300, 2000, 9), (2, 300000, 300)])
def test_topk_distill_at_any_temperature(ctx, t, tau, n, v, k):
    """Exponents of 2 below 2^-150 of the row's sum do not count, so one that does is (S - max) log2(e) / tau with three
    roundings, at most 150 * 3 * 2^-24 ln 2 < 2^-15 of what it stands for; above 2^-6 they come from an lse rounded to f32 as well.
    The teacher's log q is a difference times 1 / tau, three roundings too: q is off by 3 * 2^-24 |log q| of itself beside the usual
    2^-19 of a term."""
    S, iss, T, dl = distill_inputs(t, n, v, k, n + v)
    S[0, : v // 2] = np.finfo(S.dtype).min                 # a mask
    S[-1, 7] = S[-1, 11] = S[-1].max()                     # two words alike
    tau = float(np.float32(tau))
    dl *= np.float32(min(1, 1 / tau))
    loss, lse = fb.topk_distill(ctx, t, tau, S, iss, T)
    want, wantl, _ = ref.topk_distill(S, iss, T, tau)
    S64 = S.astype(np.float64)
    top = np.abs(S64.max(axis=1)) / tau
    within(lse, wantl, 2.0 ** -22 * (top + np.abs(wantl)) + 2.0 ** -20, "lse")
    ok, q, lq = ref.teacher(iss, T, tau, v)
    size = np.abs(lq) + np.abs(np.take_along_axis(S64, np.where(ok, iss, 0).astype(np.int64), 1)) / tau + np.abs(wantl)[:, None]
    err = tau * tau * ((q * size * (2.0 ** -19 + 3 * 2.0 ** -24 * np.abs(lq))).sum(axis=1) + 2.0 ** -21 * top + 2.0 ** -19)
    over = np.abs(want) > float(np.finfo(np.float32).max)      # a masked word of the teacher's: no f32 number
    assert np.isposinf(loss[over]).all()
    within(loss[~over], want[~over], err[~over], "loss")
    g = fb.topk_distill_grad(ctx, t, tau, S, iss, T, lse, dl)
    # differences before quotients: even 64 bits lose the logarithm of a sum beside 2^62
    p = np.exp((S64 - S64.max(axis=1, keepdims=True)) / tau)
    p = p / p.sum(axis=1, keepdims=True) * ok.any(axis=1)[:, None]
    wg, mag = p.copy(), p
    for i in range(n):
        np.add.at(wg[i], iss[i][ok[i]], -q[i][ok[i]])
        np.add.at(mag[i], iss[i][ok[i]], q[i][ok[i]])
    c = dl.astype(np.float64)[:, None] * tau
    wg, mag = wg * c, mag * c
    err = 2.0 ** -15 + (0 if tau < 2.0 ** -6 else 2.0 ** -22 * (top + np.abs(wantl)))
    out = ref.H * np.abs(wg) + ref.HMIN if t == "f16" else 1e-37
    within(half(g) if t == "f16" else g, wg, mag * (np.zeros(n) + err)[:, None] + out, "dS")


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("n,v,k,shift", [(5, 2111, 9, 1), (5, 2111, 9, 3), (400, 333, 3, 5), (3, 64, 0, 0), (0, 70, 2, 0), (4, 0, 2, 0), (2, 3, 1024, 1)])
def test_topk_distill_at_small_temperatures_of_any_shape(ctx, t, n, v, k, shift):
    S, iss, T, dl = distill_inputs(t, n, v, k, 9)
    raw = fb._bits(S).ravel()
    base = ctx.new(t + "_1d", np.concatenate([np.zeros(shift, raw.dtype), raw]))
    arrs = [ctx.new_raw(t + "_2d", base.raw + shift * raw.itemsize, n, v), ctx.new("i32_2d", iss), ctx.new("f32_2d", T), ctx.new("f32_1d", dl)]
    tau = float(np.float32(1e-3))
    loss, lse = ctx.entry_topk_distill(t, tau, *arrs[:3])
    g = ctx.entry_topk_distill_grad(t, tau, *arrs[:3], lse, arrs[3])
    want, mag = ref.topk_distill_grad(S, iss, T, tau, dl) if n and v else (np.zeros((n, v)), np.zeros((n, v)))
    out = ref.H * np.abs(want) + ref.HMIN if t == "f16" else 1e-37
    got = half(g.values()) if t == "f16" else g.values()
    assert got.shape == (n, v)
    within(got, want, 2.0 ** -15 * mag + out, "dS")        # exponents as above
    for a in [loss, lse, g, base] + arrs:
        a.free()


@pytest.mark.parametrize("n,d", [(20, 64), (300, 400)])
@pytest.mark.parametrize("weight", [0.0, -0.0, 1e-44, -1e30])
def test_vocab_xent_weights_all_alike(ctx, n, d, weight):
    X, W, ts, dl = xent_inputs(n, 200, d, 4)
    dl[:] = weight
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    dx, dw = (half(x) for x in fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl))
    if abs(weight) < 1:
        assert not dx.any() and not dw.any()               # the second one's gradients are below 2^-25
    else:
        ok = (ts >= 0) & (ts < 200)
        assert np.isinf(dx[ok]).mean() > 0.99 and not np.isnan(dx).any() and np.isinf(dw).mean() > 0.99 and not np.isnan(dw).any()


def test_losses_in_a_context_with_unified_memory(ctx):
    X, W, ts, dl = xent_inputs(50, 400, 72, 2)
    S, iss, T, ddl = distill_inputs("f16", 9, 900, 5, 3)
    want = None
    for unified in (False, True):
        with fb.Context(unified_memory=unified, profiling=unified) as c:
            l = fb.vocab_xent_f16(c, X, W, ts)
            s = fb.topk_distill(c, "f16", 2.0, S, iss, T)
            got = (*l, *fb.vocab_xent_grad_f16(c, X, W, ts, *l, dl), *s, fb.topk_distill_grad(c, "f16", 2.0, S, iss, T, s[1], ddl))
            want = want or got
            assert all(np.array_equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("n,v,d", [(1, 300, 8), (40, 700, 64), (300, 500, 64), (140, 400, 2500)])
@pytest.mark.parametrize("size", [1.0, 300.0, 20000.0, 60000.0])
def test_vocab_xent_logits_of_any_size(ctx, n, v, d, size):
    """Logits up to 60000^2 d: sums of f32 products, so right to the accumulators' truncations of their terms."""
    X, W, ts, _ = xent_inputs(n, v, d, 6)
    X = (np.clip(X.astype(np.float64), -1, 1) * size).astype(np.float16)
    W = (np.clip(W.astype(np.float64), -1, 1) * size).astype(np.float16)
    ts[:1] = (X.astype(np.float64) @ W.astype(np.float64).T).argmax(axis=1)[:1]
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    want, wantl = ref.vocab_xent(X, W, ts)
    err = ref.vocab_xent_error(X, W, ts)
    within(lse, wantl, err, "lse")
    within(loss, want, 2 * err, "loss")


@pytest.mark.parametrize("n", [1, 200])
def test_vocab_xent_gradient_of_certain_tokens_with_large_logits(ctx, n):
    """The target's logit is 1.8e7 above all others: q is 0, and the target's term at most dl 2^-22 W_t with a rounding or two."""
    X = np.full((n, 8), 3000, np.float16)
    W = np.zeros((300, 8), np.float16)
    W[:, 0], W[7, 0] = -3000, 3000
    ts, dl = np.full(n, 7, np.int32), np.full(n, 2, np.float32)
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    assert np.all(loss == 0) and np.all(lse == 9e6)
    dx, dw = (half(x) for x in fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl))
    assert np.abs(dx).max() <= 6000 * 2.0 ** -21 and np.abs(dw).max() <= 6000 * 2.0 ** -21 * n


@pytest.mark.parametrize("n,v,d", [(50, 500, 64), (300, 2000, 64), (100, 500, 2600)])
def test_vocab_xent_gradient_of_nearly_certain_tokens(ctx, n, v, d):
    """q = 1 - exp(-loss) of tokens whose target's logit is 10 to 400 and all others' are smaller, at any size of lse.

    The target's own 1 is in a sum that up to 40 more numbers are added to, each with a rounding of 2^-24: 10 with the other columns of its 32, 10 with
    the next 32, 3 with the row's other shares, 8 + 5 with other tiles', 4 to put partial sums together.  What is added is q in all, and off by
    what a logit is off by.  q is at least 2^-22.  The gradient has the other words' terms too, with their roundings: 2^-9 q."""
    r = np.random.default_rng(n)
    W = (r.normal(size=(v, d)) / d ** 0.5).astype(np.float16)
    ts = r.integers(0, v, n).astype(np.int32)
    to = np.exp(r.uniform(np.log(10), np.log(400), n))
    X = (W[ts].astype(np.float64) * to[:, None]).astype(np.float16)
    dl = np.full(n, 4096, np.float32)
    loss, lse = fb.vocab_xent_f16(ctx, X, W, ts)
    want = ref.vocab_xent(X, W, ts)[0]
    q, few = -np.expm1(-want), 40 * 2.0 ** -24
    off = few + 2 * ref.vocab_xent_error(X, W, ts) * q + 2.0 ** -22 * want
    within(loss, want, off, "loss")
    dx = half(fb.vocab_xent_grad_f16(ctx, X, W, ts, loss, lse, dl)[0])
    wx = ref.vocab_xent_grad(X, W, ts, dl)[0]
    size = np.abs(W.astype(np.float64)).max()
    err = 4096 * (off + 2.0 ** -22 + 2.0 ** -9 * q)[:, None] * 2 * size
    within(dx, wx, err + ref.H * np.abs(wx) + ref.HMIN, "dX")
