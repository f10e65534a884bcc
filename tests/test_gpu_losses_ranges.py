"""The training losses where weights, temperatures and logits are of very different sizes, against their definitions in 64 bits."""
import numpy as np
import pytest

import futhark_b200 as fb
import loss_reference as ref
from test_gpu_losses import half, within, xent_inputs

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
