"""The training losses and their gradients from their definitions, in 64 bits (numpy), with bounds of what the
library's f32 and binary16 steps may add.  A rounding to binary16 is off by at most 2^-11 of the value, or by 2^-25
where the value is subnormal; to f32 by 2^-24."""
import numpy as np

H, HMIN, F = 2.0 ** -11, 2.0 ** -25, 2.0 ** -24


def logsumexp(z):
    m = z.max(axis=1, keepdims=True) if z.shape[1] else np.full((z.shape[0], 1), -np.inf)
    m0 = np.where(np.isneginf(m), 0.0, m)
    with np.errstate(divide="ignore"):
        return (np.log(np.exp(z - m0).sum(axis=1, keepdims=True)) + m0)[:, 0]


def vocab_xent(X, W, ts):
    X, W, ts = X.astype(np.float64), W.astype(np.float64), np.asarray(ts, np.int64)
    z = X @ W.T
    lse = logsumexp(z)
    ok = (ts >= 0) & (ts < W.shape[0])
    loss = np.zeros(len(ts))
    loss[ok] = lse[ok] - z[ok, ts[ok]]
    return loss, lse


def vocab_xent_error(X, W, ts):
    """How far losses and lses may be off, per row.  A step of 16 products adds to an f32 accumulator with one
    truncation of the running sum, at most 2^-23 of sum |x w|; exp2 and the sums stay within 2^-20 of lse + 1."""
    X, W = np.abs(X.astype(np.float64)), np.abs(W.astype(np.float64))
    top = (X @ W.T).max(axis=1) if W.shape[0] else np.zeros(len(X))
    steps = X.shape[1] / 16 + 2
    return 2 * steps * 2.0 ** -23 * top + 2.0 ** -20 * (1 + top)


def vocab_xent_grad(X, W, ts, dl):
    X, W, ts, dl = X.astype(np.float64), W.astype(np.float64), np.asarray(ts, np.int64), dl.astype(np.float64)
    z = X @ W.T
    p = np.exp(z - logsumexp(z)[:, None])
    ok = (ts >= 0) & (ts < W.shape[0])
    g = p.copy()
    g[ok, ts[ok]] -= 1
    g[~ok] = 0
    g *= np.where(ok, dl, 0)[:, None]
    return g @ W, g.T @ X


def vocab_xent_grad_error(X, W, ts, dl):
    """Per element.  G rounds to binary16 relative to itself except at the target, where it is exact relative to
    w_i = dl_i q_i; dW's second operand X_i w_i 2^-(E+1) rounds once more; a q off by the loss's error moves the target's
    term by as much; f32 steps (exponents, products, sums) are within 2^-17 (1 + |lse|) of the terms."""
    dx, dw = vocab_xent_grad(X, W, ts, dl)
    err = vocab_xent_error(X, W, ts)
    Xa, Wa, ts, dl = np.abs(X.astype(np.float64)), np.abs(W.astype(np.float64)), np.asarray(ts, np.int64), np.abs(dl.astype(np.float64))
    z = X.astype(np.float64) @ W.astype(np.float64).T
    lse = logsumexp(z)
    p = np.exp(z - lse[:, None])
    ok = (ts >= 0) & (ts < W.shape[0])
    at = np.where(ok, ts, 0)
    hot = np.zeros_like(p)
    hot[np.arange(len(ts)), at] = 1
    p, hot = p * ok[:, None], hot * ok[:, None]
    pt = (p * hot).sum(axis=1)
    q = np.maximum(1 - pt, 2.0 ** -22 * np.maximum(1, np.abs(lse))) * ok
    rest = p * (1 - hot)
    f = (2.0 ** -17 * (1 + np.abs(lse)))[:, None]
    sums = (X.shape[0] + W.shape[0]) / 16 * 2.0 ** -22                    # truncations of the accumulators
    w = dl * q
    gerr = rest * (H + f + err[:, None]) * dl[:, None] + hot * (dl * (2 * err + 2.0 ** -20) + w * F)[:, None]
    gerr = gerr + (HMIN * 2.0 ** -13 * w)[:, None] * ok[:, None]
    gabs = (rest * dl[:, None] + hot * w[:, None])
    edx = gerr @ Wa + sums * (gabs @ Wa) + H * np.abs(dx) + HMIN
    fin = w[(w > 0)]
    e1 = 2.0 ** (np.floor(np.log2(fin.max())) + 1) if fin.size else 1.0
    unit = np.divide(gabs, w[:, None], out=np.zeros_like(gabs), where=w[:, None] > 0)      # |G| 2^-13
    edw = gerr.T @ Xa + (H + sums) * (gabs.T @ Xa) + e1 * HMIN * unit.sum(axis=0)[:, None] + H * np.abs(dw) + HMIN
    return edx * 1.01, edw * 1.01


def teacher(iss, T, tau, v):
    iss, T = np.asarray(iss, np.int64), T.astype(np.float64)
    ok = (iss >= 0) & (iss < v) & ~np.isneginf(T)
    t = np.where(ok, T / tau, -np.inf)
    m = t.max(axis=1, keepdims=True) if t.shape[1] else np.full((len(t), 1), -np.inf)
    m = np.where(np.isneginf(m), 0.0, m)
    e = np.where(ok, np.exp(np.where(ok, t - m, 0.0)), 0.0)
    s = e.sum(axis=1, keepdims=True)
    s1 = np.where(s == 0, 1.0, s)
    return ok, e / s1, np.where(ok, t - m - np.log(s1), 0.0)


def topk_distill(S, iss, T, tau):
    S = S.astype(np.float64)
    n, v = S.shape
    ok, q, lq = teacher(iss, T, tau, v)
    lse = logsumexp(S / tau)
    at = np.where(ok, iss, 0)
    loss = np.zeros(n)
    mag = np.zeros(n)                                      # size of the terms that make up the loss
    for i in range(n):
        j = ok[i] & (q[i] > 0)
        if j.any():
            s = S[i, at[i, j]] / tau
            loss[i] = tau * tau * (q[i, j] * (lq[i, j] - s + lse[i])).sum()
            mag[i] = tau * tau * (q[i, j] * (np.abs(lq[i, j]) + np.abs(s) + abs(lse[i]))).sum()
    return loss, lse, mag


def topk_distill_grad(S, iss, T, tau, dl):
    """The gradient and the size of its terms."""
    S = S.astype(np.float64)
    n, v = S.shape
    ok, q, _ = teacher(iss, T, tau, v)
    z = S / tau
    p = np.exp(z - logsumexp(z)[:, None])
    g = p * ok.any(axis=1)[:, None]
    a = g.copy()
    for i in range(n):
        np.add.at(g[i], iss[i][ok[i]], -q[i][ok[i]])
        np.add.at(a[i], iss[i][ok[i]], q[i][ok[i]])
    c = (dl.astype(np.float64) * tau)[:, None]
    return g * c, a * np.abs(c)


def router_balance(R, keep, iss):
    R, iss = R.astype(np.float64), np.asarray(iss, np.int64)
    n, e = R.shape
    m = R.max(axis=1, keepdims=True) if e else np.zeros((n, 1))
    m = np.where(np.isneginf(m), 0.0, m)
    x = np.exp(R - m)
    s = x.sum(axis=1, keepdims=True)
    p = x / np.where(s == 0, 1.0, s)
    flat = iss[keep].reshape(-1)
    flat = flat[(flat >= 0) & (flat < e)]
    counts = np.bincount(flat, minlength=e).astype(np.int64) if e else np.zeros(0, np.int64)
    c, kept = int(counts.sum()), int(keep.sum())
    norm = e / (c * kept) if c and kept else 0.0
    return norm * float((p[keep].sum(axis=0) * counts).sum()), counts, norm, p


def router_balance_grad(R, keep, iss, dl):
    loss, counts, norm, p = router_balance(R, keep, iss)
    c = counts - (counts.sum() // max(1, len(counts)))
    g = dl * norm * p * (c - (p * c).sum(axis=1, keepdims=True))
    a = abs(dl) * norm * p * (np.abs(c) + (p * np.abs(c)).sum(axis=1, keepdims=True))
    return g * keep[:, None], a * keep[:, None]
