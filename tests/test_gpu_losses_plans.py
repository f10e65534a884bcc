"""The gradient of the vocabulary's cross entropy where the vocabulary is worked off in pieces and each piece's sum in parts."""
import json

import pytest

import futhark_b200 as fb
import loss_reference as ref
from test_gpu_losses import borrowed, tensor, within

pytestmark = pytest.mark.gpu


# several parts in several pieces, the last one shorter; rows that are copied; more than two pieces; many parts
@pytest.mark.parametrize("n,v,d,pieces,parts", [
    (5000, 131072, 32, 2, 7), (5000, 130000, 36, 2, 7), (20000, 100000, 40, 4, 3), (2000, 900000, 65, 4, 8), (700, 800000, 16, 2, 49)])
def test_pieces_of_the_vocabulary_in_parts(n, v, d, pieces, parts):
    """All of dX and dW.  W's and X's means are away from 0, so that a part of a sum that is missing, doubled or of another piece is
    far above what roundings may add: 2^-11 for G and the scaled X each, the exponents', the accumulators' of at most
    v / (pieces parts) or n products, and the result's 2^-11 or 2^-25."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(n + d)
    dev = dict(device="cuda", generator=g)
    X = torch.randn(n, d, **dev).add_(0.5).half()
    W = torch.randn(v, d, **dev).mul_(2 / d ** 0.5).add_(0.5).half()
    ts = torch.randint(-v // 20, v, (n,), **dev).int()
    dl = torch.rand(n, **dev).add_(0.5).mul_(16)
    torch.cuda.synchronize()
    with fb.Context(profiling=True) as ctx:
        ins = [borrowed(ctx, x) for x in (X, W, ts, dl)]
        loss, lse = ctx.entry_vocab_xent_f16(*ins[:3])
        gx, gw = ctx.entry_vocab_xent_grad_f16(*ins[:3], loss, lse, ins[3])
        ctx.sync()
        plan = [e["details"] for e in json.loads(ctx.report())["events"] if e["name"].startswith("vocab_xent_grad_f16")]
        assert [(p["pieces"], p["parts"]) for p in plan] == [(pieces, parts)]
        w = W.double()
        gw_want, gw_size = torch.zeros(v, d, dtype=torch.float64, device="cuda"), torch.zeros(v, d, dtype=torch.float64, device="cuda")
        err = 0.0
        rows = max(1, 10 ** 8 // v)
        sums = (v / (pieces * parts) / 16 + 8) * 2.0 ** -22
        for a in range(0, n, rows):
            x, t = X[a:a + rows].double(), ts[a:a + rows].long()
            z = x @ w.T
            want = torch.logsumexp(z, dim=1)
            top = float(z.abs().max())
            e = 2 * (d / 16 + 2) * 2.0 ** -23 * float((x.abs() @ w.abs().T).max()) + 2.0 ** -20 * (1 + top)
            err = max(err, e)
            within(tensor(lse)[a:a + rows].cpu().numpy(), want.cpu().numpy(), e, "lse")
            p = z.sub_(want[:, None]).exp_()
            ok = t >= 0
            p[ok.nonzero()[:, 0], t[ok]] -= 1
            p *= torch.where(ok, dl[a:a + rows].double(), 0.0)[:, None]
            rel = 2 * ref.H + 4 * e + 2.0 ** -13 + sums
            wx = p @ w
            gw_want += p.T @ x
            p.abs_()
            within(tensor(gx)[a:a + rows].cpu().numpy(), wx.cpu().numpy(), (rel * (p @ w.abs())).cpu().numpy() + ref.HMIN, "dX")
            gw_size += p.T @ x.abs()
        rel = 3 * ref.H + 4 * err + 2.0 ** -13 + (n / 16 + 8) * 2.0 ** -22
        within(tensor(gw).cpu().numpy(), gw_want.cpu().numpy(), (rel * gw_size).cpu().numpy() + 2 * ref.HMIN, "dW")
        for a in [loss, lse, gx, gw] + ins:
            a.free()
