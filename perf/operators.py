"""The training-loss operators as they are measured: cross entropy over a vocabulary without the logits
(vocab_xent), distillation from a teacher's top logits (topk_distill) and the balance loss of a router
with its per-expert counts (router_balance), each with its gradient.

`run` computes them in plain torch operations, or (`own`) with the calls a program makes of this library.
Binary16 arrays are torch.float16 here and uint16 bit patterns in the library's API."""
import math

import torch

own = False


# ---- the cases ---------------------------------------------------------------------------------------------
def listed():
    return [
        # log-probability of one token during generation: the weights are read once, everything else is latency
        {"name": "xent score 1 token", "op": "xent", "train": False, "n": 1, "v": 32000, "d": 1024},
        # scoring a batch of continuations against a large vocabulary
        {"name": "xent score 64 tokens", "op": "xent", "train": False, "n": 64, "v": 131072, "d": 4096},
        # a training step whose sizes are multiples of nothing the kernels use
        {"name": "xent train odd", "op": "xent", "train": True, "n": 777, "v": 32003, "d": 1000},
        # an ordinary training step
        {"name": "xent train 4096 tokens", "op": "xent", "train": True, "n": 4096, "v": 65536, "d": 2048},
        # a large model's training step
        {"name": "xent train 8192 tokens", "op": "xent", "train": True, "n": 8192, "v": 131072, "d": 4096},
        # one row: latency
        {"name": "distill 1 row f32", "op": "distill", "t": "f32", "n": 1, "v": 32000, "k": 8, "tau": 1.0},
        # few rows over a very large vocabulary: fewer rows than multiprocessors
        {"name": "distill 16 rows f16", "op": "distill", "t": "f16", "n": 16, "v": 200000, "k": 128, "tau": 2.0},
        # rows whose length and start are not aligned
        {"name": "distill odd f32", "op": "distill", "t": "f32", "n": 2049, "v": 50001, "k": 20, "tau": 1.5},
        # an ordinary batch of a student's logits
        {"name": "distill 4096 rows f16", "op": "distill", "t": "f16", "n": 4096, "v": 131072, "k": 64, "tau": 2.0},
        # a handful of tokens and experts: latency
        {"name": "router 16 tokens f32", "op": "router", "t": "f32", "n": 16, "e": 8, "k": 2},
        # an ordinary batch, a number of experts that is no power of two
        {"name": "router 8192 tokens f16", "op": "router", "t": "f16", "n": 8192, "e": 60, "k": 4},
        # a large batch over many experts
        {"name": "router 131072 tokens f32", "op": "router", "t": "f32", "n": 131072, "e": 256, "k": 8},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["xent", "distill", "router"])
    if op == "xent":
        d = spread(32, 4096)
        if rng.random() < 0.75:                       # widths are mostly multiples of eight
            d = max(8, d // 8 * 8)
        return {"op": op, "train": rng.random() < 0.75, "n": spread(1, 8192), "v": spread(100, 131072), "d": d}
    if op == "distill":
        n, v = spread(1, 8192), spread(64, 200000)
        while n * v > 4096 * 131072:
            n //= 2
        return {"op": op, "t": rng.choice(["f16", "f32"]), "n": n, "v": v, "k": min(v, spread(1, 128)),
                "tau": round(rng.uniform(0.5, 4.0), 2)}
    e = spread(2, 512)
    n = spread(1, 262144)
    while n * e > 131072 * 256:
        n //= 2
    return {"op": op, "t": rng.choice(["f16", "f32"]), "n": n, "e": e, "k": min(e, spread(1, 16))}


# ---- inputs ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = dict(device="cuda", generator=g)
    n, s = case["n"], {"op": case["op"]}
    if case["op"] == "xent":
        v, d = case["v"], case["d"]
        s["train"] = case["train"]
        # hidden states of unit size and weights that give logits with a standard deviation of two
        s["x"] = torch.randn(n, d, **dev).half()
        s["w"] = torch.randn(v, d, **dev).mul_(2 / math.sqrt(d)).half()
        # word frequencies fall off as in text; one token in sixteen is padding, which has no target
        t = (v * torch.rand(n, **dev) ** 3).long().clamp_(max=v - 1)
        s["t"] = torch.where(torch.rand(n, **dev) < 1 / 16, -1, t).int()
        # token weights around the mean's 1/n, with a loss scale as half-precision gradients need it
        s["dl"] = torch.rand(n, **dev).add_(0.5).mul_(4096 / n)
    elif case["op"] == "distill":
        v, k = case["v"], case["k"]
        half = case["t"] == "f16"
        s["t"], s["tau"] = case["t"], case["tau"]
        s["s"] = torch.randn(n, v, **dev).mul_(3)
        s["s"] = s["s"].half() if half else s["s"]
        # a teacher that agrees with the student in part; its words in falling order, some rows with fewer of them
        s["i"] = torch.randint(0, v, (n, k), **dev)
        s["i"] = torch.where(torch.rand(n, k, **dev) < 1 / 16, -1, s["i"]).int()
        s["q"] = torch.randn(n, k, **dev).mul_(2).add_(8).sort(dim=1, descending=True)[0]
        s["dl"] = torch.rand(n, **dev).add_(0.5).mul_((4096 if half else 1) / n)
    else:
        e, k = case["e"], case["k"]
        s["t"] = case["t"]
        r = torch.randn(n, e, **dev) + torch.randn(e, **dev)          # some experts are liked more
        s["r"] = r.half() if case["t"] == "f16" else r
        i = s["r"].float().topk(k, dim=1)[1]
        s["i"] = torch.where(torch.rand(n, k, **dev) < 1 / 64, -1, i).int()   # a few assignments are dropped
        s["keep"] = torch.rand(n, **dev) >= 1 / 16                     # a few tokens are padding
        s["dl"] = torch.full((1,), 64.0 if case["t"] == "f16" else 0.01, device="cuda")
    return s


# ---- the library's calls -----------------------------------------------------------------------------------
_ctx = _stream = _event = None
_dropped = []                                          # results whose tensors are gone, with the streams they belong to


def _context():
    global _ctx, _stream, _event
    if _ctx is None:
        import futhark_b200
        _ctx = futhark_b200.Context(device="#0")
        _stream, _event = torch.cuda.ExternalStream(_ctx.stream), torch.cuda.Event()
    return _ctx


def _after(later, earlier):
    """What `later` does from now on comes after what `earlier` has been given so far."""
    _event.record(earlier)
    later.wait_event(_event)


def _wrap(ctx, t):
    """A tensor as an array of the context; the memory is borrowed."""
    name = {torch.float16: "f16", torch.float32: "f32", torch.int32: "i32", torch.bool: "bool"}[t.dtype]
    return ctx.new_raw("%s_%dd" % (name, t.dim()), t.data_ptr(), *t.shape)


class _Result:
    """An array of the context that belongs to the stream of the call, as torch's own tensors do.  When the last tensor on its memory
    is gone it goes back with the next call, behind what that stream then holds."""

    def __init__(self, a, stream):
        self.array, self.stream, self.__cuda_array_interface__ = a, stream, a.__cuda_array_interface__

    def __del__(self):
        _dropped.append((self.array, self.stream))


def _tensor(a, stream):
    t = torch.as_tensor(_Result(a, stream), device="cuda")
    return t.view(torch.float16) if t.dtype == torch.uint16 else t


def _run_own(s):
    ctx = _context()
    here = torch.cuda.current_stream()
    _after(_stream, here)                              # the library works on a stream of its own
    while _dropped:
        a, reader = _dropped.pop()
        if reader.cuda_stream != here.cuda_stream:
            _after(_stream, reader)
        a.free()
    ins = []

    def arr(t):
        ins.append(_wrap(ctx, t))
        return ins[-1]

    if s["op"] == "xent":
        x, w, t = arr(s["x"]), arr(s["w"]), arr(s["t"])
        out = ctx.entry_vocab_xent_f16(x, w, t)
        if s["train"]:
            out = out + ctx.entry_vocab_xent_grad_f16(x, w, t, out[0], out[1], arr(s["dl"]))
    elif s["op"] == "distill":
        z, i, q = arr(s["s"]), arr(s["i"]), arr(s["q"])
        out = ctx.entry_topk_distill(s["t"], s["tau"], z, i, q)
        out = out + (ctx.entry_topk_distill_grad(s["t"], s["tau"], z, i, q, out[1], arr(s["dl"])),)
    else:
        r, keep = arr(s["r"]), arr(s["keep"])
        out = ctx.entry_router_balance(s["t"], r, keep, arr(s["i"]))
        out = out + (ctx.entry_router_balance_grad(s["t"], r, keep, out[1], out[2], arr(s["dl"])),)
    for a in ins:
        a.free()
    _after(here, _stream)
    return tuple(_tensor(a, here) for a in out)


# ---- the plain forms: 32 bits, rounded once at the end --------------------------------------------------------
def _lse(z):
    m = z.max(dim=1, keepdim=True)[0]
    return (z - m).exp().sum(dim=1, keepdim=True).log() + m


def _plain_xent(s):
    x, w, t = s["x"].float(), s["w"].float(), s["t"].long()
    z = x @ w.T
    lse = _lse(z)
    ok = (t >= 0) & (t < w.shape[0])
    at = torch.where(ok, t, 0)[:, None]
    loss = torch.where(ok, (lse - z.gather(1, at))[:, 0], 0.0)
    if not s["train"]:
        return loss, lse[:, 0]
    z.sub_(lse).exp_().scatter_add_(1, at, torch.full_like(lse, -1.0))
    z.mul_(torch.where(ok, s["dl"], 0.0)[:, None])
    return loss, lse[:, 0], (z @ w).half(), (z.T @ x).half()


def _plain_distill(s):
    tau = s["tau"]
    z = s["s"].float() / tau
    i = s["i"].long()
    ok = (i >= 0) & (i < z.shape[1])
    some = ok.any(dim=1, keepdim=True)
    lq = torch.where(ok, s["q"] / tau, -torch.inf)
    lq = torch.where(some, lq, 0.0)
    lq = torch.where(ok, lq - _lse(lq), 0.0)
    q = torch.where(ok, lq.exp(), 0.0)
    lse = _lse(z)
    at = torch.where(ok, i, 0)
    loss = tau * tau * (q * (lq - z.gather(1, at) + lse)).sum(dim=1)
    p = z.sub_(lse).exp_().mul_(some)
    p = p.scatter_add_(1, at, -q).mul_((tau * s["dl"])[:, None])
    return loss, lse[:, 0], p.half() if s["t"] == "f16" else p


def _plain_router(s):
    r, keep, e = s["r"].float(), s["keep"], s["r"].shape[1]
    i = torch.where(keep[:, None], s["i"].long(), -1)
    i = torch.where((i >= 0) & (i < e), i, e).reshape(-1)
    counts = torch.zeros(e + 1, dtype=torch.int32, device=r.device).scatter_add_(0, i, torch.ones_like(i, dtype=torch.int32))[:e]
    p = (r - _lse(r)).exp() * keep[:, None]
    norm = e / (counts.sum().double() * keep.sum().double()).clamp(min=1.0)
    loss = ((p.sum(dim=0).double() * counts.double()).sum() * norm).float().reshape(1)
    # counts around their mean: where they are nearly equal the gradient is what is left of a difference
    c = (counts - counts.sum() // e).float()
    grad = p * (c - (p * c).sum(dim=1, keepdim=True)) * (norm * s["dl"].double()).float()
    return loss, counts, norm.float().reshape(1), grad.half() if s["t"] == "f16" else grad


def run(state):
    if own:
        return _run_own(state)
    return {"xent": _plain_xent, "distill": _plain_distill, "router": _plain_router}[state["op"]](state)


# ---- the definitions in 64 bits, differentiated by autograd ----------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "xent":
        w = s["w"].double().requires_grad_(case["train"])
        loss, lse, dx = [], [], []
        for a in range(0, case["n"], 1024):             # rows are independent: the logits of a few at a time
            x = s["x"][a:a + 1024].double().requires_grad_(case["train"])
            t = s["t"][a:a + 1024].long()
            lp = torch.log_softmax(x @ w.T, dim=1)
            z0 = x.detach() @ w.detach()[0]
            lse.append(z0 - lp.detach()[:, 0])
            li = torch.nn.functional.nll_loss(lp, t, ignore_index=-1, reduction="none")
            loss.append(li.detach())
            if case["train"]:
                li.backward(s["dl"][a:a + 1024].double())
                dx.append(x.grad)
        out = (torch.cat(loss), torch.cat(lse))
        return out + (torch.cat(dx), w.grad) if case["train"] else out
    if case["op"] == "distill":
        tau, loss, lse, grad = case["tau"], [], [], []
        for a in range(0, case["n"], 1024):
            z = s["s"][a:a + 1024].double().requires_grad_(True)
            i, q = s["i"][a:a + 1024].long(), s["q"][a:a + 1024].double()
            lp = torch.log_softmax(z / tau, dim=1)
            lq = torch.log_softmax(q.masked_fill(i < 0, -1e300) / tau, dim=1)
            wt = lq.exp() * (i >= 0)
            li = tau ** 2 * (wt * (torch.where(i >= 0, lq, 0.0) - lp.gather(1, i.clamp(min=0)))).sum(dim=1)
            li.backward(s["dl"][a:a + 1024].double())
            loss.append(li.detach())
            lse.append((torch.logsumexp(z.detach() / tau, dim=1)))
            grad.append(z.grad)
        return torch.cat(loss), torch.cat(lse), torch.cat(grad)
    r = s["r"].double().requires_grad_(True)
    e, keep, i = case["e"], s["keep"], s["i"].long()
    hit = (torch.nn.functional.one_hot(i.clamp(min=0), e) * ((i >= 0) & keep[:, None])[:, :, None]).sum(dim=(0, 1))
    m, c = int(keep.sum()), int(hit.sum())
    norm = e / max(1, m * c)
    loss = (torch.softmax(r, dim=1)[keep].sum(dim=0) * hit.double()).sum() * norm
    loss.backward(s["dl"][0].double())
    return loss.detach().reshape(1), None, torch.full((1,), norm, dtype=torch.float64), r.grad


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def work(case):
    n = case["n"]
    if case["op"] == "xent":
        v, d = case["v"], case["d"]
        reads, flops = 2 * (n + v) * d + 4 * n + 8 * n, 2 * n * v * d
        if not case["train"]:
            return {"bytes": reads, "flops": flops}
        # gradients as large as what they belong to; the logits' gradient meets the weights and the hidden states
        return {"bytes": 2 * reads, "flops": 3 * flops}
    if case["op"] == "distill":
        v, k, b = case["v"], case["k"], 2 if case["t"] == "f16" else 4
        return {"bytes": 2 * n * v * b + 8 * n * k + 12 * n, "flops": 8 * n * v}
    e, k, b = case["e"], case["k"], 2 if case["t"] == "f16" else 4
    return {"bytes": 2 * n * e * b + 4 * n * k + n + 8 * e, "flops": 10 * n * e}
