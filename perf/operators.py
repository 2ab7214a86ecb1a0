"""The training forms of the framework's dense maps: the calls whose speed is measured, with their
plain forms, the work they cannot do without and their results in 64 bits.

* ``ln``   layer norm over rows: ``_lib.layer_norm`` (``dir`` "fwd": with the statistics a
           backward pass needs) and ``_lib.layer_norm_backward`` ("bwd")
* ``mlp``  the gated feed-forward block of the FFN block's shared MLP: ``_lib.gated_mlp`` ("fwd":
           the serving call), and with ``_lib.gated_mlp_backward`` a training step ("train")
* ``hl``   HybridLink: ``_lib.hybridlink_train`` and ``_lib.hybridlink_backward``, a training step

``T`` is the number of rows (tokens), ``H`` the hidden size (2816 in this repository's model), ``I``
the shared MLP's width (2112).  One row is a chat's latent step or decoded token, some dozens a
batch of them, thousands a training batch's tokens or a prompt.
"""
import math
from types import SimpleNamespace

import torch

own = False

EPS = 1e-5
H0, I0 = 2816, 2112
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the norm of one latent row: launch and latency
        {"name": "ln_fwd_1", "kind": "ln", "dir": "fwd", "dtype": "bf16", "T": 1, "H": H0},
        # a training batch's rows: the memory's rate
        {"name": "ln_fwd_8192", "kind": "ln", "dir": "fwd", "dtype": "bf16", "T": 8192, "H": H0},
        # its backward pass, rows left over by every grouping
        {"name": "ln_bwd_4099", "kind": "ln", "dir": "bwd", "dtype": "bf16", "T": 4099, "H": H0},
        # parameters and rows kept in 32 bits, a width no vector load divides
        {"name": "ln_bwd_1023_odd", "kind": "ln", "dir": "bwd", "dtype": "fp32", "T": 1023, "H": 1001},
        # the shared MLP for one decoded token: the weights' stream
        {"name": "mlp_fwd_1", "kind": "mlp", "dir": "fwd", "T": 1, "H": H0, "I": I0},
        # a large served batch or a short prompt, odd size
        {"name": "mlp_fwd_193", "kind": "mlp", "dir": "fwd", "T": 193, "H": H0, "I": I0},
        # a prompt
        {"name": "mlp_fwd_4096", "kind": "mlp", "dir": "fwd", "T": 4096, "H": H0, "I": I0},
        # a training step on a handful of tokens: weights in, their gradients out
        {"name": "mlp_train_7", "kind": "mlp", "dir": "train", "T": 7, "H": H0, "I": I0},
        # a short sequence
        {"name": "mlp_train_517", "kind": "mlp", "dir": "train", "T": 517, "H": H0, "I": I0},
        # a training batch
        {"name": "mlp_train_8192", "kind": "mlp", "dir": "train", "T": 8192, "H": H0, "I": I0},
        # HybridLink trained on one step's latent rows of a batch of 32
        {"name": "hl_train_32", "kind": "hl", "dir": "train", "T": 32, "H": H0},
        # and on all latent rows of a batch of sequences, odd size
        {"name": "hl_train_2049", "kind": "hl", "dir": "train", "T": 2049, "H": H0},
    ]


def _rows(rng, most):
    """A row count spread over the logarithm of 1 .. most."""
    return min(most, max(1, int(round(math.exp(rng.uniform(0.0, math.log(most)))))))


def draw(rng):
    """One more case of these ranges, not one of the listed."""
    known = [{n: v for n, v in c.items() if n != "name"} for c in listed()]
    while True:
        case = _draw(rng)
        if case not in known:
            return case


def _draw(rng):
    kind = rng.choice(["ln", "ln", "mlp", "mlp", "mlp", "hl"])
    T = _rows(rng, {"ln": 8192, "mlp": 8192, "hl": 4096}[kind])
    if kind == "ln":
        H = rng.choice([H0, H0, 8 * rng.randint(8, 512), rng.randint(64, 4096)])
        return {"kind": kind, "dir": rng.choice(["fwd", "bwd"]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "T": T, "H": H}
    if kind == "mlp":
        H, I = rng.choice([(H0, I0), (H0, I0), (H0, 704), (2048, 512), (32 * rng.randint(8, 88), 32 * rng.randint(4, 66))])
        return {"kind": kind, "dir": rng.choice(["fwd", "train"]), "T": T, "H": H, "I": I}
    return {"kind": kind, "dir": "train", "T": T, "H": rng.choice([H0, H0, 32 * rng.randint(8, 88)])}


# ---------------------------------------------------------------------------- inputs


def _inputs(case, seed):
    """Inputs from the seed alone: rows of residual streams (each with its own mean and scale, a few
    large columns), weights at their initial scales, gradients a hundredth of the rows."""
    c = SimpleNamespace(**case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case.get("dtype", "bf16")]

    def normal(*shape, std=1.0, mean=0.0):
        t = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
        return t.mul_(std).add_(mean).to(dt)

    def residual(T, H):
        t = torch.randn(T, H, generator=g, device="cuda")
        t = t * (0.5 + torch.rand(T, 1, generator=g, device="cuda")) + 0.2 * torch.randn(T, 1, generator=g, device="cuda")
        t[:, ::211] *= 8.0
        return t.to(dt)

    s = SimpleNamespace(case=case)
    if c.kind == "ln":
        s.x = residual(c.T, c.H)
        s.w, s.b = normal(c.H, std=0.05, mean=1.0), normal(c.H, std=0.02)
        if c.dir == "bwd":
            s.dy = normal(c.T, c.H, std=0.01)
        return s
    if c.kind == "mlp":
        # the block's input is a normalised row
        s.x = normal(c.T, c.H)
        s.gate, s.up = normal(c.I, c.H, std=c.H ** -0.5), normal(c.I, c.H, std=c.H ** -0.5)
        s.down = normal(c.H, c.I, std=c.I ** -0.5)
    else:
        s.x = residual(c.T, c.H)
        std = c.H ** -0.5
        s.params = [normal(c.H, std=0.05, mean=1.0), normal(c.H, std=0.02), normal(c.H, c.H, std=std),
                    normal(c.H, std=0.02), normal(c.H, c.H, std=std), normal(c.H, std=0.02),
                    normal(c.H, std=0.05, mean=1.0), normal(c.H, std=0.02)]
    if c.dir == "train":
        s.dy = normal(c.T, c.H, std=0.01)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "ln" and case["dir"] == "bwd":
        # the statistics that the forward pass left
        x = s.x.double()
        s.mean = x.mean(-1)
        s.rstd = ((x - s.mean[:, None]).pow(2).mean(-1) + EPS).rsqrt().float()
        s.mean = s.mean.float()
    return s


# ---------------------------------------------------------------------------- the calls


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from hybridagent_amd import _lib

    c = s.case
    if c["kind"] == "ln":
        if c["dir"] == "fwd":
            y, mean, rstd = _lib.layer_norm(s.x, s.w, s.b, EPS, return_stats=True)
            return {"y": y, "mean": mean, "rstd": rstd}
        dx, dw, db = _lib.layer_norm_backward(s.dy, s.x, s.w, s.mean, s.rstd)
        return {"dx": dx, "dw": dw, "db": db}
    if c["kind"] == "mlp":
        if c["dir"] == "fwd":
            return _lib.gated_mlp(s.x, s.gate, s.up, s.down)
        y, saved = _lib.gated_mlp(s.x, s.gate, s.up, s.down, return_saved=True)
        dx, dgate, dup, ddown = _lib.gated_mlp_backward(s.dy, s.x, s.gate, s.up, s.down, saved)
        return {"y": y, "dx": dx, "dgate": dgate, "dup": dup, "ddown": ddown}
    y, saved = _lib.hybridlink_train(s.x, *s.params, EPS)
    grads = _lib.hybridlink_backward(s.dy, s.x, *s.params, saved)
    return {"y": y, "grads": list(grads)}


def _ln(x, w, b):
    mean = x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
    return (x - mean) * rstd * w + b, mean, rstd


def _ln_bwd(dy, x, w, mean, rstd):
    xh = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


_C0, _C1 = 0.7978845608028654, 0.044715


def _run_plain(s):
    c = s.case
    dt = s.x.dtype
    x = s.x.float()
    if c["kind"] == "ln":
        w = s.w.float()
        if c["dir"] == "fwd":
            y, mean, rstd = _ln(x, w, s.b.float())
            return {"y": y.to(dt), "mean": mean.squeeze(-1), "rstd": rstd.squeeze(-1)}
        dx, dw, db = _ln_bwd(s.dy.float(), x, w, s.mean[:, None], s.rstd[:, None])
        return {"dx": dx.to(dt), "dw": dw.to(dt), "db": db.to(dt)}
    if c["kind"] == "mlp":
        wg, wu, wd = s.gate.float(), s.up.float(), s.down.float()
        a, b = x @ wg.t(), x @ wu.t()
        t = torch.tanh(_C0 * (a + _C1 * a * a * a))
        act = 0.5 * a * (1.0 + t)
        h = act * b
        y = (h @ wd.t()).to(dt)
        if c["dir"] == "fwd":
            return y
        dy = s.dy.float()
        dh = dy @ wd
        slope = 0.5 * (1.0 + t) + 0.5 * a * (1.0 - t * t) * _C0 * (1.0 + 3.0 * _C1 * a * a)
        da, db = dh * b * slope, dh * act
        return {"y": y, "dx": (da @ wg + db @ wu).to(dt), "dgate": (da.t() @ x).to(dt), "dup": (db.t() @ x).to(dt),
                "ddown": (dy.t() @ h).to(dt)}
    w1, b1, p1, q1, p2, q2, w2, b2 = (p.float() for p in s.params)
    a, m1, r1 = _ln(x, w1, b1)
    z = a @ p1.t() + q1
    cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    g = z * cdf
    r = x + (g @ p2.t() + q2)
    y, m2, r2 = _ln(r, w2, b2)
    dr, dw2, db2 = _ln_bwd(s.dy.float(), r, w2, m2, r2)
    dz = (dr @ p2) * (cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)))
    da, dw1, db1 = _ln_bwd(dz @ p1, x, w1, m1, r1)
    grads = [dr + da, dw1, db1, dz.t() @ a, dz.sum(0), dr.t() @ g, dr.sum(0), dw2, db2]
    return {"y": y.to(dt), "grads": [t.to(dt) for t in grads]}


# ---------------------------------------------------------------------------- work


def work(case):
    T, H = case["T"], case["H"]
    if case["kind"] == "ln":
        e = 4 if case["dtype"] == "fp32" else 2
        if case["dir"] == "fwd":
            return {"bytes": 2 * T * H * e + 2 * H * e + 8 * T, "flops": 8 * T * H}
        return {"bytes": 3 * T * H * e + 3 * H * e + 8 * T, "flops": 14 * T * H}
    if case["kind"] == "mlp":
        I = case["I"]
        if case["dir"] == "fwd":
            return {"bytes": 6 * H * I + 4 * T * H, "flops": 6 * T * H * I}
        return {"bytes": 12 * H * I + 8 * T * H, "flops": 18 * T * H * I}
    return {"bytes": 8 * H * H + 24 * H + 8 * T * H, "flops": 12 * T * H * H}


# ---------------------------------------------------------------------------- 64-bit results


def exact(case, seed):
    s = _inputs(case, seed)
    F = torch.nn.functional
    leaf = lambda t: t.double().requires_grad_(case["dir"] != "fwd")
    x = leaf(s.x)
    if case["kind"] == "ln":
        w, b = leaf(s.w), leaf(s.b)
        y = F.layer_norm(x, (case["H"],), w, b, EPS)
        if case["dir"] == "fwd":
            var, mean = torch.var_mean(x, -1, correction=0)
            return {"y": y, "mean": mean, "rstd": (var + EPS).pow(-0.5)}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s.dy.double())
        return {"dx": dx, "dw": dw, "db": db}
    if case["kind"] == "mlp":
        wg, wu, wd = leaf(s.gate), leaf(s.up), leaf(s.down)
        y = F.linear(F.gelu(F.linear(x, wg), approximate="tanh") * F.linear(x, wu), wd)
        if case["dir"] == "fwd":
            return y
        grads = torch.autograd.grad(y, (x, wg, wu, wd), s.dy.double())
        return dict(zip(("y", "dx", "dgate", "dup", "ddown"), (y.detach(), *grads)))
    p = [leaf(t) for t in s.params]
    n = (case["H"],)
    r = x + F.linear(F.gelu(F.linear(F.layer_norm(x, n, p[0], p[1], EPS), p[2], p[3])), p[4], p[5])
    y = F.layer_norm(r, n, p[6], p[7], EPS)
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, (x, *p), s.dy.double()))}
