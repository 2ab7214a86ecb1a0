"""The attention half of a decoder layer: the calls whose speed is measured, with their plain forms,
the work they cannot do without and their results in 64 bits.

* ``norm``    RMS norm of every head of queries, keys and values with the position rotation in the
              same pass, and its gradients: ``_lib.head_norm_rope`` and
              ``_lib.head_norm_rope_backward``, a training step
* ``append``  the serving form: the same on the way into a paged key-value cache, ``_lib.append_kv``
* ``prompt``  attention over packed prompts, causal, with grouped heads: ``_lib.attention``
              (``dir`` "fwd"), and with ``_lib.attention_backward`` a training step ("train")
* ``decode``  attention of one new token per sequence over the paged cache: ``_lib.decode_attention``

``T`` is the number of tokens, ``lens`` the sequences' lengths, ``Hq`` and ``Hk`` the query and
key-value heads, ``D`` the head size, ``R`` how many of a head's columns the position turns, ``page``
the tokens of a page and ``window`` the last keys that a query sees (0: all).
"""
import math
from types import SimpleNamespace

import torch

own = False

EPS = 1e-6
THETA = 10000.0
FAR = 131072  # positions of the tables
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a training step on a handful of tokens: launch and latency
        {"name": "norm_7", "kind": "norm", "dtype": "bf16", "T": 7, "Hq": 16, "Hk": 8, "D": 256, "R": 256},
        # a training batch's tokens, rows left over by every grouping: the memory's rate
        {"name": "norm_8191", "kind": "norm", "dtype": "bf16", "T": 8191, "Hq": 16, "Hk": 8, "D": 256, "R": 256},
        # one decoded token of a chat
        {"name": "append_1", "kind": "append", "dtype": "bf16", "T": 1, "Hq": 16, "Hk": 8, "D": 256, "R": 256,
         "page": 64},
        # a long prompt on its way into the cache, a quarter of each head turned
        {"name": "append_4097", "kind": "append", "dtype": "bf16", "T": 4097, "Hq": 16, "Hk": 2, "D": 512, "R": 128,
         "page": 64},
        # a short question
        {"name": "prompt_180", "kind": "prompt", "dir": "fwd", "dtype": "bf16", "lens": "180", "Hq": 16, "Hk": 8,
         "D": 256, "window": 1024},
        # prompts of a served batch packed together, one key-value head for all
        {"name": "prompt_packed", "kind": "prompt", "dir": "fwd", "dtype": "fp16",
         "lens": "1 517 2049 33 1024 180 7 251", "Hq": 8, "Hk": 1, "D": 128, "window": 0},
        # a long document, wide heads
        {"name": "prompt_4096", "kind": "prompt", "dir": "fwd", "dtype": "bf16", "lens": "4096", "Hq": 16, "Hk": 2,
         "D": 512, "window": 0},
        # a training step on a few short sequences
        {"name": "train_233", "kind": "prompt", "dir": "train", "dtype": "fp16", "lens": "5 1 64 130 33", "Hq": 4,
         "Hk": 4, "D": 64, "window": 0},
        # a training batch
        {"name": "train_8192", "kind": "prompt", "dir": "train", "dtype": "bf16", "lens": "4096 2500 1596", "Hq": 16,
         "Hk": 8, "D": 256, "window": 0},
        # a chat's next token
        {"name": "decode_1", "kind": "decode", "dtype": "bf16", "lens": "181", "Hq": 16, "Hk": 8, "D": 256, "page": 64,
         "window": 1024},
        # a batch of chats of all ages, a layer that sees the last tokens alone
        {"name": "decode_32", "kind": "decode", "dtype": "bf16", "lens": _spread(32, 1, 4099), "Hq": 16, "Hk": 8,
         "D": 256, "page": 64, "window": 1024},
        # the same batch's longest, a layer that sees everything
        {"name": "decode_24_long", "kind": "decode", "dtype": "bf16", "lens": _spread(24, 997, 16888), "Hq": 16,
         "Hk": 2, "D": 512, "page": 64, "window": 0},
    ]


def _spread(n, least, most):
    """n lengths from least to most in equal ratios, as a text, the long ones among the short."""
    r = [int(round(least * (most / least) ** (i / (n - 1)))) for i in range(n)]
    return " ".join(str(r[i * 7 % n]) for i in range(n))


def _log(rng, least, most):
    """A size spread over the logarithm of least .. most."""
    return min(most, max(least, int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))))


def _cost(case):
    """What a case costs, of its work and of the plain form's: packed prompts as one square, decoded
    sequences as long as the longest."""
    w = work(case)
    if case["kind"] not in ("prompt", "decode"):
        return w["bytes"]
    lens = _lens(case)
    if case["kind"] == "prompt":
        return max(w["flops"] / 11e3, case["Hq"] * sum(lens) ** 2 / 16)
    return max(w["bytes"], len(lens) * max(lens) * case["Hk"] * case["D"])


def draw(rng):
    """One more case of these ranges, not one of the listed."""
    known = [{n: v for n, v in c.items() if n != "name"} for c in listed()]
    most = {}
    for c in known:  # the largest listed one of its kind bounds a drawn case
        most[c["kind"]] = max(most.get(c["kind"], 0), _cost(c))
    while True:
        case = _draw(rng)
        if case not in known and _cost(case) <= most[case["kind"]]:
            return case


def _heads(rng):
    Hk = rng.choice([1, 2, 4, 8])
    return {"Hq": Hk * rng.choice([1, 2, 3, 4, 8]), "Hk": Hk}


def _draw(rng):
    kind = rng.choice(["norm", "append", "prompt", "prompt", "decode", "decode"])
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16"]), **_heads(rng)}
    if kind in ("norm", "append"):
        D = rng.choice([64, 128, 256, 256, 512, 80, 96])
        case |= {"T": _log(rng, 1, 8192), "D": D, "R": rng.choice([D, D, D // 2, D // 4 // 8 * 8])}
        if kind == "norm":
            return {**case, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
        return {**case, "page": rng.choice([16, 32, 64, 128])}
    case |= {"D": rng.choice([64, 128, 256, 256, 512]), "window": rng.choice([0, 0, 16, 512, 1024])}
    if kind == "prompt":
        lens, n = [], rng.randint(1, 12)
        for _ in range(n):
            lens.append(_log(rng, 1, 4096))
            if sum(lens) > 8192:
                lens.pop()
        return {**case, "dir": rng.choice(["fwd", "train"]), "lens": " ".join(map(str, lens))}
    most = _log(rng, 16, 16888)
    lens = [_log(rng, 1, most) for _ in range(_log(rng, 1, 64))]
    return {**case, "lens": " ".join(map(str, lens)), "page": rng.choice([16, 32, 64, 128])}


# ---------------------------------------------------------------------------- inputs


def _lens(c):
    return [int(n) for n in c["lens"].split()]


def _tables(P, R):
    """cos and sin of position x frequency [P, R / 2], frequencies THETA^(-2 i / R), angles in 64 bits."""
    angle = torch.arange(P, device="cuda", dtype=torch.float64)[:, None] * _frequencies(R)
    return angle.cos().float(), angle.sin().float()


def _frequencies(R):
    return THETA ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)


def _inputs(case, seed):
    """Inputs from the seed alone: projections with a scale of their own per head and token, norm weights
    around one, normalised queries and keys with a few strong matches, gradients a hundredth of them."""
    c = SimpleNamespace(**case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[c.dtype]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(dt)

    def projection(T, H):
        t = torch.randn(T, H, c.D, generator=g, device="cuda")
        return (t * (0.3 + 2.0 * torch.rand(T, H, 1, generator=g, device="cuda"))).to(dt)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int32)

    s = SimpleNamespace(case=case)
    if c.kind in ("norm", "append"):
        s.q, s.k, s.v = projection(c.T, c.Hq), projection(c.T, c.Hk), projection(c.T, c.Hk)
        s.qw, s.kw = normal(c.D, std=0.1, mean=1.0), normal(c.D, std=0.1, mean=1.0)
        first = int(whole(0, FAR - c.T + 1, 1))
        s.positions = torch.arange(first, first + c.T, device="cuda", dtype=torch.int32)
    if c.kind == "norm":
        s.dq, s.dk, s.dv = (normal(*t.shape, std=0.01) for t in (s.q, s.k, s.v))
    elif c.kind == "append":
        pages = -(-c.T // c.page) + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(c.T, device="cuda") + int(whole(0, c.page, 1))
        s.slots = (order[at // c.page] * c.page + at % c.page).int()
        s.kc, s.vc = normal(pages, c.Hk, c.page, c.D), normal(pages, c.Hk, c.page, c.D)
    elif c.kind == "prompt":
        lens = _lens(case)
        T = sum(lens)
        # scores of standard deviation 1.5
        s.q, s.k, s.v = normal(T, c.Hq, c.D, std=1.5), normal(T, c.Hk, c.D), normal(T, c.Hk, c.D)
        s.cu = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
        s.dout = normal(T, c.Hq, c.D, std=0.01) if c.dir == "train" else None
    else:
        lens = _lens(case)
        need = [-(-n // c.page) for n in lens]
        pages = sum(need) + 5
        order = torch.randperm(pages, generator=g, device="cuda").int()
        s.table = torch.full((len(lens), max(need)), -1, device="cuda", dtype=torch.int32)
        for b, n in enumerate(need):
            s.table[b, :n] = order[sum(need[:b]):sum(need[:b + 1])]
        s.lengths = torch.tensor(lens, device="cuda", dtype=torch.int32)
        s.q = normal(len(lens), c.Hq, c.D, std=1.5)
        s.kc, s.vc = normal(pages, c.Hk, c.page, c.D), normal(pages, c.Hk, c.page, c.D)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("norm", "append"):
        s.cos, s.sin = _tables(FAR, case["R"])
    return s


# ---------------------------------------------------------------------------- the calls


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from hybridagent_amd import _lib

    c = s.case
    if c["kind"] == "norm":
        rot = (s.cos, s.sin, s.positions, s.qw, s.kw, EPS)
        q, k, v = _lib.head_norm_rope(s.q, s.k, s.v, *rot)
        grads = _lib.head_norm_rope_backward(s.dq, s.dk, s.dv, s.q, s.k, s.v, *rot)
        return dict(zip(("q", "k", "v", "dq", "dk", "dv", "dqw", "dkw"), (q, k, v, *grads)))
    if c["kind"] == "append":
        q = _lib.append_kv(s.q, s.k, s.v, s.cos, s.sin, s.positions, s.slots, s.kc, s.vc, s.qw, s.kw, EPS, v_norm=True)
        return {"q": q, "kc": s.kc, "vc": s.vc}
    if c["kind"] == "decode":
        return _lib.decode_attention(s.q, s.kc, s.vc, s.table, s.lengths, window=c["window"])
    if c["dir"] == "fwd":
        return _lib.attention(s.q, s.k, s.v, s.cu, window=c["window"])
    out, lse = _lib.attention(s.q, s.k, s.v, s.cu, window=c["window"], return_lse=True)
    dq, dk, dv = _lib.attention_backward(s.dout, s.q, s.k, s.v, out, lse, s.cu, window=c["window"])
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _turn(x, cos, sin):
    """Columns i and i + R / 2 of the first R turned by the position's angles."""
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


def _unit(x):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * r, r


def _norm_back(dy, x, w):
    """The gradients of the rows and the weight of x / rms(x) * w."""
    xh, r = _unit(x)
    u = dy if w is None else dy * w
    return r * (u - xh * (u * xh).mean(-1, keepdim=True)), (dy * xh).sum((0, 1))


def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v over the seen keys of [heads, rows, D], with the weights."""
    scores = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    return p @ v, p


def _run_plain(s):
    c = s.case
    dt = s.q.dtype
    D, scale = c["D"], c["D"] ** -0.5
    if c["kind"] in ("norm", "append"):
        cos, sin = s.cos[s.positions][:, None], s.sin[s.positions][:, None]
        q, k, v = s.q.float(), s.k.float(), s.v.float()
        qw, kw = s.qw.float(), s.kw.float()
        q2, k2, v2 = (t.to(dt) for t in (_turn(_unit(q)[0] * qw, cos, sin), _turn(_unit(k)[0] * kw, cos, sin),
                                         _unit(v)[0]))
        if c["kind"] == "append":
            page, row = s.slots.long() // c["page"], s.slots.long() % c["page"]
            s.kc[page, :, row] = k2
            s.vc[page, :, row] = v2
            return {"q": q2, "kc": s.kc, "vc": s.vc}
        dq, dqw = _norm_back(_turn(s.dq.float(), cos, -sin), q, qw)
        dk, dkw = _norm_back(_turn(s.dk.float(), cos, -sin), k, kw)
        dv, _ = _norm_back(s.dv.float(), v, None)
        return dict(zip(("q", "k", "v", "dq", "dk", "dv", "dqw", "dkw"),
                        (q2, k2, v2, *(t.to(dt) for t in (dq, dk, dv, dqw, dkw)))))
    g = c["Hq"] // c["Hk"]
    if c["kind"] == "decode":
        at = torch.arange(s.table.shape[1] * c["page"], device="cuda")
        seen = at < s.lengths[:, None]
        if c["window"]:
            seen = seen & (at >= s.lengths[:, None] - c["window"])
        rows = s.table.long().clamp(min=0)
        keys, values = (t[rows].float().transpose(2, 3).flatten(1, 2).transpose(1, 2) for t in (s.kc, s.vc))
        q = s.q.float().unflatten(1, (c["Hk"], g))
        return _attend(q, keys, values, seen[:, None, None], scale)[0].flatten(1, 2).to(dt)
    # the packed batch as one: a query sees its own sequence's keys
    T = s.q.shape[0]
    at = torch.arange(T, device="cuda")
    seq = torch.searchsorted(s.cu[1:].long(), at, right=True)
    seen = (seq[:, None] == seq) & (at[:, None] >= at)
    if c["window"]:
        seen &= at[:, None] - at < c["window"]
    q = s.q.float().transpose(0, 1)
    k, v = (t.float().transpose(0, 1).repeat_interleave(g, 0) for t in (s.k, s.v))
    o, p = _attend(q, k, v, seen, scale)
    out = o.transpose(0, 1).to(dt)
    if c["dir"] == "fwd":
        return out
    do = s.dout.float().transpose(0, 1)
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
    grouped = lambda t: t.unflatten(0, (c["Hk"], g)).sum(1).transpose(0, 1).to(dt)
    return {"out": out, "dq": (ds @ k).transpose(0, 1).to(dt), "dk": grouped(ds.transpose(-1, -2) @ q),
            "dv": grouped(p.transpose(-1, -2) @ do)}


# ---------------------------------------------------------------------------- work


def work(case):
    Hq, Hk, D = case["Hq"], case["Hk"], case["D"]
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] in ("norm", "append"):
        T, rows = case["T"], case["T"] * (Hq + 2 * Hk)
        tables = T * (4 * case["R"] + 4) + 2 * D * e
        if case["kind"] == "append":
            return {"bytes": 2 * rows * D * e + tables + 4 * T, "flops": 8 * rows * D}
        # in: the rows and the gradients, out: the results and the rows' gradients
        return {"bytes": 4 * rows * D * e + tables + 2 * D * e, "flops": 25 * rows * D}
    lens, w = _lens(case), case["window"]
    if case["kind"] == "decode":
        keys = sum(min(n, w) if w else n for n in lens)
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * keys * Hk * D * e + 2 * len(lens) * Hq * D * e + 4 * pages + 4 * len(lens),
                "flops": 4 * keys * Hq * D}
    T = sum(lens)
    pairs = sum(n * (n + 1) // 2 - (max(n - w, 0) * (max(n - w, 0) + 1) // 2 if w else 0) for n in lens)
    if case["dir"] == "fwd":
        return {"bytes": 2 * T * (Hq + Hk) * D * e, "flops": 4 * pairs * Hq * D}
    return {"bytes": T * (4 * Hq + 4 * Hk) * D * e, "flops": 14 * pairs * Hq * D}


# ---------------------------------------------------------------------------- 64-bit results


def _rms64(x, w):
    n = x * (x.pow(2).mean(-1, keepdim=True) + EPS).pow(-0.5)
    return n if w is None else n * w


def _rotate64(x, positions, R):
    angle = (positions.double()[:, None] * _frequencies(R))[:, None]
    z = torch.complex(x[..., :R // 2], x[..., R // 2:R]) * torch.polar(torch.ones_like(angle), angle)
    return torch.cat([z.real, z.imag, x[..., R:]], -1)


def _softmax64(q, k, v, window):
    """One sequence: queries [n, Hq, D] at the end of its keys [m, Hk, D]."""
    n, m, g = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    scores = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(q.shape[-1])
    at = torch.arange(m - n, m, device="cuda")[:, None] - torch.arange(m, device="cuda")
    hidden = (at < 0) | (at >= window) if window else at < 0
    return torch.einsum("hij,jhd->ihd", scores.masked_fill(hidden, -math.inf).softmax(-1), v)


def exact(case, seed):
    s = _inputs(case, seed)
    kind, R, w = case["kind"], case.get("R"), case.get("window")
    if kind == "norm":
        leaves = [t.double().requires_grad_() for t in (s.q, s.k, s.v, s.qw, s.kw)]
        q, k, v, qw, kw = leaves
        y = (_rotate64(_rms64(q, qw), s.positions, R), _rotate64(_rms64(k, kw), s.positions, R), _rms64(v, None))
        grads = torch.autograd.grad(y, leaves, [t.double() for t in (s.dq, s.dk, s.dv)])
        return dict(zip(("q", "k", "v", "dq", "dk", "dv", "dqw", "dkw"), (*(t.detach() for t in y), *grads)))
    if kind == "append":
        q = _rotate64(_rms64(s.q.double(), s.qw.double()), s.positions, R)
        k = _rotate64(_rms64(s.k.double(), s.kw.double()), s.positions, R)
        kc, vc = (t.double().transpose(1, 2).flatten(0, 1) for t in (s.kc, s.vc))
        kc[s.slots.long()], vc[s.slots.long()] = k, _rms64(s.v.double(), None)
        return {"q": q, **{n: t.unflatten(0, (-1, case["page"])).transpose(1, 2) for n, t in (("kc", kc), ("vc", vc))}}
    lens = _lens(case)
    if kind == "decode":
        out = []
        for b, n in enumerate(lens):
            first = max(n - w, 0) if w else 0
            at = torch.arange(first, n, device="cuda")
            page, row = s.table[b].long()[at // case["page"]], at % case["page"]
            out.append(_softmax64(s.q[b:b + 1].double(), s.kc[page, :, row].double(), s.vc[page, :, row].double(), 0))
        return torch.cat(out)
    train = case["dir"] == "train"
    parts = {"out": [], "dq": [], "dk": [], "dv": []}
    first = 0
    for n in lens:
        q, k, v = (t[first:first + n].double().requires_grad_(train) for t in (s.q, s.k, s.v))
        y = _softmax64(q, k, v, w)
        parts["out"].append(y.detach())
        if train:
            for name, t in zip(("dq", "dk", "dv"), torch.autograd.grad(y, (q, k, v), s.dout[first:first + n].double())):
                parts[name].append(t)
        first += n
    if not train:
        return torch.cat(parts["out"])
    return {name: torch.cat(t) for name, t in parts.items()}
