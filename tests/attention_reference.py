"""The attention half of a decoder layer in 64 bits, from the formulas, with the element by element
bounds of the kernels' errors: rounding to a type is off by u = eps / 2 of the value at most, fp32
sums of n terms by n 2^-24 of the sum of their magnitudes."""
import math

import torch

F32 = 2.0 ** -24
# exp2 and log2 of the hardware, their arguments' products and a rescaling or two: some units in the last place
FUN = 2.0 ** -20


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the step of the smallest numbers: fp16's end near the weights of long sequences."""
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def normal(seed, *shape, dtype=torch.bfloat16, std=1.0, mean=0.0, device="cuda:0"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=device) * std + mean).to(dtype)


def offsets(lens, device="cuda:0"):
    return torch.tensor([0, *lens], device=device).cumsum(0).to(torch.int32)


def seen_keys(n, m, causal, window, device):
    """[n, m]: whether query i, at i + m - n, sees key j."""
    at = torch.arange(n, device=device)[:, None] + (m - n)
    j = torch.arange(m, device=device)
    seen = torch.ones(n, m, dtype=torch.bool, device=device)
    if causal:
        seen = j <= at
        if window:
            seen = seen & (j > at - window)
    return seen


def attend(q, k, v, scale, causal, window, dtype, dout=None):
    """One sequence, q [n, Hq, D], k, v [m, Hk, D]: {name: (value, bound)} of out, lse and with dout of
    dq, dk and dv."""
    n, Hq, D = q.shape
    m, Hk = k.shape[:2]
    g = Hq // Hk
    u, tiny = half_step(dtype), least(dtype)
    Q = q.double().transpose(0, 1)
    K, V = (t.double().transpose(0, 1).repeat_interleave(g, 0) for t in (k, v))
    seen = seen_keys(n, m, causal, window, q.device)
    s = scale * (Q @ K.transpose(1, 2))
    es = (D + 4) * F32 * scale * (Q.abs() @ K.abs().transpose(1, 2))  # the scores' error
    s = s.masked_fill(~seen, -math.inf)
    empty = ~seen.any(-1)
    top = s.amax(-1, keepdim=True) if m else s.new_zeros(Hq, n, 1)
    top = top.masked_fill(empty[:, None], 0.0)
    p = (s - top).exp()
    l = p.sum(-1, keepdim=True)
    w = p / l.masked_fill(l == 0, 1.0)
    es = es.masked_fill(~seen, 0.0)
    far = es.amax(-1, keepdim=True) if m else es.new_zeros(Hq, n, 1)
    e32 = 2 * far + FUN + m * F32 + F32 * (s - top).abs().masked_fill(~seen, 0.0)
    out = w @ V
    eout = ((w * (u + e32) + tiny) * seen) @ V.abs() + u * out.abs() + tiny
    lse = (top + l.log()).squeeze(-1)
    res = {"out": (out, eout), "lse": (lse, (far + FUN + m * F32).squeeze(-1) + 2.0 ** -21 * lse.abs().nan_to_num(0, 0, 0))}
    res = {"out": tuple(t.transpose(0, 1) for t in res["out"]), "lse": res["lse"]}
    if dout is None:
        return res
    G = dout.double().transpose(0, 1)
    dp = G @ V.transpose(1, 2)
    delta = (G * out).sum(-1, keepdim=True)
    ds = w * (dp - delta)
    # lse is in fp32
    ew = e32 + 2.0 ** -21 * lse.abs().nan_to_num(0, 0, 0).unsqueeze(-1)
    edp = (D + 4) * F32 * (G.abs() @ V.abs().transpose(1, 2))
    edelta = (G.abs() * eout).sum(-1, keepdim=True) + (D + 4) * F32 * (G * out).abs().sum(-1, keepdim=True)
    eds = (w * (edp + edelta) + (u + ew) * ds.abs() + ew * w * (dp.abs() + delta.abs()) * F32 + tiny) * seen
    ep = (w * (u + ew) + tiny) * seen
    fold = lambda t: t.unflatten(0, (Hk, g)).sum(1).transpose(0, 1)
    dq, dk, dv = scale * (ds @ K), scale * (ds.transpose(1, 2) @ Q), w.transpose(1, 2) @ G
    many = (m + n * g) * F32
    end = lambda v, e, mag: (v, e + many * mag + u * v.abs() + tiny)
    res["dq"] = tuple(t.transpose(0, 1) for t in end(dq, scale * (eds @ K.abs()), scale * (ds.abs() @ K.abs())))
    res["dk"] = end(fold(dk), fold(scale * (eds.transpose(1, 2) @ Q.abs())),
                    fold(scale * (ds.abs().transpose(1, 2) @ Q.abs())))
    res["dv"] = end(fold(dv), fold(ep.transpose(1, 2) @ G.abs()), fold(w.transpose(1, 2) @ G.abs()))
    return res


def packed(q, k, v, cu_q, cu_k, scale, causal, window, dout=None):
    """``attend`` over packed sequences; rows behind the last are zero."""
    a, b = cu_q.tolist(), cu_k.tolist()
    Tq, Hq, D = q.shape
    res = {"out": [torch.zeros(Tq, Hq, D, dtype=torch.float64, device=q.device) for _ in range(2)],
           "lse": [torch.full((Hq, Tq), -math.inf, dtype=torch.float64, device=q.device),
                   torch.zeros(Hq, Tq, dtype=torch.float64, device=q.device)]}
    if dout is not None:
        res["dq"] = [torch.zeros_like(res["out"][0]) for _ in range(2)]
        for n in ("dk", "dv"):
            res[n] = [torch.zeros(k.shape, dtype=torch.float64, device=q.device) for _ in range(2)]
    for i in range(len(a) - 1):
        one = attend(q[a[i]:a[i + 1]], k[b[i]:b[i + 1]], v[b[i]:b[i + 1]], scale, causal, window, q.dtype,
                     None if dout is None else dout[a[i]:a[i + 1]])
        for name, pair in one.items():
            for t, x in zip(res[name], pair):
                if name == "lse":
                    t[:, a[i]:a[i + 1]] = x
                elif name in ("out", "dq"):
                    t[a[i]:a[i + 1]] = x
                else:
                    t[b[i]:b[i + 1]] = x
    return res


def check(got, want, what, slack=0.0):
    """got against (value, bound), element by element; equal where the value is not finite."""
    value, bound = want
    assert got.shape == value.shape, (what, got.shape, value.shape)
    got = got.double()
    fine = value.isfinite()
    assert torch.equal(got[~fine].nan_to_num(nan=1e300), value[~fine].nan_to_num(nan=1e300)), f"{what}: not finite"
    off = (got - value).abs()[fine]
    over = off > bound[fine] + slack
    share = float((off / bound[fine].clamp(min=1e-300)).max()) if off.numel() else 0.0
    print(f"{what}: {share:.3f} of the bound", flush=True)
    assert not bool(over.any() | off.isnan().any()), f"{what}: {int(over.sum())} of {off.numel()} beyond their bound ({share:.2f})"


def rope_tables(P, R, theta=10000.0, device="cuda:0"):
    angle = torch.arange(P, device=device, dtype=torch.float64)[:, None] * theta ** (
        -torch.arange(0, R, 2, device=device, dtype=torch.float64) / R)
    return angle.cos().float(), angle.sin().float()
