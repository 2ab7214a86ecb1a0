"""HybridLink's training form element by element against its formula in 64 bits.

The operands of the products (a, g, dr, dz) and the results are rounded to bf16 once, from
fp32: a rounding moves a value v by at most U |v|, U = 2^-8, and where roundings add up they are
independent, each uniform within that.  So for every element the variance of what reaches it
is carried along the formula, (U v)^2 / 3 for a rounding, squared weights for a map's, and an
element may be off by eight standard deviations, U of itself for its own rounding, and fp32's
share: 64 E32 of the magnitudes in its last sum (E32 = 2^-24; the sums before it, some 1e-5 of
their values, are in the 2 % that the deviations are widened by, as are terms of second order).
A wrong row, column, or group of lanes of a tile is a whole value off, some thirty deviations."""
import math

import pytest
import torch

import test_gpu_training as base
from hybridagent_amd import _lib

pytestmark = pytest.mark.gpu

U, E32 = 2.0 ** -8, 2.0 ** -24
BF = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert _lib.available(), "libw4a16moe.so must be built"
    return torch.device("cuda:0")


def _rounded(v, var):
    """The variance of v after a rounding to bf16."""
    return var + (U * v).square() / 3


def _norm_var(var, xh, scale):
    """Through v -> scale (v - mean v - xh mean(v xh)), the part of a norm that is linear in v."""
    n = var.shape[-1]
    return scale.square() * (var + var.mean(-1, keepdim=True) / n
                             + xh.square() * (xh.square() * var).mean(-1, keepdim=True) / n)


def _stats(x, eps):
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    return (x - mean) * rstd, rstd


def _mean(v):
    return v.mean(-1, keepdim=True)


def expected(h, params, dout, eps=1e-5):
    """[(name, value, variance, fp32's share)] of out, dh and the eight parameters' gradients."""
    h, w1, b1, p1, q1, p2, q2, w2, b2, d = (t.double() for t in (h, *params, dout))
    s1, s2 = p1.square(), p2.square()
    x1, r1 = _stats(h, eps)
    a = x1 * w1 + b1
    va = _rounded(a, torch.zeros_like(a))
    z = a @ p1.t() + q1
    vz = va @ s1.t()
    cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    phi = torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    slope, curve = cdf + z * phi, phi * (2 - z * z)
    g = z * cdf
    vg = _rounded(g, slope.square() * vz)
    r = h + g @ p2.t() + q2
    vr = vg @ s2.t()
    x2, r2 = _stats(r, eps)
    vx2 = _norm_var(vr, x2, r2)                     # of x2 = (r - mean) rstd
    n = h.shape[-1]
    rows = []
    out = x2 * w2 + b2
    rows.append(("out", out, w2.square() * vx2, out.abs() + b2.abs()))
    # dr = rstd (e - mean e - x2 m), e = d w2, m = mean(e x2); x2 and rstd carry r's deviations
    e = d * w2
    m = _mean(e * x2)
    dr = r2 * (e - _mean(e) - x2 * m)
    vm = _mean(e.square() * vx2) / n
    rel = _mean(x2.square() * vr * r2.square()) / n  # of rstd, relative
    vdr = r2.square() * (m.square() * vx2 + x2.square() * vm) + dr.square() * rel
    vdr_op = _rounded(dr, vdr)
    dg = dr @ p2
    vdg = vdr_op @ s2
    dz = dg * slope
    vdz = slope.square() * vdg + (dg * curve).square() * vz
    vdz_op = _rounded(dz, vdz)
    da = dz @ p1
    vda = vdz_op @ s1
    c = da * w1
    back = r1 * (c - _mean(c) - x1 * _mean(c * x1))
    dh = dr + back
    f32 = r2 * (e.abs() + _mean(e.abs()) + x2.abs() * _mean((e * x2).abs())) \
        + r1 * (c.abs() + _mean(c.abs()) + x1.abs() * _mean((c * x1).abs()))
    rows.append(("dh", dh, vdr + _norm_var(w1.square() * vda, x1, r1), f32))
    rows.append(("dln1_w", (da * x1).sum(0), (vda * x1.square()).sum(0), (da * x1).abs().sum(0)))
    rows.append(("dln1_b", da.sum(0), vda.sum(0), da.abs().sum(0)))
    rows.append(("dp1_w", dz.t() @ a, vdz_op.t() @ a.square() + dz.square().t() @ va, dz.abs().t() @ a.abs()))
    rows.append(("dp1_b", dz.sum(0), vdz_op.sum(0), dz.abs().sum(0)))
    rows.append(("dp2_w", dr.t() @ g, vdr_op.t() @ g.square() + dr.square().t() @ vg, dr.abs().t() @ g.abs()))
    rows.append(("dp2_b", dr.sum(0), vdr.sum(0), dr.abs().sum(0)))
    rows.append(("dln2_w", (d * x2).sum(0), (d.square() * vx2).sum(0), (d * x2).abs().sum(0)))
    rows.append(("dln2_b", d.sum(0), torch.zeros(n, dtype=d.dtype, device=d.device), d.abs().sum(0)))
    return rows


def _check(got, want, what):
    for p, (name, v, var, f32) in zip(got, want):
        tol = 1.02 * 8 * var.sqrt() + U * v.abs() + 64 * E32 * f32
        e = (p.double() - v).abs()
        print(f"{what} {name}: worst {float((e / tol.clamp_min(1e-300)).max()):.3f} of the tolerance", flush=True)
        assert (e <= tol).all(), f"{what} {name}: {int((e > tol).sum())} of {e.numel()} beyond the tolerance"


def _shapes(test):
    """The (T, H) that a test of the whole results runs."""
    return [v for mark in test.pytestmark if mark.name == "parametrize" for v in mark.args[1]]


SHAPES = [s for t in (base.test_hybridlink_training, base.test_hybridlink_few_rows_of_wide_or_narrow_outputs,
                      base.test_hybridlink_every_tile) for s in _shapes(t)]


@pytest.mark.parametrize("T,H", SHAPES + [(513, 2816), (2049, 2816)])
def test_every_element(dev, T, H):
    h, params, dout = base._link_inputs(dev, T, H, 700 + T + H)
    out, saved = _lib.hybridlink_train(h, *params)
    grads = _lib.hybridlink_backward(dout, h, *params, saved)
    _check((out, *grads), expected(h, params, dout), f"{T}x{H}")


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("T", [5, 40, 64, 300, 700])
def test_a_row_that_is_not_finite_stays_alone(dev, T, bad):
    """The other rows of out and dh keep their bits, whatever one row of h or of dout holds; the
    gradients of the parameters sum over all rows and are not finite."""
    H, r = 96, 3
    h, params, dout = base._link_inputs(dev, T, H, 800 + T)
    out, saved = _lib.hybridlink_train(h, *params)
    dh = _lib.hybridlink_backward(dout, h, *params, saved)[0]
    others = torch.arange(T, device=dev) != r
    h2, d2 = h.clone(), dout.clone()
    h2[r], d2[r] = bad, bad
    out2, saved2 = _lib.hybridlink_train(h2, *params)
    assert torch.equal(out2[others], out[others]) and not torch.isfinite(out2[r]).any()
    for grads in (_lib.hybridlink_backward(dout, h2, *params, saved2), _lib.hybridlink_backward(d2, h, *params, saved)):
        assert torch.equal(grads[0][others], dh[others]) and not torch.isfinite(grads[0][r]).any()
        assert not any(torch.isfinite(t).any() for t in grads[1:7])


def test_what_lies_around_the_weights_is_not_read(dev):
    """The linears' weights between rows that are not finite: the same bits."""
    T, H = 70, 96
    h, params, dout = base._link_inputs(dev, T, H, 900)
    wide = [torch.full((H + 2, H), math.nan, dtype=BF, device=dev) for _ in range(2)]
    views = [w[1:-1].copy_(p) for w, p in zip(wide, (params[2], params[4]))]
    padded = [*params[:2], views[0], params[3], views[1], *params[5:]]
    out, saved = _lib.hybridlink_train(h, *params)
    out2, saved2 = _lib.hybridlink_train(h, *padded)
    assert torch.equal(out, out2)
    for p, q in zip(_lib.hybridlink_backward(dout, h, *params, saved),
                    _lib.hybridlink_backward(dout, h, *padded, saved2)):
        assert torch.equal(p, q)


def test_offsets_past_32_bits(dev):
    """Rows whose bytes pass 2^32: out and dh of the last ones as for those rows alone, and the
    gradients of the parameters, to which only they contribute."""
    H, M, n = 2816, 800_000, 700
    h, params, dout = base._link_inputs(dev, n, H, 950)
    hs, ds = (torch.zeros(M, H, dtype=BF, device=dev) for _ in range(2))
    hs[-n:], ds[-n:] = h, dout
    out, saved = _lib.hybridlink_train(hs, *params)
    got = _lib.hybridlink_backward(ds, hs, *params, saved)
    assert not got[0][:-n].any()
    _check((out[-n:], got[0][-n:], *got[1:]), expected(h, params, dout), "the last rows")
