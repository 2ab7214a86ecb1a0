"""The bits that HybridLink's training form keeps, on inputs whose intermediates are known.

With one row the gradients of the linears' biases are the rows that the products take:
dp2_b is dr and dp1_b is dz, as bf16, so that each step of the backward pass can be
checked by itself, element by element, against its formula in 64 bits.  A rounding to
bf16 moves a value by at most U = 2^-8 of it; fp32 arithmetic is bounded where it is used."""
import pytest
import torch

from hybridagent_amd import _lib

pytestmark = pytest.mark.gpu

U, E32 = 2.0 ** -8, 2.0 ** -24
BF = torch.bfloat16
SQ2 = 2.0 ** 0.5


@pytest.fixture(scope="module")
def dev():
    assert _lib.available(), "libw4a16moe.so must be built"
    return torch.device("cuda:0")


def _normal(dev, seed, *shape, std=1.0, mean=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std + mean).to(BF)


def _within(got, want, tol, what):
    d = (got.double() - want).abs()
    print(f"{what}: worst {float((d / tol.clamp_min(1e-300)).max()):.3f} of the tolerance", flush=True)
    assert (d <= tol).all(), f"{what}: {int((d > tol).sum())} of {d.numel()} beyond the tolerance"


def _phi(z):
    return torch.exp(-0.5 * z * z) / (2.0 * torch.pi) ** 0.5


def _cdf(z):
    return 0.5 * torch.special.erfc(-z / SQ2)


@pytest.mark.parametrize("reps", [1, 3, 80], ids=["stream", "several rows", "tiles"])
def test_exact_gelu_and_its_slope(dev, reps):
    """gelu(z) and its slope far into the tails.  With pre_ln's parameters zero z is proj1's bias,
    exactly; with proj2 the identity dg is dr.  dp2_w[i, j] = dr_i g_j has the rounding of g and its
    own; the tail's exponential may be off by 2^-15 of itself (|z| <= 12).  All rows are the same, so
    their sums are those of one row (exact: times a power of two, or fp32 sums)."""
    H = 512
    z = torch.linspace(-12, 12, H, device=dev).to(BF)
    zero, eye = torch.zeros(H, dtype=BF, device=dev), torch.eye(H, dtype=BF, device=dev)
    h = _normal(dev, 1, 1, H).expand(reps, H).contiguous()
    dout = _normal(dev, 2, 1, H).expand(reps, H).contiguous()
    one = torch.ones(H, dtype=BF, device=dev)
    params = [zero, zero, eye, z, eye, zero, one, zero]
    _, saved = _lib.hybridlink_train(h, *params)
    grads = _lib.hybridlink_backward(dout, h, *params, saved)
    one_row = _lib.hybridlink_backward(dout[:1], h[:1], *params, _lib.hybridlink_train(h[:1], *params)[1])
    dr, dz, dp2_w = one_row[6].double(), grads[4].double() / reps, grads[5].double() / reps
    z = z.double()
    want = dr[:, None] * (z * _cdf(z))
    _within(dp2_w, want, (2 * U + U * U + 2.0 ** -15 + 8 * reps * E32) * want.abs(), "dr x gelu(z)")
    # the slope Phi + z phi: each term's 2^-15, and the result's roundings (dz's, the sum's)
    want = dr * (_cdf(z) + z * _phi(z))
    tol = (2 * U + U * U + 8 * reps * E32) * want.abs() + 2.0 ** -15 * dr.abs() * (_cdf(z) + (z * _phi(z)).abs())
    _within(dz, want, tol, "dr x gelu'(z)")


# ---------------------------------------------------------------- what stays in 32 bits

H = 256


def _signs(dev):
    """A row of as many 1 as -1: its mean is 0 and its variance 1, exactly; with eps = 0 rstd is 1."""
    p = torch.randperm(H, generator=torch.Generator(device=dev).manual_seed(5), device=dev)
    return torch.where(p < H // 2, 1.0, -1.0)[None].to(BF)


def _step(h, params, dout, eps):
    out, saved = _lib.hybridlink_train(h, *params, eps)
    return out, _lib.hybridlink_backward(dout, h, *params, saved)


def _f32(p, q):
    """fp32's share in the sums of p q^T."""
    return 64 * E32 * (p.abs() @ q.abs().t())


def test_slope_of_the_unrounded_z(dev):
    """dz = (dr W2) gelu'(z), rounded once: z itself is not rounded (near the slope's zero a rounded z
    costs more than dz's own rounding)."""
    h = _signs(dev)
    w1, b1, p1, q1, p2, q2 = (_normal(dev, 10 + i, *s, std=std) for i, (s, std) in enumerate(
        [((H,), 0.5), ((H,), 0.5), ((H, H), 0.06), ((H,), 0.5), ((H, H), 0.06), ((H,), 0.5)]))
    one, zero = torch.ones(H, dtype=BF, device=dev), torch.zeros(H, dtype=BF, device=dev)
    _, grads = _step(h, [w1, b1, p1, q1, p2, q2, one, zero], _normal(dev, 17, 1, H), 0.0)
    a = (h.float() * w1.float() + b1.float()).to(BF).double()
    z = a @ p1.double().t() + q1.double()
    dr = grads[6].double()[None]
    dg = dr @ p2.double()
    slope = _cdf(z) + z * _phi(z)
    want = dg * slope
    tol = U * want.abs() + _f32(dr, p2.double().t()) * slope.abs() \
        + dg.abs() * ((_phi(z) * (2 - z * z)).abs() * _f32(a, p1.double()) + 2.0 ** -20)
    _within(grads[4][None], want, tol, "dz")


def test_gradient_of_h_is_rounded_once(dev):
    """dh = dr + LN'(da), rounded once: neither the residual's dr nor da is rounded before.  z is exact
    here (a in quarters, W1 in 64ths) and past where gelu is the identity, so g is z rounded; W2 has
    sixteen values a row, which keeps fp32's share in r small."""
    h = _signs(dev)
    g = torch.Generator(device=dev).manual_seed(20)
    at = lambda *s: torch.randint(-4, 5, s, generator=g, device=dev)
    b1, p1 = (at(H) / 4).to(BF), (at(H, H) / 64).to(BF)
    p2 = torch.zeros(H, H, device=dev)
    p2.scatter_(1, torch.rand(H, H, generator=g, device=dev).argsort(1)[:, :16], 0.2)
    p2 = (p2 * torch.randn(H, H, generator=g, device=dev)).to(BF)
    one, zero = torch.ones(H, dtype=BF, device=dev), torch.zeros(H, dtype=BF, device=dev)
    q1 = torch.full((H,), 18.0, dtype=BF, device=dev)
    dout = _normal(dev, 21, 1, H)
    _, grads = _step(h, [one, b1, p1, q1, p2, zero, one, zero], dout, 0.0)
    a = h.double() + b1.double()
    z = a @ p1.double().t() + 18
    assert z.min() > 13.5
    gz = z.to(BF).double()
    r = h.double() + gz @ p2.double().t()
    er = _f32(gz, p2.double()).max()
    rstd = r.var(unbiased=False) ** -0.5
    xh, d = (r - r.mean()) * rstd, dout.double()
    dr = rstd * (d - d.mean() - xh * (d * xh).mean())
    edr = 8 * rstd * er * dr.abs().max() + 64 * E32 * rstd * d.abs().max()
    dz = grads[4].double()[None]
    da, x1 = dz @ p1.double(), h.double()
    want = dr + da - da.mean() - x1 * (da * x1).mean()
    tol = U * want.abs() + edr + 3 * _f32(dz, p1.double().t()).max() + 64 * E32 * da.abs().max()
    _within(grads[0], want, tol, "dh")


def test_rows_far_from_zero(dev):
    """r = h + proj2(g) is normalised as it is: rounded to bf16 beside an h of 128 it would lose all of
    proj2.  pre_ln of a constant row gives its bias, exactly; the roundings of g, independent, stay
    within eight of their sums' standard deviations, and post_ln passes at most 2 + |xh| of it on."""
    T = 5
    h = torch.full((T, H), 128.0, dtype=BF, device=dev)
    a = _normal(dev, 30, H)
    p1, q1, p2, q2 = (_normal(dev, 31 + i, *s, std=std) for i, (s, std) in enumerate(
        [((H, H), 0.06), ((H,), 0.5), ((H, H), 0.06), ((H,), 0.5)]))
    one, zero = torch.ones(H, dtype=BF, device=dev), torch.zeros(H, dtype=BF, device=dev)
    out, _ = _step(h, [one, a, p1, q1, p2, q2, one, zero], _normal(dev, 36, T, H), 1e-5)
    z = a.double()[None] @ p1.double().t() + q1.double()
    g = z * _cdf(z)
    r = 128 + g @ p2.double().t() + q2.double()
    er = (8 / 3 ** 0.5 * ((U * g) ** 2 @ (p2.double().t() ** 2)).sqrt()).max() + _f32(g, p2.double()).max() + 128 * 4 * E32
    rstd = (r.var(unbiased=False) + 1e-5) ** -0.5
    xh = (r - r.mean()) * rstd
    _within(out, xh.expand(T, H), U * xh.abs() + rstd * er * (2 + xh.abs()), "out")
