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
