"""Layer norm's backward pass at the edges of its numbers."""
import pytest
import torch

from hybridagent_amd import _lib

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    assert _lib.available(), "libw4a16moe.so must be built"
    return torch.device("cuda:0")


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H", [39, 40, 72, 200])
@pytest.mark.parametrize("M", [3, 600], ids=["workgroup", "wavefront"])
def test_constant_rows_whose_mean_over_the_deviation_overflows(dev, M, H, dt):
    """Rows of 2^120: their sums are exact, x - mean is 0, rstd is eps^-1/2 = 316, and mean rstd is
    past fp32.  xh is 0 all along the row, so dx = rstd (g - mean g) and dw = 0.  A sum of H terms is
    off by (H + 8) 2^-24 of its terms' sizes at most, dx's own rounding by half a step."""
    g = torch.Generator(device=dev).manual_seed(M + H)
    x = torch.full((M, H), 2.0 ** 120, device=dev).to(dt)
    w, dy = (torch.randn(*s, generator=g, device=dev).to(dt) for s in ((H,), (M, H)))
    _, mean, rstd = _lib.layer_norm(x, w, w, return_stats=True)
    assert (mean == 2.0 ** 120).all() and torch.isinf(mean * rstd).all()
    dx, dw, db = _lib.layer_norm_backward(dy, x, w, mean, rstd)
    p = dy.double() * w.double()
    r = rstd.double()[:, None]
    want = r * (p - p.mean(-1, keepdim=True))
    tol = torch.finfo(dt).eps / 2 * want.abs() + (H + 8) * E32 * r * (p.abs() + p.abs().mean(-1, keepdim=True))
    assert ((dx.double() - want).abs() <= tol).all()
    assert not dw.any()
    wb, n = dy.double().sum(0), (M + 8) * E32 * dy.double().abs().sum(0)
    assert ((db.double() - wb).abs() <= torch.finfo(dt).eps / 2 * wb.abs() + n).all()
