"""The differentiable forms as a program uses them."""
import pytest
import torch

import test_gpu_training as base
from hybridagent_amd import _lib, training

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert _lib.available(), "libw4a16moe.so must be built"
    return torch.device("cuda:0")


def _normal(dev, seed, *shape, std=1.0, mean=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std + mean).to(BF)


def _mlp(dev, T, H, I):
    return [_normal(dev, 1, T, H), _normal(dev, 2, I, H, std=H ** -0.5), _normal(dev, 3, I, H, std=H ** -0.5),
            _normal(dev, 4, H, I, std=I ** -0.5)]


def _link(dev, T, H):
    p = [_normal(dev, 5 + i, H, std=0.1, mean=1.0 if i in (0, 6) else 0.0) for i in range(8)]
    p[2], p[4] = _normal(dev, 7, H, H, std=H ** -0.5), _normal(dev, 9, H, H, std=H ** -0.5)
    return [_normal(dev, 4, T, H), *p]


@pytest.mark.parametrize("T", [3, 130])
@pytest.mark.parametrize("name", ["gated_mlp", "hybridlink", "layer_norm"])
def test_gradient_at_an_odd_address(dev, name, T):
    """The gradient that reaches a call is a slice of a concatenation's, two bytes past a multiple of
    16: the same gradients as from one at its own address (bit for bit where the sums' order does not
    depend on the address)."""
    H = 96
    args = {"gated_mlp": lambda: _mlp(dev, T, H, 64), "hybridlink": lambda: _link(dev, T, H),
            "layer_norm": lambda: [_normal(dev, 4, T, H), _normal(dev, 5, H), _normal(dev, 6, H)]}[name]()
    leaves = [t.requires_grad_() for t in args]
    y = getattr(training, name)(*leaves)
    flat = _normal(dev, 20, 1 + T * H)
    grad = flat[1:].view(T, H)
    assert grad.data_ptr() % 16 == 2
    want = torch.autograd.grad(y, leaves, grad.clone(), retain_graph=True)
    got = torch.autograd.grad(torch.cat([torch.zeros(1, dtype=BF, device=dev), y.flatten()]), leaves, flat)
    for p, q in zip(got, want):
        if name == "layer_norm":  # other loads, another order: a rounding and some of fp32's
            e = (p.double() - q.double()).abs()
            assert (e <= 2 * 2.0 ** -8 * q.double().abs() + 1e-4).all()
        else:
            assert torch.equal(p, q)


# the tiles of the input's gradient that the shapes of the other tests leave out
@pytest.mark.parametrize("T,H,I", [(1699, 1824, 32), (4105, 448, 32)])
def test_gated_mlp_more_tiles(dev, T, H, I):
    base.test_gated_mlp(dev, T, H, I)
