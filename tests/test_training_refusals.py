"""What the differentiable forms refuse, on the CPU: the library's calls are stood in for by torch."""
import pytest
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from hybridagent_amd import _lib, training

H, I = 64, 96


def _tensors():
    g = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=g)
    return {"layer_norm": [n(3, H), n(H), n(H)],
            "gated_mlp": [n(3, H), n(I, H), n(I, H), n(H, I)],
            "hybridlink": [n(3, H), n(H), n(H), n(H, H), n(H), n(H, H), n(H), n(H), n(H)]}


@pytest.fixture
def calls(monkeypatch):
    """The library's forward calls, as torch: what they get is counted."""
    got = []

    def stand_in(name, f):
        def call(*args, **kw):
            got.append(name)
            return f(*args)
        monkeypatch.setattr(_lib, name, call)

    stand_in("layer_norm", lambda x, w, b, eps: F.layer_norm(x.detach(), w.shape, w.detach(), b.detach(), eps))
    stand_in("gated_mlp", lambda x, *w: x.detach() * 1)
    stand_in("hybridlink", lambda h, *p: h.detach() * 1)
    return got


@pytest.mark.parametrize("name", ["layer_norm", "gated_mlp", "hybridlink"])
def test_forward_mode_derivatives(calls, name):
    """A tangent on any argument is refused, with gradients enabled or not; without one the calls go on,
    inside a level of forward-mode differentiation too."""
    f, args = getattr(training, name), _tensors()[name]
    with forward_ad.dual_level():
        assert f(*args).shape == args[0].shape
        for i in range(len(args)):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                f(*dual)
    assert calls == [name]
    assert f(*args).shape == args[0].shape
