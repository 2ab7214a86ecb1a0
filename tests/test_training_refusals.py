"""What the differentiable forms refuse, on the CPU: the library's calls are stood in for by torch."""
import pytest
import torch
import torch.nn.functional as F
import torch.nn.utils.parametrize
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


# ---------------------------------------------------------------- the module reads its submodules' parameters


def _link():
    torch.manual_seed(2)
    return training.HybridLink(H, dtype=torch.float32)


class _Adapter(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


class _Wrapper(torch.nn.Module):
    def __init__(self, m):
        super().__init__()
        self.weight, self.bias = m.weight, m.bias


HOOKS = {"forward": lambda m: m.register_forward_hook(lambda *a: None),
         "forward_pre": lambda m: m.register_forward_pre_hook(lambda *a: None),
         "full_backward": lambda m: m.register_full_backward_hook(lambda *a: None),
         "full_backward_pre": lambda m: m.register_full_backward_pre_hook(lambda *a: None)}


@pytest.mark.parametrize("name", ["pre_ln", "proj1", "proj2", "post_ln"])
@pytest.mark.parametrize("hook", HOOKS)
def test_hooks_on_submodules_are_refused(calls, name, hook):
    link = _link()
    handle = HOOKS[hook](getattr(link, name))
    with torch.no_grad():
        with pytest.raises(ValueError, match=f"{name} has hooks"):
            link(torch.zeros(3, H))
        handle.remove()
        link(torch.zeros(3, H))
    assert calls == ["hybridlink"]


@pytest.mark.parametrize("name", ["pre_ln", "proj1", "proj2", "post_ln"])
def test_other_submodules_are_refused(calls, name):
    for swap in (lambda m: _Adapter(H, H), _Wrapper, lambda m: torch.nn.Identity()):
        link = _link()
        setattr(link, name, swap(getattr(link, name)))
        with pytest.raises(ValueError, match=f"{name} must be"):
            link(torch.zeros(3, H))
    link = _link()
    getattr(link, name).forward = lambda x: x
    with pytest.raises(ValueError, match=f"{name} must be"):
        link(torch.zeros(3, H))
    link = _link()
    getattr(link, name).bias = None
    with pytest.raises(ValueError, match="a weight and a bias"):
        link(torch.zeros(3, H))
    assert not calls


def test_one_eps(calls):
    link = _link()
    link.post_ln.eps = 1e-6
    with pytest.raises(ValueError, match="one eps"):
        link(torch.zeros(3, H))
    link.pre_ln.eps = 1e-6
    with torch.no_grad():
        link(torch.zeros(3, H))
    assert calls == ["hybridlink"]


def test_parametrized_weights_are_read(monkeypatch):
    """A parametrization is part of the weight that is read, and the module itself may have hooks."""
    class Twice(torch.nn.Module):
        def forward(self, w):
            return 2 * w

    link = _link()
    w = link.proj1.weight.detach().clone()
    torch.nn.utils.parametrize.register_parametrization(link.proj1, "weight", Twice())
    seen = []
    monkeypatch.setattr(_lib, "hybridlink", lambda h, *p: seen.append(p[2]) or h)
    link.register_forward_hook(lambda *a: seen.append("hook"))
    with torch.no_grad():
        link(torch.zeros(3, H))
    assert torch.equal(seen[0], 2 * w) and seen[1] == "hook"


# ---------------------------------------------------------------- captured graphs


@pytest.mark.parametrize("name", ["layer_norm", "gated_mlp", "hybridlink"])
def test_no_pass_of_a_recorded_step_is_captured(monkeypatch, name):
    """While the stream is capturing, neither a forward pass that records nor a recorded backward pass
    reaches the library; outside a capture both do."""
    args = [t.requires_grad_() for t in _tensors()[name]]
    reached = []
    forward, backward = {"layer_norm": ("layer_norm", "layer_norm_backward"),
                         "gated_mlp": ("gated_mlp", "gated_mlp_backward"),
                         "hybridlink": ("hybridlink_train", "hybridlink_backward")}[name]
    kept = (torch.zeros(3), torch.zeros(3)) if name == "layer_norm" else (torch.zeros(1),)

    def run_forward(x, *a, **kw):
        reached.append("forward")
        return (x.detach() * 1, *kept)

    def run_backward(*a, **kw):
        reached.append("backward")
        return tuple(torch.zeros_like(t) for t in args)

    monkeypatch.setattr(_lib, forward, run_forward)
    monkeypatch.setattr(_lib, backward, run_backward)
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    y = getattr(training, name)(*args)
    capturing[0] = True
    with pytest.raises(RuntimeError, match="cannot be captured"):
        y.sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="cannot be captured"):
        getattr(training, name)(*args)
    assert reached == ["forward"] and all(t.grad is None for t in args)
    capturing[0] = False
    y.sum().backward()
    assert reached == ["forward", "backward"] and all(t.grad is not None for t in args)
