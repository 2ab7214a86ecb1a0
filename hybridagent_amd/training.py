"""Differentiable forms of the framework's dense maps, on the HIP library.

The reference trains HybridLink and the dense weights around the experts
through torch's autograd (hybrid_sft/train.py, hybrid_agent/hybridlink.py);
these are the same maps with hand-written backward passes:

* ``layer_norm``  nn.LayerNorm (hybridlink.py:20,23)
* ``gated_mlp``   the shared MLP of a decoder layer (backends.py:105-108)
* ``hybridlink``  HybridLink.forward (hybridlink.py:17-28), and ``HybridLink``,
  the module with the reference's parameter names
* ``head_norm_rope``, ``attention``  the attention half of a decoder layer
  (the installed model's attention, backends.py:173-196): the heads' norms with
  the position rotation, and attention over packed sequences

Each is one pair of library calls (``_lib.layer_norm`` and
``_lib.layer_norm_backward``, ...), differentiable once, in reverse mode.  Code that captures
a training step into a graph calls those pairs itself: the functions here
refuse to record a backward pass while the stream is capturing, and to run a
recorded one there.  Autograd adds up a leaf's gradients on the stream of the
first graph that used it; with such a graph alive, a backward pass captured on
another stream ends the process.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib


def _wants_grad(*tensors) -> bool:
    """Whether the call records a backward pass; refuses where it cannot, and forward-mode
    derivatives, which a library call would drop (a level of them is open for any to be there)."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("forward-mode derivatives are not supported: the gradients here are reverse-mode only")
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors):
        return False
    _refuse_capture()
    return True


def _refuse_capture() -> None:
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a differentiable call cannot be captured into a graph: call the forward and backward "
                           "functions of hybridagent_amd._lib in the captured code instead")


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _lib.layer_norm(x, weight, bias, eps, return_stats=True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias = bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture()
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = _lib.layer_norm_backward(dy, x, weight, mean, rstd, bias=ctx.bias)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension of bf16, fp16 or fp32 rows."""
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _lib.layer_norm(x, weight, bias, eps)


class _GatedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_w, up_w, down_w):
        y, saved = _lib.gated_mlp(x, gate_w, up_w, down_w, return_saved=True)
        ctx.save_for_backward(x, gate_w, up_w, down_w, saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture()
        return _lib.gated_mlp_backward(dy, *ctx.saved_tensors, needs=ctx.needs_input_grad)


def gated_mlp(x: torch.Tensor, gate_w: torch.Tensor, up_w: torch.Tensor, down_w: torch.Tensor) -> torch.Tensor:
    """(gelu_tanh(x gate_w^T) * (x up_w^T)) down_w^T on bf16 [..., H]."""
    if _wants_grad(x, gate_w, up_w, down_w):
        return _GatedMLP.apply(x, gate_w, up_w, down_w)
    return _lib.gated_mlp(x, gate_w, up_w, down_w)


class _HybridLink(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, eps, *params):
        out, saved = _lib.hybridlink_train(h, *params, eps)
        ctx.save_for_backward(h, *params, saved)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        _refuse_capture()
        h, *params, saved = ctx.saved_tensors
        dh, *grads = _lib.hybridlink_backward(dout, h, *params, saved)
        return (dh, None, *grads)


def hybridlink(h: torch.Tensor, ln1_w: torch.Tensor, ln1_b: torch.Tensor, p1_w: torch.Tensor, p1_b: torch.Tensor,
               p2_w: torch.Tensor, p2_b: torch.Tensor, ln2_w: torch.Tensor, ln2_b: torch.Tensor,
               eps: float = 1e-5) -> torch.Tensor:
    """HybridLink of bf16 [..., H]: with a backward pass where an argument wants a gradient, else
    the inference call (``_lib.hybridlink``; the two round their intermediates at different points)."""
    params = (ln1_w, ln1_b, p1_w, p1_b, p2_w, p2_b, ln2_w, ln2_b)
    if _wants_grad(h, *params):
        return _HybridLink.apply(h, eps, *params)
    return _lib.hybridlink(h, *params, eps)


def _constants(**tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} has no gradient here: detach it")


class _HeadNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_weight, k_weight, cos, sin, positions, eps):
        out = _lib.head_norm_rope(q, k, v, cos, sin, positions, q_weight, k_weight, eps)
        ctx.save_for_backward(q, k, v, cos, sin, positions, q_weight, k_weight)
        ctx.eps = eps
        return out if v is not None else out[:2]

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk, dv=None):
        _refuse_capture()
        weights = ctx.needs_input_grad[3] or ctx.needs_input_grad[4]
        grads = _lib.head_norm_rope_backward(dq, dk, dv, *ctx.saved_tensors, ctx.eps, weights=weights)
        return (*grads, None, None, None, None)


def head_norm_rope(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, cos: torch.Tensor | None,
                   sin: torch.Tensor | None, positions: torch.Tensor, q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, eps: float = 1e-6):
    """(q, k, v) with every head normed and q and k turned (``_lib.head_norm_rope``); cos and sin are
    constants."""
    if _wants_grad(q, k, v, q_weight, k_weight, cos, sin):
        _constants(cos=cos, sin=sin)
        out = _HeadNormRope.apply(q, k, v, q_weight, k_weight, cos, sin, positions, eps)
        return out if v is not None else (*out, None)
    return _lib.head_norm_rope(q, k, v, cos, sin, positions, q_weight, k_weight, eps)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale, causal, window):
        out, lse = _lib.attention(q, k, v, cu_q, cu_k, scale, causal, window, return_lse=True)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k)
        ctx.mask = scale, causal, window
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        _refuse_capture()
        grads = _lib.attention_backward(dout, *ctx.saved_tensors, *ctx.mask, needs=ctx.needs_input_grad[:3])
        return (*grads, None, None, None, None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor | None = None,
              scale: float | None = None, causal: bool = True, window: int = 0) -> torch.Tensor:
    """Attention over packed sequences (``_lib.attention``)."""
    if _wants_grad(q, k, v):
        return _Attention.apply(q, k, v, cu_q, cu_k, scale, causal, window)
    return _lib.attention(q, k, v, cu_q, cu_k, scale, causal, window)


def _weight_and_bias(m: nn.Module | None, name: str, kind: type):
    """m's parameters, all of m that is used: refuses what m's own call would do besides."""
    if not isinstance(m, kind) or type(m).forward is not kind.forward or "forward" in m.__dict__:
        raise ValueError(f"{name} must be an nn.{kind.__name__} with its own forward, got {type(m).__name__}: "
                         "HybridLink reads its weight and bias and does not call it")
    if m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks:
        raise ValueError(f"{name} has hooks, which would not run: HybridLink reads its weight and bias and does "
                         "not call it")
    weight, bias = m.weight, m.bias
    if weight is None or bias is None:
        raise ValueError(f"{name} must have a weight and a bias")
    return weight, bias


class HybridLink(nn.Module):
    """R(h) = post_ln(h + proj2(GELU(proj1(pre_ln(h))))) with the reference module's parameter names
    (hybridlink.py:17-28), so its state dict loads as it is.

    The submodules hold the parameters and are not called: adapters in their place, hooks on them
    and two norms of different eps are refused (a parametrization of a weight or bias works)."""

    def __init__(self, hidden_size: int, eps: float = 1e-5, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str | None = None) -> None:
        super().__init__()
        kw = {"dtype": dtype, "device": device}
        self.pre_ln = nn.LayerNorm(hidden_size, eps=eps, **kw)
        self.proj1 = nn.Linear(hidden_size, hidden_size, **kw)
        self.proj2 = nn.Linear(hidden_size, hidden_size, **kw)
        self.post_ln = nn.LayerNorm(hidden_size, eps=eps, **kw)

    def forward(self, h: torch.Tensor) -> torch.Tensor:
        mods = self._modules
        pre_ln, post_ln = mods["pre_ln"], mods["post_ln"]
        params = (*_weight_and_bias(pre_ln, "pre_ln", nn.LayerNorm),
                  *_weight_and_bias(mods["proj1"], "proj1", nn.Linear),
                  *_weight_and_bias(mods["proj2"], "proj2", nn.Linear),
                  *_weight_and_bias(post_ln, "post_ln", nn.LayerNorm))
        if pre_ln.eps != post_ln.eps:
            raise ValueError(f"pre_ln and post_ln must have one eps, got {pre_ln.eps} and {post_ln.eps}")
        return hybridlink(h, *params, pre_ln.eps)
