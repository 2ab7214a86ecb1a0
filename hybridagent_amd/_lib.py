"""ctypes binding of libw4a16moe.so (the C ABI declared in include/w4a16moe.h).

Tensors stay owned by PyTorch: this module checks device / dtype / shape /
contiguity, allocates outputs and workspaces through torch's caching
allocator, passes raw device pointers plus ``torch.cuda.current_stream()``,
and maps non-zero status codes to ``ValueError`` (bad arguments) or
``RuntimeError`` (launch failures).  There is no CPU fallback: every entry
point requires CUDA (HIP) tensors and the built library, and raises if
either is missing.
"""
from __future__ import annotations

import ctypes
import os
import threading
import warnings
import weakref
from dataclasses import dataclass
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "libw4a16moe.so"

W4A16_OK = 0
_STATUS_EXC = {1: ValueError, 2: ValueError, 3: ValueError, 4: ValueError, 5: ValueError,
               6: RuntimeError}

# kinds of tiled weight copies (enum w4a16_tiled_kind)
TILED_GATE_UP_DECODE, TILED_DOWN_DECODE, TILED_GATE_UP_PREFILL, TILED_DOWN_PREFILL = 0, 1, 2, 3


class TiledExpertsC(ctypes.Structure):
    """struct w4a16_tiled_experts: the tiled copies of one expert stack and its shape."""
    _fields_ = [("E", ctypes.c_int64), ("H", ctypes.c_int64), ("I", ctypes.c_int64),
                ("group_size", ctypes.c_int64),
                ("gu_decode", ctypes.c_void_p), ("gu_decode_bytes", ctypes.c_size_t),
                ("dn_decode", ctypes.c_void_p), ("dn_decode_bytes", ctypes.c_size_t),
                ("gu_prefill", ctypes.c_void_p), ("gu_prefill_bytes", ctypes.c_size_t),
                ("dn_prefill", ctypes.c_void_p), ("dn_prefill_bytes", ctypes.c_size_t)]


# name -> (restype, argtypes); the exact set declared in include/w4a16moe.h
_VP, _I64, _SZ, _F32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float
_TP = ctypes.POINTER(TiledExpertsC)
_HEADS = (_VP, _I64, _I64)  # [tokens, heads, D]: the pointer, elements between tokens and between heads
SIGNATURES = {
    "w4a16moe_version": (ctypes.c_int, []),
    "w4a16moe_status_string": (ctypes.c_char_p, [ctypes.c_int]),
    "w4a16_dequantize": (ctypes.c_int, [_VP, _VP, _VP, _I64, _I64, _I64, _VP]),
    "w4a16_linear_workspace_bytes": (_SZ, [_I64, _I64, _I64]),
    "w4a16_add_rms_norm": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _I64, _I64, _F32, _VP]),
    "w4a16_linear": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "w4a16_hybridlink_workspace_bytes": (_SZ, [_I64, _I64]),
    "w4a16_hybridlink": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _I64, _I64,
                                        _F32, _VP, _SZ, _VP]),
    "moe_router_workspace_bytes": (_SZ, [_I64, _I64, _I64]),
    "moe_router_topk": (ctypes.c_int, [_VP, _VP, _F32, _VP, _VP, _F32, _I64, _I64, _I64, _I64,
                                       _VP, _VP, _VP, _VP, _SZ, _VP]),
    "moe_topk_from_logits": (ctypes.c_int, [_VP, _VP, _I64, _I64, _I64, _VP, _VP, _VP]),
    "moe_sort_workspace_bytes": (_SZ, [_I64, _I64, _I64]),
    "moe_sort_permute": (ctypes.c_int, [_VP, _I64, _I64, _I64, _VP, _VP, _VP, _SZ, _VP]),
    "moe_workspace_bytes": (_SZ, [_I64, _I64, _I64, _I64, _I64]),
    "moe_forward": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _I64, _I64, _I64, _I64,
                                   _I64, _I64, _VP, _SZ, _VP]),
    "moe_forward_static": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _I64, _I64, _I64, _I64,
                                          _I64, _I64, _VP]),
    "moe_plan": (ctypes.c_int, [_VP, _VP, _I64, _I64, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_gate_up": (ctypes.c_int, [_VP, _VP, _VP, _I64, _I64, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_down": (ctypes.c_int, [_VP, _VP, _I64, _I64, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_combine": (ctypes.c_int, [_VP, _VP, _VP, _I64, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_layer_workspace_bytes": (_SZ, [_I64, _I64, _I64, _I64, _I64]),
    "moe_bf16_experts_workspace_bytes": (_SZ, [_I64, _I64, _I64, _I64, _I64]),
    "moe_bf16_experts_forward": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _I64, _I64, _I64, _I64, _I64,
                                                _VP, _SZ, _VP]),
    "moe_ffn_block_workspace_bytes": (_SZ, [_I64, _I64, _I64, _I64, _I64, _I64]),
    "moe_ffn_block_forward": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _F32, _VP, _VP, _VP,
                                             _VP, _VP, _VP, _VP, _VP, _VP, _VP, _F32, _VP, _I64, _I64, _I64,
                                             _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_layer_forward": (ctypes.c_int, [_VP, _VP, _F32, _VP, _VP, _F32, _VP, _VP, _VP, _VP, _VP, _VP,
                                         _VP, _VP, _I64, _I64, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "w4a16_tiled_bytes": (_SZ, [ctypes.c_int, _I64, _I64, _I64, _I64]),
    "w4a16_tile": (ctypes.c_int, [ctypes.c_int, _VP, _VP, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_gate_up_tiled": (ctypes.c_int, [_VP, _VP, _VP, _TP, _I64, _I64, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_down_tiled": (ctypes.c_int, [_VP, _VP, _TP, _I64, _I64, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_forward_tiled": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _TP, _VP, _I64, _I64, _I64, _I64, _I64,
                                         _I64, _VP, _SZ, _VP]),
    "moe_layer_forward_tiled": (ctypes.c_int, [_VP, _VP, _F32, _VP, _VP, _F32, _VP, _VP, _VP, _VP, _VP, _TP,
                                               _VP, _VP, _VP, _I64, _I64, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_layer_forward_add_norm": (ctypes.c_int, [_VP, _VP, _F32, _VP, _VP, _F32, _VP, _VP, _VP, _VP, _VP, _TP,
                                                  _VP, _VP, _VP, _VP, _F32, _VP, _VP, _I64, _I64, _I64, _I64, _I64,
                                                  _I64, _VP, _SZ, _VP]),
    "moe_ffn_block_forward_tiled": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _F32, _VP, _VP,
                                                   _VP, _VP, _VP, _VP, _VP, _TP, _VP, _VP, _VP, _F32, _VP, _I64,
                                                   _I64, _I64, _I64, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "moe_ffn_block_routing_offsets": (ctypes.c_int, [_I64, _I64, _I64, _I64, _I64, _I64,
                                                     ctypes.POINTER(_SZ), ctypes.POINTER(_SZ)]),
    "w4a16_layer_norm": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_int, _I64, _I64, _F32, _VP]),
    "w4a16_layer_norm_backward_workspace_bytes": (_SZ, [_I64, _I64]),
    "w4a16_layer_norm_backward": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_int, _I64, _I64,
                                                 _VP, _SZ, _VP]),
    "w4a16_gated_mlp_workspace_bytes": (_SZ, [_I64, _I64, _I64]),
    "w4a16_gated_mlp_saved_bytes": (_SZ, [_I64, _I64]),
    "w4a16_gated_mlp": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _SZ, _I64, _I64, _I64, _VP, _SZ, _VP]),
    "w4a16_gated_mlp_backward_workspace_bytes": (_SZ, [_I64, _I64, _I64]),
    "w4a16_gated_mlp_backward": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _SZ, _VP, _VP, _VP, _VP, _I64, _I64,
                                                _I64, _VP, _SZ, _VP]),
    "w4a16_hybridlink_saved_bytes": (_SZ, [_I64, _I64]),
    "w4a16_hybridlink_train_workspace_bytes": (_SZ, [_I64, _I64]),
    "w4a16_hybridlink_train": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _SZ, _I64, _I64,
                                              _F32, _VP, _SZ, _VP]),
    "w4a16_hybridlink_backward_workspace_bytes": (_SZ, [_I64, _I64]),
    "w4a16_hybridlink_backward": (ctypes.c_int, [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _SZ, _VP, _VP, _VP, _VP, _VP, _VP,
                                                 _VP, _VP, _VP, _I64, _I64, _VP, _SZ, _VP]),
    "w4a16_head_norm_rope": (ctypes.c_int, [*_HEADS * 3, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, ctypes.c_int,
                                            *[_I64] * 6, _F32, _VP]),
    "w4a16_head_norm_rope_backward_workspace_bytes": (_SZ, [_I64] * 4),
    "w4a16_head_norm_rope_backward": (ctypes.c_int, [_VP, _VP, _VP, *_HEADS * 3, *[_VP] * 10, ctypes.c_int,
                                                     *[_I64] * 6, _F32, _VP, _SZ, _VP]),
    "w4a16_append_kv": (ctypes.c_int, [*_HEADS * 3, *[_VP] * 10, _I64, _VP, _I64, ctypes.c_int, ctypes.c_int,
                                       *[_I64] * 8, _F32, _VP]),
    "w4a16_attention_workspace_bytes": (_SZ, [_I64] * 7),
    "w4a16_attention": (ctypes.c_int, [*_HEADS * 3, _VP, _VP, _VP, _VP, ctypes.c_int, *[_I64] * 6, _F32,
                                       ctypes.c_int, _I64, _VP, _SZ, _VP]),
    "w4a16_attention_backward_workspace_bytes": (_SZ, [_I64] * 7),
    "w4a16_attention_backward": (ctypes.c_int, [_VP, *_HEADS * 3, *[_VP] * 7, ctypes.c_int, *[_I64] * 6, _F32,
                                                ctypes.c_int, _I64, _VP, _SZ, _VP]),
    "w4a16_decode_attention_workspace_bytes": (_SZ, [_I64] * 5),
    "w4a16_decode_attention": (ctypes.c_int, [*_HEADS, _VP, _I64, _VP, _I64, _VP, _VP, _VP, ctypes.c_int,
                                              *[_I64] * 7, _F32, _I64, _VP, _SZ, _VP]),
}

_lib = None


def load(path: os.PathLike | str | None = None) -> ctypes.CDLL:
    """Load (once) and return the library; raise if it has not been built."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path is not None else LIB_PATH
    if not p.exists():
        raise RuntimeError(
            f"{p} not found: the W4A16 MoE HIP library is not built "
            "(run `python -m hybridagent_amd.build`); there is no fallback path")
    lib = ctypes.CDLL(str(p))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if path is None:
        _lib = lib
    return lib


def available() -> bool:
    """True when the library file exists and loads."""
    try:
        load()
        return True
    except (RuntimeError, OSError):
        return False


def status_string(status: int) -> str:
    return load().w4a16moe_status_string(status).decode()


def _check(status: int, what: str) -> None:
    if status != W4A16_OK:
        exc = _STATUS_EXC.get(status, RuntimeError)
        raise exc(f"{what}: {status_string(status)} (status {status})")


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# The current device and its current stream's handle without a context manager
# and a Stream object per call (what torch's own generated code uses): 0.2 us
# against 3.2 us, on calls of 6-30 us.
_get_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _raw_stream = torch._C._cuda_getCurrentRawStream
else:
    def _raw_stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


def _stream(device: torch.device) -> int:
    return _raw_stream(device.index if device.index is not None else _get_device())


def _call(what: str, dev: torch.device, fn, *args) -> None:
    """fn(*args, the current stream of dev), run with dev current."""
    index = dev.index
    if _get_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _raw_stream(index))
    if status != W4A16_OK:
        _check(status, what)


def _require_gpu(*tensors: torch.Tensor) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        d = t.device
        if d == dev:
            continue
        if d.type != "cuda":
            raise RuntimeError(
                "hybridagent_amd W4A16 kernels run on the GPU only (got a CPU tensor); "
                "there is no CPU fallback")
        if dev is not None:
            raise ValueError(f"tensors on different devices: {dev} vs {d}")
        dev = d
    return dev


def _bf16(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    return t.contiguous()


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """t as a matrix of rows of `width` (t itself if it is one)."""
    return t if t.dim() == 2 and t.shape[1] == width else t.reshape(-1, width)


def _like(out: torch.Tensor, shape) -> torch.Tensor:
    """out in the leading shape of the call's rows (out itself for a matrix)."""
    return out if len(shape) == 2 else out.reshape(shape)


def _i32(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32, got {t.dtype}")
    return t.contiguous()


def _workspace(nbytes: int, device) -> torch.Tensor | None:
    if nbytes == 0:
        return None
    return torch.empty((nbytes,), dtype=torch.uint8, device=device)


def infer_group_size(K: int, n_groups: int) -> int:
    """Group size G (power of two >= 32) with ceil(K / G) == n_groups."""
    if n_groups <= 0:
        raise ValueError("scale has no groups")
    if n_groups == 1:
        g = 32
        while g < K:
            g *= 2
        return g
    g = 32
    while g <= K:
        if -(-K // g) == n_groups:
            return g
        g *= 2
    raise ValueError(f"no power-of-two group size gives ceil({K}/G) == {n_groups}")


# --------------------------------------------------------------------------- ops

def dequantize(packed: torch.Tensor, scale: torch.Tensor, group_size: int | None = None) -> torch.Tensor:
    """bf16 [..., N, K] = bf16_RNE(q * s)   (quantization.py:132-137)."""
    dev = _require_gpu(packed, scale)
    packed = _i32(packed, "packed")
    scale = _bf16(scale, "scale")
    K = packed.shape[-1] * 8
    if scale.shape[:-1] != packed.shape[:-1]:
        raise ValueError(f"scale leading shape {tuple(scale.shape)} does not match packed {tuple(packed.shape)}")
    G = group_size or infer_group_size(K, scale.shape[-1])
    if scale.shape[-1] != -(-K // G):
        raise ValueError(f"scale has {scale.shape[-1]} groups, expected ceil({K}/{G})")
    out = torch.empty((*packed.shape[:-1], K), dtype=torch.bfloat16, device=dev)
    rows = packed.numel() // max(1, packed.shape[-1])
    _call("w4a16_dequantize", dev, load().w4a16_dequantize, _ptr(packed), _ptr(scale), _ptr(out), rows, K, G)
    return out


def add_rms_norm(h: torch.Tensor, weight: torch.Tensor, eps: float,
                 delta: torch.Tensor | None = None):
    """(x, y): x = bf16(h + delta) (h itself without delta), y = RMSNorm(x) * weight in fp32,
    rounded to bf16 (TF:modeling_gemma4.py:197-215); h, delta [..., H] bf16."""
    dev = _require_gpu(h, weight, delta)
    h = _bf16(h, "h")
    weight = _bf16(weight, "weight")
    H = h.shape[-1]
    if weight.shape != (H,):
        raise ValueError(f"weight must be [{H}]")
    h2 = _rows(h, H)
    d2 = None
    if delta is not None:
        d2 = _rows(_bf16(delta, "delta"), H)
        if d2.shape != h2.shape:
            raise ValueError("delta must have the shape of h")
    M = h2.shape[0]
    y = torch.empty_like(h2)
    x = torch.empty_like(h2) if d2 is not None else h2
    _call("w4a16_add_rms_norm", dev, load().w4a16_add_rms_norm, _ptr(h2), _ptr(d2), _ptr(weight),
          _ptr(x) if d2 is not None else None, _ptr(y), M, H, float(eps))
    return x.reshape(h.shape), _like(y, h.shape)


def hybridlink(h: torch.Tensor, ln1_w: torch.Tensor, ln1_b: torch.Tensor, p1_w: torch.Tensor,
               p1_b: torch.Tensor, p2_w: torch.Tensor, p2_b: torch.Tensor, ln2_w: torch.Tensor,
               ln2_b: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """HybridLink R(h) = post_ln(h + proj2(GELU(proj1(pre_ln(h)))))  (hybridlink.py:17-28);
    h [..., H] bf16, LayerNorm/Linear parameters bf16 in the nn.Module layout."""
    params = (ln1_w, ln1_b, p1_w, p1_b, p2_w, p2_b, ln2_w, ln2_b)
    dev = _require_gpu(h, *params)
    h = _bf16(h, "h")
    H = h.shape[-1]
    names = ("pre_ln weight", "pre_ln bias", "proj1 weight", "proj1 bias", "proj2 weight",
             "proj2 bias", "post_ln weight", "post_ln bias")
    params = tuple(_bf16(p, n) for p, n in zip(params, names))
    for i, p in enumerate(params):
        want = (H, H) if i == 2 or i == 4 else (H,)
        if p.shape != want:
            raise ValueError(f"{names[i]} must be {list(want)}, got {list(p.shape)}")
    h2 = _rows(h, H)
    B = h2.shape[0]
    out = torch.empty_like(h2)
    lib = load()
    nbytes = lib.w4a16_hybridlink_workspace_bytes(B, H)
    ws = _workspace(nbytes, dev)
    _call("w4a16_hybridlink", dev, lib.w4a16_hybridlink, _ptr(h2), *[_ptr(p) for p in params], _ptr(out), B, H,
          float(eps), _ptr(ws), nbytes)
    return _like(out, h.shape)


def linear(x: torch.Tensor, w_packed: torch.Tensor, w_scale: torch.Tensor,
           bias: torch.Tensor | None = None, group_size: int | None = None) -> torch.Tensor:
    """y = x @ dequant(W)^T (+ bias)   (quantization.py:171-175); x [..., K] bf16."""
    dev = _require_gpu(x, w_packed, w_scale, bias)
    x = _bf16(x, "x")
    w_packed = _i32(w_packed, "weight_packed")
    w_scale = _bf16(w_scale, "weight_scale")
    if bias is not None:
        bias = _bf16(bias, "bias")
    N, K8 = w_packed.shape
    K = K8 * 8
    if x.shape[-1] != K:
        raise ValueError(f"x has {x.shape[-1]} features, weight expects {K}")
    if w_scale.shape[0] != N:
        raise ValueError("weight_scale rows do not match weight_packed")
    G = group_size or infer_group_size(K, w_scale.shape[-1])
    if w_scale.shape[-1] != -(-K // G):
        raise ValueError(f"weight_scale has {w_scale.shape[-1]} groups, expected ceil({K}/{G})")
    x2 = _rows(x, K)
    M = x2.shape[0]
    y = torch.empty((M, N), dtype=torch.bfloat16, device=dev)
    lib = load()
    nbytes = lib.w4a16_linear_workspace_bytes(M, K, G)
    ws = _workspace(nbytes, dev)
    _call("w4a16_linear", dev, lib.w4a16_linear, _ptr(x2), _ptr(w_packed), _ptr(w_scale), _ptr(bias), _ptr(y), M, N,
          K, G, _ptr(ws), nbytes)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], N)


def router_topk(hidden: torch.Tensor, router_scale: torch.Tensor, scalar_root: float,
                proj_w: torch.Tensor, per_expert_scale: torch.Tensor, eps: float, top_k: int,
                return_logits: bool = False):
    """Router of backends.py:111-117 -> (top_k_weights fp32, top_k_index int64[, logits bf16])."""
    dev = _require_gpu(hidden, router_scale, proj_w, per_expert_scale)
    H = hidden.shape[-1]
    h2 = _rows(_bf16(hidden, "hidden"), H)
    router_scale = _bf16(router_scale, "router scale")
    proj_w = _bf16(proj_w, "router proj weight")
    per_expert_scale = _bf16(per_expert_scale, "per_expert_scale")
    E = proj_w.shape[0]
    if proj_w.shape[1] != H or router_scale.numel() != H or per_expert_scale.numel() != E:
        raise ValueError("router parameter shapes do not match hidden size / expert count")
    M = h2.shape[0]
    idx = torch.empty((M, top_k), dtype=torch.int64, device=dev)
    w = torch.empty((M, top_k), dtype=torch.float32, device=dev)
    logits = torch.empty((M, E), dtype=torch.bfloat16, device=dev) if return_logits else None
    lib = load()
    nbytes = lib.moe_router_workspace_bytes(M, H, E)
    ws = _workspace(nbytes, dev)
    _call("moe_router_topk", dev, lib.moe_router_topk, _ptr(h2), _ptr(router_scale), float(scalar_root), _ptr(proj_w),
          _ptr(per_expert_scale), float(eps), M, H, E, top_k, _ptr(logits), _ptr(idx), _ptr(w), _ptr(ws), nbytes)
    if return_logits:
        return w, idx, logits
    return w, idx


def topk_from_logits(logits: torch.Tensor, per_expert_scale: torch.Tensor, top_k: int):
    """softmax/top-k/renormalise/per-expert scale on given bf16 logits [M, E]."""
    dev = _require_gpu(logits, per_expert_scale)
    logits = _bf16(logits, "logits")
    per_expert_scale = _bf16(per_expert_scale, "per_expert_scale")
    M, E = logits.shape
    idx = torch.empty((M, top_k), dtype=torch.int64, device=dev)
    w = torch.empty((M, top_k), dtype=torch.float32, device=dev)
    _call("moe_topk_from_logits", dev, load().moe_topk_from_logits, _ptr(logits), _ptr(per_expert_scale), M, E, top_k,
          _ptr(idx), _ptr(w))
    return w, idx


def sort_permute(top_k_index: torch.Tensor, num_experts: int):
    """(sorted_pos int32 [M*k], expert_offsets int32 [E+1])   (quantization.py:266-276)."""
    dev = _require_gpu(top_k_index)
    idx = top_k_index.to(torch.int64).contiguous()
    M, k = idx.shape
    sorted_pos = torch.empty(M * k, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    lib = load()
    nbytes = lib.moe_sort_workspace_bytes(max(M, 1), k, num_experts)
    ws = _workspace(nbytes, dev)
    _call("moe_sort_permute", dev, lib.moe_sort_permute, _ptr(idx), M, k, num_experts, _ptr(sorted_pos), _ptr(offsets),
          _ptr(ws), nbytes)
    return sorted_pos, offsets


def _routing(idx: torch.Tensor, w: torch.Tensor, rows: int):
    """(top_k_index int64, top_k_weights fp32), [rows, k] each, contiguous."""
    # explicit widths: reshape(0, -1) is ambiguous for an empty batch
    if idx.dim() != 2 or idx.shape[0] != rows:
        idx = idx.reshape(rows, idx.shape[-1])
    if w.dim() != 2 or w.shape[0] != rows:
        w = w.reshape(rows, w.shape[-1])
    if idx.dtype != torch.int64:
        idx = idx.to(torch.int64)
    if w.dtype != torch.float32:
        w = w.to(torch.float32)
    if w.shape != idx.shape:
        raise ValueError("top_k_weights and top_k_index shapes differ")
    return idx.contiguous(), w.contiguous()


def moe_forward(hidden_states: torch.Tensor, top_k_index: torch.Tensor, top_k_weights: torch.Tensor,
                gu_packed: torch.Tensor, gu_scale: torch.Tensor, dn_packed: torch.Tensor,
                dn_scale: torch.Tensor, group_size: int | None = None, *, tiles="auto") -> torch.Tensor:
    """W4A16 MoE layer output [T, H] bf16  (quantization.py:88-129).  ``tiles``: the
    stack's tiled weight copies (a TiledWeights), None for none, or "auto" for the
    ones registered for these tensors (register_tiles)."""
    dev = _require_gpu(hidden_states, top_k_index, top_k_weights, gu_packed, gu_scale, dn_packed, dn_scale)
    H = hidden_states.shape[-1]
    x = _rows(_bf16(hidden_states, "hidden_states"), H)
    gu_packed = _i32(gu_packed, "gate_up_packed")
    dn_packed = _i32(dn_packed, "down_packed")
    gu_scale = _bf16(gu_scale, "gate_up_scale")
    dn_scale = _bf16(dn_scale, "down_scale")
    if gu_packed.shape[-1] * 8 != H:
        raise ValueError(f"expert weight shape {tuple(gu_packed.shape)} does not match hidden size {H}")
    E, H, I, G = _expert_shape(gu_packed, gu_scale, dn_packed, dn_scale, group_size)
    idx, w = _routing(top_k_index, top_k_weights, x.shape[0])
    M, k = idx.shape
    out = torch.empty((M, H), dtype=torch.bfloat16, device=dev)
    lib = load()
    nbytes = lib.moe_workspace_bytes(max(M, 1), k, E, H, I)
    ws = _workspace(nbytes, dev)
    st = _resolve_tiles(tiles, gu_packed, gu_scale, dn_packed, dn_scale, E, H, I, G)
    head = (_ptr(x), _ptr(idx), _ptr(w), _ptr(gu_packed), _ptr(gu_scale), _ptr(dn_packed), _ptr(dn_scale))
    tail = (_ptr(out), M, k, E, H, I, G, _ptr(ws), nbytes)
    if st is None:
        _call("moe_forward", dev, lib.moe_forward, *head, *tail)
    else:
        _call("moe_forward_tiled", dev, lib.moe_forward_tiled, *head, st, *tail)
    return _like(out, hidden_states.shape)


@dataclass
class TiledWeights:
    """Load-time tiled copies of one expert stack's packed weights (a re-layout
    beside quantization.py:325-430; the packed tensors stay as they are): the
    decode streamers' copies (group size 128, 32 or 64; at 32 and 64 they hold
    the group scales too) and the prefill GEMM's.  Any of them may be None:
    that kernel then reads the packed tensors."""
    E: int
    H: int
    I: int
    group_size: int
    gu_decode: torch.Tensor | None = None
    dn_decode: torch.Tensor | None = None
    gu_prefill: torch.Tensor | None = None
    dn_prefill: torch.Tensor | None = None

    def struct(self) -> TiledExpertsC:
        """The w4a16_tiled_experts the *_tiled entry points take: of the copies as they are
        now (the fields are compared on every call; only the C structure is kept, and a
        changed one is a new structure)."""
        copies = (self.gu_decode, self.dn_decode, self.gu_prefill, self.dn_prefill)
        key = (self.E, self.H, self.I, self.group_size,
               *[None if t is None else (t.data_ptr(), t.numel() * t.element_size()) for t in copies])
        held = self.__dict__.get("_struct")
        if held is not None and held[0] == key:
            return held[1]
        fields = [v for c in key[4:] for v in (c or (None, 0))]
        st = TiledExpertsC(*key[:4], *fields)
        self.__dict__["_struct"] = (key, st)
        return st

    def __getstate__(self):
        # (copies and pickles carry the fields alone)
        return {k: v for k, v in self.__dict__.items() if k != "_struct"}

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.gu_decode, self.dn_decode, self.gu_prefill,
                                                          self.dn_prefill) if t is not None)


def tiled_bytes(kind: int, E: int, H: int, I: int, group_size: int) -> int:
    """Bytes of a tiled copy of ``kind`` (TILED_*) for the shape, 0 where none exists."""
    return load().w4a16_tiled_bytes(kind, E, H, I, group_size)


def _tile(kind: int, packed: torch.Tensor, scale: torch.Tensor | None, E: int, H: int, I: int, G: int):
    nbytes = tiled_bytes(kind, E, H, I, G)
    if nbytes == 0:
        return None
    dev = packed.device
    tiled = torch.empty(nbytes // 4, dtype=torch.int32, device=dev)
    _call("w4a16_tile", dev, load().w4a16_tile, kind, _ptr(packed), _ptr(scale), E, H, I, G, _ptr(tiled), nbytes)
    return tiled


def _expert_shape(gu_packed, gu_scale, dn_packed, dn_scale, group_size):
    E, two_i, h8 = gu_packed.shape
    H, I = h8 * 8, two_i // 2
    if dn_packed.shape != (E, H, I // 8) or two_i % 2:
        raise ValueError(f"expert weight shapes {tuple(gu_packed.shape)} / {tuple(dn_packed.shape)} do not match")
    G = group_size or infer_group_size(H, gu_scale.shape[-1])
    if gu_scale.shape != (E, two_i, -(-H // G)) or dn_scale.shape != (E, H, -(-I // G)):
        raise ValueError(f"scale shapes {tuple(gu_scale.shape)} / {tuple(dn_scale.shape)} "
                         f"do not match group size {G}")
    return E, H, I, G


def tile_experts(gu_packed: torch.Tensor, gu_scale: torch.Tensor, dn_packed: torch.Tensor,
                 dn_scale: torch.Tensor, group_size: int | None = None, decode: bool = True,
                 prefill: bool = True) -> TiledWeights:
    """The tiled copies of an expert stack (gate_up_packed [E, 2I, H/8], down_packed
    [E, H, I/8] and their scales): ``decode`` the decode streamers' (where they have
    a tiled form for the group size), ``prefill`` the prefill GEMM's.  About one more
    copy of the expert weights per kind asked for."""
    dev = _require_gpu(gu_packed, gu_scale, dn_packed, dn_scale)
    gu_packed, dn_packed = _i32(gu_packed, "gate_up_packed"), _i32(dn_packed, "down_packed")
    gu_scale, dn_scale = _bf16(gu_scale, "gate_up_scale"), _bf16(dn_scale, "down_scale")
    E, H, I, G = _expert_shape(gu_packed, gu_scale, dn_packed, dn_scale, group_size)
    tw = TiledWeights(E, H, I, G)
    if decode:
        tw.gu_decode = _tile(TILED_GATE_UP_DECODE, gu_packed, gu_scale, E, H, I, G)
        tw.dn_decode = _tile(TILED_DOWN_DECODE, dn_packed, dn_scale, E, H, I, G)
    if prefill:
        tw.gu_prefill = _tile(TILED_GATE_UP_PREFILL, gu_packed, None, E, H, I, G)
        tw.dn_prefill = _tile(TILED_DOWN_PREFILL, dn_packed, None, E, H, I, G)
    del dev
    return tw


# ------------------------------------------------------------ tiled-copy registry
# The reference's entry points pass only the packed tensors (the 7 arguments of
# fused_triton_4bit_moe_forward / hybrid_agent::fused_4bit_moe, quantization.py:88-96,
# backends.py:48-60, and the 22 of _ffn_moe_4bit_step).  Copies registered for a
# stack are found from those tensors: keyed by the packed gate_up buffer's address,
# valid while all four tensors are the ones tiled (same addresses, shapes and
# version counters -- an in-place reload through copy_ / load_state_dict bumps the
# counter).  A stale entry is dropped and the call reads the packed tensors.
_REGISTRY: dict[int, tuple] = {}
_REGISTRY_LOCK = threading.Lock()


def _version_of(t: torch.Tensor):
    # inference-mode tensors keep no version counter (and cannot be changed in
    # place outside inference mode)
    try:
        return t._version
    except RuntimeError:
        return None


def _signature(*ts: torch.Tensor) -> tuple:
    return tuple([(t.data_ptr(), t.shape, _version_of(t)) for t in ts])


def register_tiles(gu_packed: torch.Tensor, gu_scale: torch.Tensor, dn_packed: torch.Tensor,
                   dn_scale: torch.Tensor, tiles: TiledWeights) -> None:
    """Make ``tiles`` the copies every forward finds for this expert stack."""
    key = gu_packed.data_ptr()
    entry = (_signature(gu_packed, gu_scale, dn_packed, dn_scale), tiles)
    with _REGISTRY_LOCK:
        _REGISTRY[key] = entry
    # the entry goes when the packed tensor does (its address may be reused)
    weakref.finalize(gu_packed, _drop_if_same, key, entry)


def _drop_if_same(key: int, entry) -> None:
    with _REGISTRY_LOCK:
        if _REGISTRY.get(key) is entry:
            del _REGISTRY[key]


def unregister_tiles(gu_packed: torch.Tensor) -> None:
    with _REGISTRY_LOCK:
        _REGISTRY.pop(gu_packed.data_ptr(), None)


def lookup_tiles(gu_packed: torch.Tensor, gu_scale: torch.Tensor, dn_packed: torch.Tensor,
                 dn_scale: torch.Tensor) -> TiledWeights | None:
    """The registered copies of this expert stack, or None (none, or stale: then dropped)."""
    if not _REGISTRY:
        return None
    key = gu_packed.data_ptr()
    with _REGISTRY_LOCK:
        entry = _REGISTRY.get(key)
        if entry is None:
            return None
        if entry[0] != _signature(gu_packed, gu_scale, dn_packed, dn_scale):
            del _REGISTRY[key]
            stale = True
        else:
            return entry[1]
    if stale:
        warnings.warn("the tiled copies of an expert stack were dropped: its weights changed after they were "
                      "made (tile them again to use them); this call reads the packed weights", RuntimeWarning,
                      stacklevel=3)
    return None


def _resolve_tiles(tiles, gu_packed, gu_scale, dn_packed, dn_scale, E, H, I, G):
    """``tiles`` "auto": the registry's (if made for this call's shape and group
    size); None: none; else the given TiledWeights, which must be for this shape
    (the C ABI checks it again)."""
    if isinstance(tiles, str):
        if tiles != "auto":
            raise ValueError("tiles must be 'auto', None or a TiledWeights")
        tiles = lookup_tiles(gu_packed, gu_scale, dn_packed, dn_scale)
        if tiles is not None and (tiles.E, tiles.H, tiles.I, tiles.group_size) != (E, H, I, G):
            tiles = None
    if tiles is None:
        return None
    if (tiles.E, tiles.H, tiles.I, tiles.group_size) != (E, H, I, G):
        raise ValueError(f"tiled copies are for (E, H, I, G) = {(tiles.E, tiles.H, tiles.I, tiles.group_size)}, "
                         f"the call is {(E, H, I, G)}")
    return ctypes.byref(tiles.struct())


def moe_layer_forward(router_in: torch.Tensor, router_scale: torch.Tensor, scalar_root: float,
                      proj_w: torch.Tensor, per_expert_scale: torch.Tensor, eps: float, top_k: int,
                      hidden_states: torch.Tensor, gu_packed: torch.Tensor, gu_scale: torch.Tensor,
                      dn_packed: torch.Tensor, dn_scale: torch.Tensor, group_size: int | None = None,
                      *, tiles="auto"):
    """Router (backends.py:111-117) on ``router_in`` + experts (quantization.py:88-129) on
    ``hidden_states`` in one call -> (out [T, H] bf16, top_k_weights fp32, top_k_index int64).
    ``tiles`` as for moe_forward."""
    dev = _require_gpu(router_in, router_scale, proj_w, per_expert_scale, hidden_states, gu_packed,
                       gu_scale, dn_packed, dn_scale)
    H = hidden_states.shape[-1]
    r2 = _rows(_bf16(router_in, "router_in"), H)
    x = _rows(_bf16(hidden_states, "hidden_states"), H)
    if r2.shape != x.shape:
        raise ValueError("router input and expert input must have the same shape")
    router_scale = _bf16(router_scale, "router scale")
    proj_w = _bf16(proj_w, "router proj weight")
    per_expert_scale = _bf16(per_expert_scale, "per_expert_scale")
    gu_packed, dn_packed = _i32(gu_packed, "gate_up_packed"), _i32(dn_packed, "down_packed")
    gu_scale, dn_scale = _bf16(gu_scale, "gate_up_scale"), _bf16(dn_scale, "down_scale")
    if gu_packed.shape[-1] * 8 != H:
        raise ValueError("expert weight shapes do not match the hidden size")
    E, H, I, G = _expert_shape(gu_packed, gu_scale, dn_packed, dn_scale, group_size)
    if proj_w.shape != (E, H):
        raise ValueError("router weight shape does not match the experts")
    M = x.shape[0]
    out = torch.empty((M, H), dtype=torch.bfloat16, device=dev)
    idx = torch.empty((M, top_k), dtype=torch.int64, device=dev)
    w = torch.empty((M, top_k), dtype=torch.float32, device=dev)
    lib = load()
    nbytes = lib.moe_layer_workspace_bytes(max(M, 1), top_k, E, H, I)
    ws = _workspace(nbytes, dev)
    st = _resolve_tiles(tiles, gu_packed, gu_scale, dn_packed, dn_scale, E, H, I, G)
    common = (_ptr(r2), _ptr(router_scale), float(scalar_root), _ptr(proj_w), _ptr(per_expert_scale), float(eps),
              _ptr(x), _ptr(gu_packed), _ptr(gu_scale), _ptr(dn_packed), _ptr(dn_scale))
    tail = (_ptr(out), _ptr(idx), _ptr(w), M, top_k, E, H, I, G, _ptr(ws), nbytes)
    if st is None:
        _call("moe_layer_forward", dev, lib.moe_layer_forward, *common, *tail)
    else:
        _call("moe_layer_forward_tiled", dev, lib.moe_layer_forward_tiled, *common, st, *tail)
    return _like(out, hidden_states.shape), w, idx


def moe_layer_forward_add_norm(router_in: torch.Tensor, router_scale: torch.Tensor, scalar_root: float,
                               proj_w: torch.Tensor, per_expert_scale: torch.Tensor, eps: float, top_k: int,
                               hidden_states: torch.Tensor, gu_packed: torch.Tensor, gu_scale: torch.Tensor,
                               dn_packed: torch.Tensor, dn_scale: torch.Tensor, norm_weight: torch.Tensor,
                               norm_eps: float, group_size: int | None = None, *, tiles="auto"):
    """moe_layer_forward on (router_in = h, hidden_states), then h_out = bf16(h + out) and
    y = RMSNorm(h_out) * norm_weight (add_rms_norm's arithmetic), the combine, the add and
    the norm in one launch where the layer has a combine launch of its own (the latent
    harness's step) -> (h_out, y, out, top_k_weights, top_k_index)."""
    dev = _require_gpu(router_in, router_scale, proj_w, per_expert_scale, hidden_states, gu_packed,
                       gu_scale, dn_packed, dn_scale, norm_weight)
    H = hidden_states.shape[-1]
    r2 = _rows(_bf16(router_in, "router_in"), H)
    x = _rows(_bf16(hidden_states, "hidden_states"), H)
    if r2.shape != x.shape:
        raise ValueError("router input and expert input must have the same shape")
    norm_weight = _bf16(norm_weight, "norm weight")
    if norm_weight.shape != (H,):
        raise ValueError(f"norm weight must be [{H}]")
    router_scale = _bf16(router_scale, "router scale")
    proj_w = _bf16(proj_w, "router proj weight")
    per_expert_scale = _bf16(per_expert_scale, "per_expert_scale")
    gu_packed, dn_packed = _i32(gu_packed, "gate_up_packed"), _i32(dn_packed, "down_packed")
    gu_scale, dn_scale = _bf16(gu_scale, "gate_up_scale"), _bf16(dn_scale, "down_scale")
    E, H, I, G = _expert_shape(gu_packed, gu_scale, dn_packed, dn_scale, group_size)
    if proj_w.shape != (E, H):
        raise ValueError("router weight shape does not match the experts")
    M = x.shape[0]
    out = torch.empty((M, H), dtype=torch.bfloat16, device=dev)
    h_out = torch.empty((M, H), dtype=torch.bfloat16, device=dev)
    y = torch.empty((M, H), dtype=torch.bfloat16, device=dev)
    idx = torch.empty((M, top_k), dtype=torch.int64, device=dev)
    w = torch.empty((M, top_k), dtype=torch.float32, device=dev)
    lib = load()
    nbytes = lib.moe_layer_workspace_bytes(max(M, 1), top_k, E, H, I)
    ws = _workspace(nbytes, dev)
    st = _resolve_tiles(tiles, gu_packed, gu_scale, dn_packed, dn_scale, E, H, I, G)
    _call("moe_layer_forward_add_norm", dev, lib.moe_layer_forward_add_norm,
          _ptr(r2), _ptr(router_scale), float(scalar_root), _ptr(proj_w), _ptr(per_expert_scale), float(eps),
          _ptr(x), _ptr(gu_packed), _ptr(gu_scale), _ptr(dn_packed), _ptr(dn_scale), st, _ptr(out), _ptr(idx), _ptr(w),
          _ptr(norm_weight), float(norm_eps), _ptr(h_out), _ptr(y), M, top_k, E, H, I, G, _ptr(ws), nbytes)
    shape = hidden_states.shape
    return _like(h_out, shape), _like(y, shape), _like(out, shape), w, idx


def bf16_experts_forward(hidden_states: torch.Tensor, top_k_index: torch.Tensor, top_k_weights: torch.Tensor,
                         gate_up_proj: torch.Tensor, down_proj: torch.Tensor) -> torch.Tensor:
    """MoE output [T, H] with unquantised bf16 experts (backends.py:209-283):
    gate_up_proj [E, 2I, H], down_proj [E, H, I] (Gemma4TextExperts parameters)."""
    dev = _require_gpu(hidden_states, top_k_index, top_k_weights, gate_up_proj, down_proj)
    H = hidden_states.shape[-1]
    x = _rows(_bf16(hidden_states, "hidden_states"), H)
    gu = _bf16(gate_up_proj, "gate_up_proj")
    dn = _bf16(down_proj, "down_proj")
    E, two_i, h = gu.shape
    I = two_i // 2
    if h != H or two_i % 2 or dn.shape != (E, H, I):
        raise ValueError(f"expert weight shapes {tuple(gu.shape)} / {tuple(dn.shape)} do not match hidden size {H}")
    idx, w = _routing(top_k_index, top_k_weights, x.shape[0])
    M, k = idx.shape
    out = torch.empty((M, H), dtype=torch.bfloat16, device=dev)
    lib = load()
    nbytes = lib.moe_bf16_experts_workspace_bytes(max(M, 1), k, E, H, I)
    ws = _workspace(nbytes, dev)
    _call("moe_bf16_experts_forward", dev, lib.moe_bf16_experts_forward, _ptr(x), _ptr(idx), _ptr(w), _ptr(gu),
          _ptr(dn), _ptr(out), M, k, E, H, I, _ptr(ws), nbytes)
    return _like(out, hidden_states.shape)


def ffn_block(residual: torch.Tensor, attn_out: torch.Tensor, post_attn_ln_w: torch.Tensor,
              pre_ff_ln_w: torch.Tensor, mlp_gate_w: torch.Tensor, mlp_up_w: torch.Tensor,
              mlp_down_w: torch.Tensor, post_ff_ln1_w: torch.Tensor, router_scale: torch.Tensor,
              router_scalar_root: float, router_proj_w: torch.Tensor, router_per_expert_scale: torch.Tensor,
              pre_ff_ln2_w: torch.Tensor, gu_packed: torch.Tensor, gu_scale: torch.Tensor,
              dn_packed: torch.Tensor, dn_scale: torch.Tensor, post_ff_ln2_w: torch.Tensor,
              post_ff_ln_w: torch.Tensor, layer_scalar: torch.Tensor, eps: float, top_k: int,
              group_size: int | None = None, *, tiles="auto", return_routing: bool = False):
    """The post-attention FFN block ``_ffn_moe_4bit_step`` (backends.py:77-126), same
    arguments in the same order: residual / attn_out [..., H] bf16 -> [..., H] bf16.
    ``tiles`` as for moe_forward.  With ``return_routing`` also the routing the block's
    router step took: (out, top_k_index int64 [M, k], top_k_weights fp32 [M, k])."""
    dense = (post_attn_ln_w, pre_ff_ln_w, mlp_gate_w, mlp_up_w, mlp_down_w, post_ff_ln1_w, router_scale,
             router_proj_w, router_per_expert_scale, pre_ff_ln2_w, post_ff_ln2_w, post_ff_ln_w)
    dev = _require_gpu(residual, attn_out, *dense, gu_packed, gu_scale, dn_packed, dn_scale, layer_scalar)
    H = residual.shape[-1]
    res = _rows(_bf16(residual, "residual"), H)
    att = _rows(_bf16(attn_out, "attn_out"), H)
    if att.shape != res.shape:
        raise ValueError("attn_out must have the shape of residual")
    names = ("post_attention_layernorm", "pre_feedforward_layernorm", "mlp.gate_proj", "mlp.up_proj",
             "mlp.down_proj", "post_feedforward_layernorm_1", "router.scale", "router.proj",
             "router.per_expert_scale", "pre_feedforward_layernorm_2", "post_feedforward_layernorm_2",
             "post_feedforward_layernorm")
    dense = tuple(_bf16(t, n) for t, n in zip(dense, names))
    (post_attn_ln_w, pre_ff_ln_w, mlp_gate_w, mlp_up_w, mlp_down_w, post_ff_ln1_w, router_scale,
     router_proj_w, router_per_expert_scale, pre_ff_ln2_w, post_ff_ln2_w, post_ff_ln_w) = dense
    # layer_scalar is a bf16 buffer once the model is loaded in bf16; other
    # dtypes are rounded to it (the product is a bf16 tensor either way)
    ls = layer_scalar
    if ls.shape != (1,) or ls.dtype != torch.bfloat16:
        ls = layer_scalar.reshape(-1)[:1].to(torch.bfloat16).contiguous()
    for t, n in ((post_attn_ln_w, names[0]), (pre_ff_ln_w, names[1]), (post_ff_ln1_w, names[5]),
                 (router_scale, names[6]), (pre_ff_ln2_w, names[9]), (post_ff_ln2_w, names[10]),
                 (post_ff_ln_w, names[11])):
        if t.shape != (H,):
            raise ValueError(f"{n} weight must be [{H}]")
    Im = mlp_gate_w.shape[0]
    if mlp_gate_w.shape != (Im, H) or mlp_up_w.shape != (Im, H) or mlp_down_w.shape != (H, Im):
        raise ValueError("shared MLP weights must be gate/up [Im, H] and down [H, Im]")
    gu_packed, dn_packed = _i32(gu_packed, "gate_up_packed"), _i32(dn_packed, "down_packed")
    gu_scale, dn_scale = _bf16(gu_scale, "gate_up_scale"), _bf16(dn_scale, "down_scale")
    if gu_packed.shape[-1] * 8 != H:
        raise ValueError("expert weight shapes do not match the hidden size")
    E, H, I, G = _expert_shape(gu_packed, gu_scale, dn_packed, dn_scale, group_size)
    if router_proj_w.shape != (E, H):
        raise ValueError("router weight shape does not match the experts")
    M = res.shape[0]
    out = torch.empty((M, H), dtype=torch.bfloat16, device=dev)
    lib = load()
    nbytes = lib.moe_ffn_block_workspace_bytes(max(M, 1), top_k, E, H, I, Im)
    ws = _workspace(nbytes, dev)
    st = _resolve_tiles(tiles, gu_packed, gu_scale, dn_packed, dn_scale, E, H, I, G)
    head = (_ptr(res), _ptr(att), _ptr(post_attn_ln_w), _ptr(pre_ff_ln_w), _ptr(mlp_gate_w), _ptr(mlp_up_w),
            _ptr(mlp_down_w), _ptr(post_ff_ln1_w), _ptr(router_scale), float(router_scalar_root),
            _ptr(router_proj_w), _ptr(router_per_expert_scale), _ptr(pre_ff_ln2_w), _ptr(gu_packed),
            _ptr(gu_scale), _ptr(dn_packed), _ptr(dn_scale))
    tail = (_ptr(post_ff_ln2_w), _ptr(post_ff_ln_w), _ptr(ls), float(eps), _ptr(out), M, int(top_k), E, H, I, Im,
            G, _ptr(ws), nbytes)
    if st is None:
        _call("moe_ffn_block_forward", dev, lib.moe_ffn_block_forward, *head, *tail)
    else:
        _call("moe_ffn_block_forward_tiled", dev, lib.moe_ffn_block_forward_tiled, *head, st, *tail)
    out = _like(out, residual.shape)
    if not return_routing:
        return out
    if M == 0:
        return out, torch.empty((0, top_k), dtype=torch.int64, device=dev), \
            torch.empty((0, top_k), dtype=torch.float32, device=dev)
    io, wo = ctypes.c_size_t(), ctypes.c_size_t()
    _check(lib.moe_ffn_block_routing_offsets(M, top_k, E, H, I, Im, ctypes.byref(io), ctypes.byref(wo)),
           "moe_ffn_block_routing_offsets")
    n = M * top_k
    idx = ws[io.value:io.value + 8 * n].view(torch.int64).reshape(M, top_k).clone()
    w = ws[wo.value:wo.value + 4 * n].view(torch.float32).reshape(M, top_k).clone()
    return out, idx, w


# ------------------------------------------------------------------ training forms

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # enum w4a16_dtype


def _rows_like(t: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
    """t of the shape and type of ``like`` (a gradient of it), as contiguous rows."""
    if t.shape != like.shape or t.dtype != like.dtype:
        raise ValueError(f"{name} must be {like.dtype} {list(like.shape)}, got {t.dtype} {list(t.shape)}")
    return _rows(t.contiguous(), t.shape[-1])


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t at a multiple of 16 bytes.  A caller places its own tensors so; where autograd puts a
    gradient (a slice of a concatenation's, say) it has no say in."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _saved(t: torch.Tensor, nbytes: int) -> torch.Tensor:
    if t.dtype != torch.uint8 or t.dim() != 1 or not t.is_contiguous() or t.numel() != nbytes:
        raise ValueError(f"saved must be the uint8 [{nbytes}] that the forward call of this shape returned")
    return t


def _ln_params(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None):
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError("x must have a last dimension")
    H = x.shape[-1]
    for t, n in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.shape != (H,) or t.dtype != x.dtype):
            raise ValueError(f"{n} must be {x.dtype} [{H}], got {t.dtype} {list(t.shape)}")
    return dt, H


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, eps: float = 1e-5,
               return_stats: bool = False):
    """nn.LayerNorm over the last dimension (hybridlink.py:20,23) of bf16, fp16 or fp32 rows,
    weight and bias [H] of the same type; statistics in fp32.  With ``return_stats``
    (y, mean, rstd), float32 of x's leading shape, for ``layer_norm_backward``."""
    dev = _require_gpu(x, weight, bias)
    dt, H = _ln_params(x, weight, bias)
    x2 = _rows(x.contiguous(), H)
    M = x2.shape[0]
    y = torch.empty_like(x2)
    mean = rstd = None
    if return_stats:
        lead = x.shape[:-1]
        mean = torch.empty(lead, dtype=torch.float32, device=dev)
        rstd = torch.empty(lead, dtype=torch.float32, device=dev)
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    _call("w4a16_layer_norm", dev, load().w4a16_layer_norm, _ptr(x2), _ptr(weight), _ptr(bias), _ptr(y), _ptr(mean),
          _ptr(rstd), dt, M, H, float(eps))
    y = _like(y, x.shape)
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor,
                        rstd: torch.Tensor, bias: bool = True):
    """(dx, dweight, dbias) of ``layer_norm`` for the gradient ``dy`` of its output; ``mean`` and
    ``rstd`` are what the forward returned.  dbias is None where ``bias`` is False.  The sums
    over the rows are taken in fp32, in an order set by the shape, the type and the tensors'
    alignment to 16 bytes."""
    dev = _require_gpu(dy, x, weight, mean, rstd)
    dt, H = _ln_params(x, weight, None)
    dy2 = _rows_like(dy, "dy", x)
    for t, n in ((mean, "mean"), (rstd, "rstd")):
        if t.shape != x.shape[:-1] or t.dtype != torch.float32:
            raise ValueError(f"{n} must be float32 {list(x.shape[:-1])}, got {t.dtype} {list(t.shape)}")
    x2 = _rows(x.contiguous(), H)
    weight, mean, rstd = weight.contiguous(), mean.contiguous(), rstd.contiguous()
    M = x2.shape[0]
    dx = torch.empty_like(x2)
    dw = torch.empty_like(weight)
    db = torch.empty_like(weight) if bias else None
    lib = load()
    nbytes = lib.w4a16_layer_norm_backward_workspace_bytes(M, H)
    ws = _workspace(nbytes, dev)
    _call("w4a16_layer_norm_backward", dev, lib.w4a16_layer_norm_backward, _ptr(dy2), _ptr(x2), _ptr(weight),
          _ptr(mean), _ptr(rstd), _ptr(dx), _ptr(dw), _ptr(db), dt, M, H, _ptr(ws), nbytes)
    return _like(dx, x.shape), dw, db


def _mlp_weights(x: torch.Tensor, gate_w: torch.Tensor, up_w: torch.Tensor, down_w: torch.Tensor):
    if x.dim() == 0:
        raise ValueError("x must have a last dimension")
    H = x.shape[-1]
    gate_w, up_w, down_w = _bf16(gate_w, "gate_w"), _bf16(up_w, "up_w"), _bf16(down_w, "down_w")
    I = gate_w.shape[0]
    if gate_w.shape != (I, H) or up_w.shape != (I, H) or down_w.shape != (H, I):
        raise ValueError(f"the weights must be gate/up [I, {H}] and down [{H}, I], got {list(gate_w.shape)}, "
                         f"{list(up_w.shape)}, {list(down_w.shape)}")
    return gate_w, up_w, down_w, H, I


def gated_mlp(x: torch.Tensor, gate_w: torch.Tensor, up_w: torch.Tensor, down_w: torch.Tensor,
              return_saved: bool = False):
    """The gated feed-forward block (the shared MLP of backends.py:105-108):
    y = (gelu_tanh(x gate_w^T) * (x up_w^T)) down_w^T on bf16 [..., H], weights in the nn.Linear
    layout.  With ``return_saved`` (y, saved): what ``gated_mlp_backward`` needs, one uint8 tensor
    of about 10 bytes per row and column of I."""
    dev = _require_gpu(x, gate_w, up_w, down_w)
    x = _bf16(x, "x")
    gate_w, up_w, down_w, H, I = _mlp_weights(x, gate_w, up_w, down_w)
    x2 = _rows(x, H)
    M = x2.shape[0]
    y = torch.empty_like(x2)
    lib = load()
    nbytes = lib.w4a16_gated_mlp_workspace_bytes(M, H, I)
    ws = _workspace(nbytes, dev)
    saved, nsaved = None, 0
    if return_saved:
        nsaved = lib.w4a16_gated_mlp_saved_bytes(M, I)
        saved = torch.empty((nsaved,), dtype=torch.uint8, device=dev)
    _call("w4a16_gated_mlp", dev, lib.w4a16_gated_mlp, _ptr(x2), _ptr(gate_w), _ptr(up_w), _ptr(down_w), _ptr(y),
          _ptr(saved) if nsaved else None, nsaved, M, H, I, _ptr(ws), nbytes)
    y = _like(y, x.shape)
    return (y, saved) if return_saved else y


def gated_mlp_backward(dy: torch.Tensor, x: torch.Tensor, gate_w: torch.Tensor, up_w: torch.Tensor,
                       down_w: torch.Tensor, saved: torch.Tensor, needs=(True, True, True, True)):
    """(dx, dgate_w, dup_w, ddown_w) of ``gated_mlp`` for the gradient ``dy`` of its output and the
    ``saved`` of that forward call.  ``needs``: which of the four are wanted; the others are None
    and not computed (a frozen weight's)."""
    dev = _require_gpu(dy, x, gate_w, up_w, down_w, saved)
    x = _bf16(x, "x")
    gate_w, up_w, down_w, H, I = _mlp_weights(x, gate_w, up_w, down_w)
    dy2 = _aligned(_rows_like(dy, "dy", x))
    x2 = _rows(x, H)
    M = x2.shape[0]
    lib = load()
    nsaved = lib.w4a16_gated_mlp_saved_bytes(M, I)
    saved = _saved(saved, nsaved)
    if len(needs) != 4:
        raise ValueError("needs must say for each of dx, dgate_w, dup_w and ddown_w whether it is wanted")
    dx, dg, du, dd = (torch.empty_like(t) if n else None for t, n in zip((x2, gate_w, up_w, down_w), needs))
    nbytes = lib.w4a16_gated_mlp_backward_workspace_bytes(M, H, I)
    ws = _workspace(nbytes, dev)
    _call("w4a16_gated_mlp_backward", dev, lib.w4a16_gated_mlp_backward, _ptr(dy2), _ptr(x2), _ptr(gate_w),
          _ptr(up_w), _ptr(down_w), _ptr(saved), nsaved, _ptr(dx), _ptr(dg), _ptr(du), _ptr(dd), M, H, I, _ptr(ws),
          nbytes)
    return None if dx is None else _like(dx, x.shape), dg, du, dd


def _link_params(h: torch.Tensor, params):
    names = ("pre_ln weight", "pre_ln bias", "proj1 weight", "proj1 bias", "proj2 weight", "proj2 bias",
             "post_ln weight", "post_ln bias")
    if h.dim() == 0:
        raise ValueError("h must have a last dimension")
    H = h.shape[-1]
    params = tuple(_bf16(p, n) for p, n in zip(params, names))
    for i, p in enumerate(params):
        want = (H, H) if i in (2, 4) else (H,)
        if p.shape != want:
            raise ValueError(f"{names[i]} must be {list(want)}, got {list(p.shape)}")
    return params, H


def hybridlink_train(h: torch.Tensor, ln1_w: torch.Tensor, ln1_b: torch.Tensor, p1_w: torch.Tensor,
                     p1_b: torch.Tensor, p2_w: torch.Tensor, p2_b: torch.Tensor, ln2_w: torch.Tensor,
                     ln2_b: torch.Tensor, eps: float = 1e-5):
    """``hybridlink`` (hybridlink.py:17-28) for training -> (out, saved): ``saved`` is what
    ``hybridlink_backward`` needs, one uint8 tensor of about 12 bytes per element of h.  Only
    what a product takes is rounded to bf16, once, from fp32 (``hybridlink`` rounds where the
    torch modules do)."""
    dev = _require_gpu(h, ln1_w, ln1_b, p1_w, p1_b, p2_w, p2_b, ln2_w, ln2_b)
    h = _bf16(h, "h")
    params, H = _link_params(h, (ln1_w, ln1_b, p1_w, p1_b, p2_w, p2_b, ln2_w, ln2_b))
    h2 = _rows(h, H)
    B = h2.shape[0]
    out = torch.empty_like(h2)
    lib = load()
    nsaved = lib.w4a16_hybridlink_saved_bytes(B, H)
    saved = torch.empty((nsaved,), dtype=torch.uint8, device=dev)
    nbytes = lib.w4a16_hybridlink_train_workspace_bytes(B, H)
    ws = _workspace(nbytes, dev)
    _call("w4a16_hybridlink_train", dev, lib.w4a16_hybridlink_train, _ptr(h2), *[_ptr(p) for p in params], _ptr(out),
          _ptr(saved), nsaved, B, H, float(eps), _ptr(ws), nbytes)
    return _like(out, h.shape), saved


def hybridlink_backward(dout: torch.Tensor, h: torch.Tensor, ln1_w: torch.Tensor, ln1_b: torch.Tensor,
                        p1_w: torch.Tensor, p1_b: torch.Tensor, p2_w: torch.Tensor, p2_b: torch.Tensor,
                        ln2_w: torch.Tensor, ln2_b: torch.Tensor, saved: torch.Tensor):
    """(dh, then the gradients of the eight parameters in their order) of ``hybridlink_train`` for
    the gradient ``dout`` of its output and the ``saved`` of that forward call."""
    dev = _require_gpu(dout, h, ln1_w, ln1_b, p1_w, p1_b, p2_w, p2_b, ln2_w, ln2_b, saved)
    h = _bf16(h, "h")
    params, H = _link_params(h, (ln1_w, ln1_b, p1_w, p1_b, p2_w, p2_b, ln2_w, ln2_b))
    d2 = _aligned(_rows_like(dout, "dout", h))
    h2 = _rows(h, H)
    B = h2.shape[0]
    lib = load()
    nsaved = lib.w4a16_hybridlink_saved_bytes(B, H)
    saved = _saved(saved, nsaved)
    dh = torch.empty_like(h2)
    grads = tuple(torch.empty_like(p) for p in params)
    nbytes = lib.w4a16_hybridlink_backward_workspace_bytes(B, H)
    ws = _workspace(nbytes, dev)
    _call("w4a16_hybridlink_backward", dev, lib.w4a16_hybridlink_backward, _ptr(d2), _ptr(h2), _ptr(params[0]),
          _ptr(params[2]), _ptr(params[4]), _ptr(params[6]), _ptr(saved), nsaved, _ptr(dh),
          *[_ptr(g) for g in grads], B, H, _ptr(ws), nbytes)
    return (_like(dh, h.shape), *grads)


# ------------------------------------------------------------------ attention

# The calls of a decoded token take 5 to 15 us on the GPU: what the host does in front of them is
# kept to one pass over the arguments (devices by number, strides and sizes read once).


def _gpu_of(*tensors: torch.Tensor | None) -> int:
    """The number of the GPU that all tensors are on (``_require_gpu``'s errors)."""
    index = -2  # -1: the host
    for t in tensors:
        if t is not None:
            i = t.get_device()
            if i != index:
                if i < 0 or index >= 0:
                    _require_gpu(*tensors)
                    raise RuntimeError("tensors on different devices")
                index = i
    return index


def _launch(what: str, index: int, fn, *args) -> None:
    """fn(*args, the current stream of GPU ``index``), run with it current."""
    if _get_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status != W4A16_OK:
        _check(status, what)


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _dense(t: torch.Tensor):
    """t contiguous, at a multiple of 16 bytes, and its address."""
    p = t.data_ptr()
    if p & 15 or not t.is_contiguous():
        t = _aligned(t.contiguous())
        p = t.data_ptr()
    return t, p


_NO_HEADS = (None, 0, 0)
_LANES = {torch.bfloat16: 8, torch.float16: 8, torch.float32: 4}  # elements of 16 bytes


def _heads(t: torch.Tensor, name: str):
    """t [tokens, heads, D] as the kernels take it, and its pointer and strides for them: D contiguous, the
    other strides as they are where every row starts at a multiple of 16 bytes and they are 64 MiB at
    most, else a copy."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head size], got {list(t.shape)}")
    a, b, c = t.stride()
    p = t.data_ptr()
    lanes = _LANES.get(t.dtype, 8)
    if c != 1 or (a | b) % lanes or p & 15 or a > lanes << 22 or b > lanes << 22:
        t = t.clone(memory_format=torch.contiguous_format)  # a size of one leaves contiguous()'s strides open
        p, (a, b, c) = t.data_ptr(), t.stride()
    return t, (p, a, b)


def _head_type(t: torch.Tensor, name: str, fp32: bool) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None or (dt == 2 and not fp32):
        raise ValueError(f"{name} must be bfloat16{', float16 or float32' if fp32 else ' or float16'}, got {t.dtype}")
    return dt


def _index(t: torch.Tensor, name: str, *shape: int) -> torch.Tensor:
    if t.dtype != torch.int32 or t.shape != shape:
        raise ValueError(f"{name} must be int32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _rope_args(q, k, v, cos, sin, positions, q_weight, k_weight, fp32: bool):
    """What the forms of the heads' norm check alike -> (type, q, k, v, the pointers and strides of these,
    (cos, sin, positions, weights), the pointers of these, sizes)."""
    dtype = q.dtype
    dt = _head_type(q, "q", fp32)
    q, args = _heads(q, "q")
    T, Hq, D = q.shape
    k, more = _heads(k, "k")
    args += more
    shape = k.shape
    if k.dtype != dtype or shape[0] != T or shape[2] != D:
        raise ValueError(f"k must be {dtype} [{T}, heads, {D}], got {k.dtype} {list(shape)}")
    if v is not None:
        v, more = _heads(v, "v")
        args += more
        if v.dtype != dtype or v.shape != shape:
            raise ValueError(f"v must be {dtype} {list(shape)}, got {v.dtype} {list(v.shape)}")
    else:
        args += _NO_HEADS
    P = R = 0
    pc = ps = pq = pk = None
    if cos is not None and sin is not None:
        table = cos.shape
        if cos.dtype != torch.float32 or sin.dtype != torch.float32 or len(table) != 2 or sin.shape != table:
            raise ValueError("cos and sin must be float32 [positions, half the turned columns], got "
                             f"{cos.dtype} {list(table)} and {sin.dtype} {list(sin.shape)}")
        P, R = table[0], 2 * table[1]
        cos, pc = _dense(cos)
        sin, ps = _dense(sin)
    elif cos is not None or sin is not None:
        raise ValueError("cos and sin are given together")
    positions = _index(positions, "positions", T)
    if q_weight is not None and k_weight is not None:
        for t, n in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            if t.dtype != dtype or t.shape != (D,):
                raise ValueError(f"{n} must be {dtype} [{D}], got {t.dtype} {list(t.shape)}")
        q_weight, pq = _dense(q_weight)
        k_weight, pk = _dense(k_weight)
    elif q_weight is not None or k_weight is not None:
        raise ValueError("q_weight and k_weight are given together")
    return (dt, q, k, v, args, (cos, sin, positions, q_weight, k_weight), (pc, ps, positions.data_ptr(), pq, pk),
            (T, Hq, shape[1], D, P, R))


def head_norm_rope(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, cos: torch.Tensor | None,
                   sin: torch.Tensor | None, positions: torch.Tensor, q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, eps: float = 1e-6):
    """RMS norm of every head and the position rotation in one pass -> (q, k, v), dense.

    q [T, Hq, D], k, v [T, Hk, D] of bf16, fp16 or fp32, any strides; weights [D] (None, both: no
    norm); cos, sin float32 [P, R / 2]: token t's columns i and i + R / 2 of q and k (i < R / 2) are
    turned by row ``positions[t]`` (int32).  v (may be None) is normed without a weight.  A position
    that the tables do not have makes its token's q and k NaN."""
    index = _gpu_of(q, k, v, cos, sin, positions, q_weight, k_weight)
    dt, q, k, v, heads, rot, at, sizes = _rope_args(q, k, v, cos, sin, positions, q_weight, k_weight, True)
    yq, yk = _dense_like(q), _dense_like(k)
    yv = None if v is None else _dense_like(v)
    _launch("w4a16_head_norm_rope", index, load().w4a16_head_norm_rope, *heads, *at, yq.data_ptr(), yk.data_ptr(),
            _ptr(yv), dt, *sizes, eps)
    return yq, yk, yv


def head_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor | None, q: torch.Tensor,
                            k: torch.Tensor, v: torch.Tensor | None, cos: torch.Tensor | None,
                            sin: torch.Tensor | None, positions: torch.Tensor, q_weight: torch.Tensor | None = None,
                            k_weight: torch.Tensor | None = None, eps: float = 1e-6, weights: bool = True):
    """(dq, dk, dv, dq_weight, dk_weight) of ``head_norm_rope`` for the gradients of its outputs.  The
    weights' are None without weights and where ``weights`` is False; dv is None without v.  The sums
    over the rows are taken in fp32, in an order set by the shapes."""
    index = _gpu_of(q, k, v, cos, sin, positions, q_weight, k_weight, dq, dk, dv)
    dt, q, k, v, heads, rot, at, sizes = _rope_args(q, k, v, cos, sin, positions, q_weight, k_weight, True)
    if (dv is None) != (v is None):
        raise ValueError("dv is given with v")
    for t, x, n in ((dq, q, "dq"), (dk, k, "dk"), (dv, v, "dv")):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError(f"{n} must be {x.dtype} {list(x.shape)}, got {t.dtype} {list(t.shape)}")
    dq, pq = _dense(dq)
    dk, pk = _dense(dk)
    dv, pv = (None, None) if dv is None else _dense(dv)
    xq, xk = torch.empty_like(dq), torch.empty_like(dk)
    xv = None if dv is None else torch.empty_like(dv)
    wq = wk = ws = None
    nbytes, lib = 0, load()
    if weights and q_weight is not None:
        wq, wk = torch.empty_like(rot[3]), torch.empty_like(rot[4])
        nbytes = lib.w4a16_head_norm_rope_backward_workspace_bytes(*sizes[:4])
        ws = q.new_empty(nbytes, dtype=torch.uint8)
    _launch("w4a16_head_norm_rope_backward", index, lib.w4a16_head_norm_rope_backward, pq, pk, pv, *heads, *at,
            xq.data_ptr(), xk.data_ptr(), _ptr(xv), _ptr(wq), _ptr(wk), dt, *sizes, eps, _ptr(ws), nbytes)
    return xq, xk, xv, wq, wk


def _cache_args(k_cache: torch.Tensor, v_cache: torch.Tensor, dtype: torch.dtype, D: int):
    """(the pointers and bytes between pages of a paged cache [pages, Hk, page size, D], its sizes);
    every page is dense."""
    shape = k_cache.shape
    if len(shape) != 4 or shape[3] != D or v_cache.shape != shape or k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError(f"k_cache and v_cache must be {dtype} [pages, heads, page size, {D}], got {k_cache.dtype} "
                         f"{list(shape)} and {v_cache.dtype} {list(v_cache.shape)}")
    pages, H, page, _ = shape
    args = []
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        a, b, c, d = t.stride()
        p = t.data_ptr()
        if pages == 1:  # the strides of a size of one are any
            a = H * page * D
        if (b != page * D and H != 1) or c != D or d != 1 or (p | 2 * a) & 15:
            raise ValueError(f"{n} must have dense pages at multiples of 16 bytes, got strides {t.stride()}")
        args += (p, a)
    return args, pages, H, page


def append_kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor | None, sin: torch.Tensor | None,
              positions: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
              v_norm: bool = False, return_kv: bool = False):
    """``head_norm_rope`` on the way into a paged cache -> q, dense; token t's keys and values (normed
    without a weight where ``v_norm``) go to row ``slots[t]`` (int32; page x page size + row) of
    k_cache, v_cache [pages, Hk, page size, D], bf16 or fp16.  A slot outside the cache (-1: a
    padding token's) is not written; two tokens of a call must not share one.  With ``return_kv``
    (q, k, v), dense, for ``attention`` over the same prompt."""
    if v is None:
        raise ValueError("v must be given")
    index = _gpu_of(q, k, v, cos, sin, positions, q_weight, k_weight, slots, k_cache, v_cache)
    dt, q, k, v, heads, rot, at, sizes = _rope_args(q, k, v, cos, sin, positions, q_weight, k_weight, False)
    slots = _index(slots, "slots", sizes[0])
    cache, pages, H, page = _cache_args(k_cache, v_cache, q.dtype, sizes[3])
    if H != sizes[2]:
        raise ValueError(f"the cache has {H} heads, k {sizes[2]}")
    out = _dense_like(q)
    yk, yv = (_dense_like(k), _dense_like(v)) if return_kv else (None, None)
    pc, ps, pp, pq, pk = at
    _launch("w4a16_append_kv", index, load().w4a16_append_kv, *heads, pc, ps, pp, slots.data_ptr(), pq, pk,
            out.data_ptr(), _ptr(yk), _ptr(yv), *cache, dt, bool(v_norm), *sizes, pages, page, eps)
    return (out, yk, yv) if return_kv else out


def _group(Hq: int, Hk: int, D: int) -> None:
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"the query heads must be a multiple of the key-value heads, got {Hq} and {Hk}")
    if D not in (64, 128, 256, 512):
        raise ValueError(f"the head size must be 64, 128, 256 or 512, got {D}")


def _attention_args(q, k, v, cu_q, cu_k, scale, causal, window):
    dt = _head_type(q, "q", False)
    q, args = _heads(q, "q")
    k, more = _heads(k, "k")
    v, last = _heads(v, "v")
    Tq, Hq, D = q.shape
    Tk, Hk, _ = shape = k.shape
    if k.dtype != q.dtype or v.dtype != q.dtype or shape[2] != D or v.shape != shape:
        raise ValueError(f"k and v must be {q.dtype} [tokens, heads, {D}], got {k.dtype} {list(shape)} and {v.dtype} "
                         f"{list(v.shape)}")
    _group(Hq, Hk, D)
    if cu_q.dim() != 1 or cu_q.numel() == 0:
        raise ValueError(f"cu_q must be int32 [sequences + 1], got {list(cu_q.shape)}")
    n = cu_q.shape[0]
    cu_q = _index(cu_q, "cu_q", n)
    if cu_k is None:
        if Tk != Tq:
            raise ValueError("without cu_k the queries and keys are of the same tokens")
        cu_k = cu_q
    else:
        cu_k = _index(cu_k, "cu_k", n)
    if window and not causal:
        raise ValueError("a window needs a causal mask")
    sizes = (n - 1, Tq, Tk, Hq, Hk, D, D ** -0.5 if scale is None else scale, bool(causal), window)
    return dt, q, k, v, args + more + last, cu_q, cu_k, sizes


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor | None = None,
              scale: float | None = None, causal: bool = True, window: int = 0, return_lse: bool = False):
    """Attention over packed sequences -> [Tq, Hq, D]; with ``return_lse`` also the scores' log sum of
    exponentials, float32 [Hq, Tq], for ``attention_backward``.

    q [Tq, Hq, D], k, v [Tk, Hk, D] of bf16 or fp16, any strides, D 64, 128, 256 or 512, Hq a
    multiple of Hk.  Sequence b has the queries ``cu_q[b] .. cu_q[b + 1] - 1`` and the keys of
    ``cu_k`` (int32, from 0 on; None: the same); its last query stands at its last key.  Causal: a
    query sees the keys up to where it stands, with ``window`` the last so many of them.  A query
    that sees none, and rows behind the last sequence, are zero; one whose scores are all minus
    infinity is NaN.  ``scale`` is D^-1/2 if None."""
    index = _gpu_of(q, k, v, cu_q, cu_k)
    dt, q, k, v, heads, cu_q, cu_k, sizes = _attention_args(q, k, v, cu_q, cu_k, scale, causal, window)
    out = _dense_like(q)
    lse = q.new_empty((sizes[3], sizes[1]), dtype=torch.float32) if return_lse else None
    lib = load()
    nbytes = lib.w4a16_attention_workspace_bytes(*sizes[:6], window)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch("w4a16_attention", index, lib.w4a16_attention, *heads, cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(),
            _ptr(lse), dt, *sizes, _ptr(ws), nbytes)
    return (out, lse) if return_lse else out


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor | None = None,
                       scale: float | None = None, causal: bool = True, window: int = 0, needs=(True, True, True)):
    """(dq, dk, dv) of ``attention`` for the gradient ``dout`` of its output and the ``out`` and ``lse`` of
    that forward call.  ``needs``: which of the three are wanted; the others are None."""
    index = _gpu_of(q, k, v, cu_q, cu_k, dout, out, lse)
    dt, q, k, v, heads, cu_q, cu_k, sizes = _attention_args(q, k, v, cu_q, cu_k, scale, causal, window)
    for t, n in ((dout, "dout"), (out, "out")):
        if t.shape != q.shape or t.dtype != q.dtype:
            raise ValueError(f"{n} must be {q.dtype} {list(q.shape)}, got {t.dtype} {list(t.shape)}")
    Tq, Hq = sizes[1], sizes[3]
    if lse.shape != (Hq, Tq) or lse.dtype != torch.float32:
        raise ValueError(f"lse must be float32 {[Hq, Tq]}, got {lse.dtype} {list(lse.shape)}")
    if len(needs) != 3:
        raise ValueError("needs must say for each of dq, dk and dv whether it is wanted")
    dout, pd = _dense(dout)
    out, po = _dense(out)
    lse = lse.contiguous()
    dq = torch.empty_like(dout) if needs[0] else None
    dk, dv = (_dense_like(k), _dense_like(v)) if needs[1] or needs[2] else (None, None)
    lib = load()
    nbytes = lib.w4a16_attention_backward_workspace_bytes(*sizes[:6], window)
    ws = q.new_empty(nbytes, dtype=torch.uint8)
    _launch("w4a16_attention_backward", index, lib.w4a16_attention_backward, pd, *heads, po, lse.data_ptr(),
            cu_q.data_ptr(), cu_k.data_ptr(), _ptr(dq), _ptr(dk), _ptr(dv), dt, *sizes, ws.data_ptr(), nbytes)
    return dq, dk if needs[1] else None, dv if needs[2] else None


def decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                     lengths: torch.Tensor, scale: float | None = None, window: int = 0) -> torch.Tensor:
    """Attention of one new token per sequence over a paged cache -> [B, Hq, D].

    q [B, Hq, D] of bf16 or fp16, any strides; k_cache, v_cache [pages, Hk, page size, D]; sequence
    b's key j lies in row j % page size of page ``block_table[b, j / page size]``; it has
    ``lengths[b]`` of them (both int32), of which the token sees the last ``window`` (0: all).  A
    length of zero gives zeros; a length that the table does not cover, a page that the cache does
    not have, or scores that are all minus infinity NaN.  Tables of few pages (heads of 128 and
    less 1024 keys, 256 512, 512 256) take one launch and no workspace, whatever the lengths."""
    index = _gpu_of(q, k_cache, v_cache, block_table, lengths)
    dt = _head_type(q, "q", False)
    q, heads = _heads(q, "q")
    B, Hq, D = q.shape
    cache, pages, Hk, page = _cache_args(k_cache, v_cache, q.dtype, D)
    _group(Hq, Hk, D)
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be int32 [{B}, pages of a sequence], got {list(block_table.shape)}")
    width = block_table.shape[1]
    block_table = _index(block_table, "block_table", B, width)
    lengths = _index(lengths, "lengths", B)
    out = _dense_like(q)
    lib = load()
    nbytes = lib.w4a16_decode_attention_workspace_bytes(B, Hq, Hk, D, width * page)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch("w4a16_decode_attention", index, lib.w4a16_decode_attention, *heads, *cache,
            block_table.data_ptr(), lengths.data_ptr(), out.data_ptr(), dt, B, Hq, Hk, D, pages, page, width,
            D ** -0.5 if scale is None else scale, window, _ptr(ws), nbytes)
    return out


class MoEStages:
    """The four stages of ``moe_forward`` on one preallocated workspace.

    For callers that schedule or time the stages separately (the benchmark
    times ``gate_up`` alone); ``forward`` runs all four.  Sizes are fixed at
    construction; the workspace carries the routing plan and intermediates
    between stages, so calls must be made in order on one stream.
    """

    def __init__(self, M: int, top_k: int, E: int, H: int, I: int, group_size: int, device):
        self.M, self.k, self.E, self.H, self.I, self.G = M, top_k, E, H, I, group_size
        self.device = torch.device(device)
        self.lib = load()
        nbytes = self.lib.moe_workspace_bytes(max(M, 1), top_k, E, H, I)
        self.ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self.out = torch.empty((M, H), dtype=torch.bfloat16, device=self.device)

    def _dims(self):
        return self.M, self.k, self.E, self.H, self.I

    def plan(self, hidden: torch.Tensor, top_k_index: torch.Tensor) -> None:
        s = _stream(self.device)
        _check(self.lib.moe_plan(_ptr(hidden), _ptr(top_k_index), *self._dims(), self.G, _ptr(self.ws),
                                 self.ws.numel(), s), "moe_plan")

    def gate_up(self, hidden: torch.Tensor, gu_packed: torch.Tensor, gu_scale: torch.Tensor,
                tiles: TiledWeights | None = None) -> None:
        """Grouped gate_up GEMM; ``tiles`` (the stack's TiledWeights) serve the kernels
        that read them."""
        s = _stream(self.device)
        if tiles is None:
            _check(self.lib.moe_gate_up(_ptr(hidden), _ptr(gu_packed), _ptr(gu_scale), *self._dims(), self.G,
                                        _ptr(self.ws), self.ws.numel(), s), "moe_gate_up")
        else:
            st = tiles.struct()
            _check(self.lib.moe_gate_up_tiled(_ptr(hidden), _ptr(gu_packed), _ptr(gu_scale), ctypes.byref(st),
                                              *self._dims(), self.G, _ptr(self.ws), self.ws.numel(), s),
                   "moe_gate_up_tiled")

    def down(self, dn_packed: torch.Tensor, dn_scale: torch.Tensor, tiles: TiledWeights | None = None) -> None:
        """Grouped down GEMM; ``tiles`` serve the kernels that read them."""
        s = _stream(self.device)
        if tiles is None:
            _check(self.lib.moe_down(_ptr(dn_packed), _ptr(dn_scale), *self._dims(), self.G, _ptr(self.ws),
                                     self.ws.numel(), s), "moe_down")
        else:
            st = tiles.struct()
            _check(self.lib.moe_down_tiled(_ptr(dn_packed), _ptr(dn_scale), ctypes.byref(st), *self._dims(),
                                           self.G, _ptr(self.ws), self.ws.numel(), s), "moe_down_tiled")

    def combine(self, top_k_index: torch.Tensor, top_k_weights: torch.Tensor) -> torch.Tensor:
        s = _stream(self.device)
        _check(self.lib.moe_combine(_ptr(top_k_index), _ptr(top_k_weights), _ptr(self.out), *self._dims(),
                                    _ptr(self.ws), self.ws.numel(), s), "moe_combine")
        return self.out

    def forward(self, hidden, top_k_index, top_k_weights, gu_packed, gu_scale, dn_packed, dn_scale):
        for t in (hidden, top_k_index, top_k_weights, gu_packed, gu_scale, dn_packed, dn_scale):
            if not t.is_contiguous() or t.device != self.device:
                raise ValueError("MoEStages.forward expects contiguous tensors on its device")
        self.plan(hidden, top_k_index)
        self.gate_up(hidden, gu_packed, gu_scale)
        self.down(dn_packed, dn_scale)
        return self.combine(top_k_index, top_k_weights)
