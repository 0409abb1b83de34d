"""Expert routing for any scoring rule, with its gradient.

``route`` in the package serves the reference operator's one rule (sigmoid scores, a bf16
bias, groups; ``solution/cuda/kernel.cu:388-516``) bit for bit. ``route_experts`` takes softmax
or sigmoid scores, an optional bias, optional groups, and logits of three types, and is
differentiable.
"""
from __future__ import annotations

import ctypes

import torch

from . import FMOE_OK, FmoeRouteOut, _check_tensor, _raise, load_library

# the current stream's handle without a Stream object around it (half the host time of a call)
_stream_handle = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)

DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"top2": 0, "max": 1}


class FmoeRouter(ctypes.Structure):
    _fields_ = [("num_tokens", ctypes.c_int64), ("logits_stride", ctypes.c_int64),
                ("num_experts", ctypes.c_int32), ("top_k", ctypes.c_int32),
                ("n_group", ctypes.c_int32), ("topk_group", ctypes.c_int32),
                ("score", ctypes.c_int32), ("group_score", ctypes.c_int32),
                ("renormalize", ctypes.c_int32), ("logits_dtype", ctypes.c_int32),
                ("bias_dtype", ctypes.c_int32), ("scale", ctypes.c_float)]


def _code(table, value, name):
    if value not in table:
        raise ValueError(f"{name} must be one of {', '.join(table)}, got {value!r}")
    return table[value]


def _expect(t, name, shape, dtype, dev):
    """_check_tensor and the device, in one test for the arguments that are as they should be."""
    if not (isinstance(t, torch.Tensor) and t.shape == shape and t.dtype is dtype
            and t.device == dev and t.is_contiguous()):
        _check_tensor(t, name, shape, dtype)
        raise ValueError(f"{name} must be on {dev}, got {t.device}")


def _call(where, dev, name, *args):
    """The library's function `name` on dev's current stream; raises what it reports."""
    lib = load_library()
    if dev.index == torch.cuda.current_device():
        rc = getattr(lib, name)(*args, _stream_handle(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = getattr(lib, name)(*args, _stream_handle(dev.index))
    if rc != FMOE_OK:
        _raise(lib, rc, where)


def _logits(logits):
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2:
        raise ValueError("logits must be 2D")
    if logits.device.type != "cuda":
        raise ValueError("logits must be a CUDA tensor")
    if logits.dtype not in DTYPE_CODES:
        raise TypeError(f"logits dtype mismatch: expected float32, bfloat16 or float16, got "
                        f"{logits.dtype}")
    # rows may be padded; anything else (transposed, broadcast) is laid out first
    E = logits.shape[1]
    if logits.stride(1) != 1 and E > 1 or logits.stride(0) < E and logits.shape[0] > 1:
        logits = logits.contiguous()
    return logits


def _router(logits, top_k, score, n_group, topk_group, group_score, renormalize, scale,
            bias_dtype=torch.float32):
    T, E = logits.shape
    return FmoeRouter(T, logits.stride(0) if T > 1 else E, E, int(top_k), int(n_group),
                      int(topk_group), _code(_SCORES, score, "score"),
                      _code(_GROUP_SCORES, group_score, "group_score"), int(bool(renormalize)),
                      DTYPE_CODES[logits.dtype], DTYPE_CODES[bias_dtype], float(scale))


def _forward(logits, bias, top_k, score, n_group, topk_group, group_score, renormalize, scale):
    logits = _logits(logits)
    T, E = logits.shape
    bias_dtype = torch.float32
    if bias is not None:
        if not isinstance(bias, torch.Tensor):
            raise ValueError("bias must be a torch.Tensor")
        bias_dtype = bias.dtype
        if bias_dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"bias dtype mismatch: expected float32 or bfloat16, got {bias_dtype}")
        _expect(bias, "bias", (E,), bias_dtype, logits.device)
    r = _router(logits, top_k, score, n_group, topk_group, group_score, renormalize, scale,
                bias_dtype)
    dev = logits.device
    idx = torch.empty(T, max(int(top_k), 0), dtype=torch.int32, device=dev)
    w = torch.empty(T, max(int(top_k), 0), dtype=torch.float32, device=dev)
    out = FmoeRouteOut(idx.data_ptr(), w.data_ptr())
    _call("route_experts", dev, "fmoe_route_experts", ctypes.byref(r), logits.data_ptr(),
          None if bias is None else bias.data_ptr(), ctypes.byref(out))
    return idx, w


def route_experts_backward(grad_w: torch.Tensor, logits: torch.Tensor, topk_idx: torch.Tensor, *,
                           score: str = "softmax", renormalize: bool = True, scale: float = 1.0):
    """The gradient of the logits from that of the weights (fmoe_route_experts_backward).

    ``topk_idx`` [T, K] are the picks of ``route_experts``, ``grad_w`` fp32 [T, K]; ``score``,
    ``renormalize`` and ``scale`` as there (groups and bias only decide the picks). Returns
    [T, E] in the logits' type."""
    logits = _logits(logits)
    T, E = logits.shape
    if not isinstance(topk_idx, torch.Tensor) or topk_idx.dim() != 2:
        raise ValueError("topk_idx must be 2D")
    K = topk_idx.shape[1]
    dev = logits.device
    _expect(topk_idx, "topk_idx", (T, K), torch.int32, dev)
    if isinstance(grad_w, torch.Tensor):
        grad_w = grad_w.contiguous()  # a gradient may arrive broadcast
    _expect(grad_w, "grad_w", (T, K), torch.float32, dev)
    r = _router(logits, K, score, 1, 1, "top2", renormalize, scale)
    out = torch.empty(T, E, dtype=logits.dtype, device=dev)
    _call("route_experts_backward", dev, "fmoe_route_experts_backward", ctypes.byref(r),
          grad_w.data_ptr(), logits.data_ptr(), topk_idx.data_ptr(), out.data_ptr())
    return out


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, top_k, score, n_group, topk_group, group_score, renormalize,
                scale):
        idx, w = _forward(logits, bias, top_k, score, n_group, topk_group, group_score,
                          renormalize, scale)
        ctx.save_for_backward(logits, idx)
        ctx.how = dict(score=score, renormalize=renormalize, scale=scale)
        ctx.mark_non_differentiable(idx)
        return idx, w

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, grad_w):
        logits, idx = ctx.saved_tensors
        grad = route_experts_backward(grad_w, logits, idx, **ctx.how)
        return (grad,) + (None,) * 8


def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax",
                  bias: torch.Tensor | None = None, n_group: int = 1, topk_group: int = 1,
                  group_score: str = "top2", renormalize: bool = True, scale: float = 1.0):
    """Routes each token to ``top_k`` experts: (topk_idx int32 [T, K], topk_w fp32 [T, K]).

    ``logits`` [T, E] (fp32, bf16 or fp16; E <= 1024), ``bias`` [E] (fp32 or bf16) is added to
    the scores for the choice only. The rule is that of fmoe_route_experts (include/fmoe.h): an
    expert with a logit of -inf or NaN is never picked, a token with fewer than ``top_k`` usable
    experts gets -1 with weight 0 in the places left, ties go to the lower index and the order is
    that of exact arithmetic. ``group_score`` is "top2" (sum of a group's two best) or "max".
    With ``renormalize`` the picked weights sum to ``scale``. Differentiable in the logits, the
    picks held fixed; the bias gets no gradient. The results go to ``forward_fp4`` or
    ``forward_routed``."""
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return _RouteExperts.apply(logits, bias, top_k, score, n_group, topk_group, group_score,
                                   renormalize, scale)
    return _forward(logits, bias, top_k, score, n_group, topk_group, group_score, renormalize,
                    scale)
