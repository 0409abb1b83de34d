"""Expert routing for any scoring rule, with its gradient.

``route`` in the package serves the reference operator's one rule (sigmoid scores, a bf16
bias, groups; ``solution/cuda/kernel.cu:388-516``) bit for bit. ``route_experts`` takes softmax
or sigmoid scores, an optional bias, optional groups, and logits of three types, and is
differentiable.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util

import torch

from . import LIB_PATH, load_library

_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"top2": 0, "max": 1}
_module = None


class FmoeRouter(ctypes.Structure):
    """The C argument block, for callers of the C ABI (fmoe_route_experts) through ctypes."""

    _fields_ = [("num_tokens", ctypes.c_int64), ("logits_stride", ctypes.c_int64),
                ("num_experts", ctypes.c_int32), ("top_k", ctypes.c_int32),
                ("n_group", ctypes.c_int32), ("topk_group", ctypes.c_int32),
                ("score", ctypes.c_int32), ("group_score", ctypes.c_int32),
                ("renormalize", ctypes.c_int32), ("logits_dtype", ctypes.c_int32),
                ("bias_dtype", ctypes.c_int32), ("scale", ctypes.c_float)]


def binding():
    """The compiled entry points (lib/fmoe_torch.so, csrc/torch_binding.cpp)."""
    global _module
    if _module is None:
        load_library()
        path = LIB_PATH.with_name("fmoe_torch.so")
        if not path.exists():
            raise RuntimeError(f"torch binding not built: {path} (run `python "
                               f"fused-moe-yws_b200/build.py`)")
        built = path.with_suffix(".version")  # compiled code of another torch may crash this one
        if built.exists() and built.read_text() != torch.__version__:
            raise RuntimeError(f"torch binding built for torch {built.read_text()}, this is "
                               f"{torch.__version__} (run `python fused-moe-yws_b200/build.py`)")
        loader = importlib.machinery.ExtensionFileLoader("fmoe_torch", str(path))
        spec = importlib.util.spec_from_file_location("fmoe_torch", path, loader=loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        _module = module
    return _module


def code(table, value, name):
    if value not in table:
        raise ValueError(f"{name} must be one of {', '.join(table)}, got {value!r}")
    return table[value]


def _forward(logits, bias, top_k, score, n_group, topk_group, group_score, renormalize, scale):
    return (_module or binding()).route_experts(
        logits, top_k, code(_SCORES, score, "score"), bias, n_group, topk_group,
        code(_GROUP_SCORES, group_score, "group_score"), renormalize, scale)


def route_experts_backward(grad_w: torch.Tensor, logits: torch.Tensor, topk_idx: torch.Tensor, *,
                           score: str = "softmax", renormalize: bool = True, scale: float = 1.0):
    """The gradient of the logits from that of the weights (fmoe_route_experts_backward).

    ``topk_idx`` [T, K] are the picks of ``route_experts``, ``grad_w`` fp32 [T, K]; ``score``,
    ``renormalize`` and ``scale`` as there (groups and bias only decide the picks). Returns
    [T, E] in the logits' type."""
    return (_module or binding()).route_experts_backward(
        grad_w, logits, topk_idx, code(_SCORES, score, "score"), renormalize, scale)


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
    that of the logits, with a bias that of the biased scores in 64 bits. ``group_score`` is "top2" (sum of a group's two best) or "max".
    With ``renormalize`` the picked weights sum to ``scale``. Differentiable in the logits, the
    picks held fixed, in reverse mode alone (a forward-mode tangent is refused); the bias gets no
    gradient. The results go to ``forward_fp4`` or ``forward_routed``, which have no backward pass;
    the gradient is for a training program's own expert layer."""
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return _RouteExperts.apply(logits, bias, top_k, score, n_group, topk_group, group_score,
                                   renormalize, scale)
    return _forward(logits, bias, top_k, score, n_group, topk_group, group_score, renormalize,
                    scale)
