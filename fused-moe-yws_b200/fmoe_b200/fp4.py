"""Matrices of 4-bit blocks: quantisation, products (include/fmoe.h, fmoe_fp4_*).

``"mxfp4"``: 32 values share a power of two. ``"nvfp4"``: 16 values share an e4m3 scale, and a
matrix may have an fp32 global scale ``g`` beside them, which lets the e4m3 scales cover the
matrix's range: ``g = x.abs().amax() / (6 * 448)`` puts the largest block at the top of it.
"""
from __future__ import annotations

import ctypes
import dataclasses

import torch

from . import FMOE_OK, _raise, load_library, router
from .router import binding, code

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}


class FmoeFp4Matrix(ctypes.Structure):
    """The C argument blocks, for callers of the C ABI (fmoe_fp4_*) through ctypes."""

    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("global_scale", ctypes.c_void_p), ("rows", ctypes.c_int64),
                ("cols", ctypes.c_int64), ("batch", ctypes.c_int32), ("format", ctypes.c_int32)]


class FmoeFp4Problem(ctypes.Structure):
    _fields_ = [("num_tokens", ctypes.c_int64), ("hidden_size", ctypes.c_int32),
                ("intermediate_size", ctypes.c_int32), ("num_local_experts", ctypes.c_int32),
                ("top_k", ctypes.c_int32), ("local_expert_offset", ctypes.c_int32),
                ("format", ctypes.c_int32), ("dtype", ctypes.c_int32)]


class FmoeFp4Tensors(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in (
        "hidden_states", "topk_idx", "topk_w", "w13", "w13_scales", "w13_global", "w2",
        "w2_scales", "w2_global", "input_scale", "intermediate_scale", "output")]


@dataclasses.dataclass
class Fp4Tensor:
    """A 4-bit matrix [rows, cols], or a stack of them [batch, rows, cols].

    ``codes`` uint8 [..., rows, cols / 2], ``scales`` uint8 [..., ceil(rows / 128),
    ceil(cols / (4 block)), 512] in the tensor cores' layout (include/fmoe.h),
    ``global_scale`` fp32, one element per matrix, or None. ``from_rows`` takes scales that lie
    row by row, as checkpoints hold them."""

    codes: torch.Tensor
    scales: torch.Tensor
    format: str
    global_scale: torch.Tensor | None = None

    @property
    def shape(self) -> tuple:
        return (*self.codes.shape[:-1], self.codes.shape[-1] * 2)

    @property
    def device(self):
        return self.codes.device

    @staticmethod
    def tile_scales(scales: torch.Tensor) -> torch.Tensor:
        """Scale bytes [..., rows, blocks] in the tensor cores' layout (a new tensor)."""
        *lead, M, B = scales.shape
        m, b, n = -(-M // 128), -(-B // 4), len(lead)
        full = scales.new_zeros(*lead, m * 128, b * 4)
        full[..., :M, :B] = scales
        full = full.view(*lead, m, 4, 32, b, 4)
        return full.permute(*range(n), n, n + 3, n + 2, n + 1, n + 4).reshape(
            *lead, m, b, 512).contiguous()

    @classmethod
    def from_rows(cls, codes, scales, format, global_scale=None) -> "Fp4Tensor":
        """From scales [..., rows, cols / block] (uint8, or the 8-bit float type itself)."""
        code(FORMATS, format, "format")
        if scales.element_size() != 1:
            raise TypeError(f"scales dtype mismatch: expected 8 bits, got {scales.dtype}")
        if tuple(scales.shape) != (*codes.shape[:-1], codes.shape[-1] * 2 // BLOCK[format]):
            raise ValueError("scales must be [..., rows, cols / block]")
        return cls(codes, cls.tile_scales(scales.view(torch.uint8)), format, global_scale)


def quantize_fp4(x: torch.Tensor, format: str, *, global_scale: torch.Tensor | None = None,
                 out: Fp4Tensor | None = None) -> Fp4Tensor:
    """Quantises ``x`` [rows, cols] or [batch, rows, cols] (fp32, bf16 or fp16; cols a multiple
    of 32) to ``format``. ``global_scale`` (nvfp4; fp32 on the device, one element per matrix) is
    used and kept in the result; ``out`` is filled instead of new tensors."""
    number = code(FORMATS, format, "format")
    held = (None, None)
    if out is not None:
        if not isinstance(out, Fp4Tensor) or out.format != format:
            raise ValueError("out must have the format, shape and device of the result")
        held = (out.codes, out.scales)
    codes, scales = (router._module or binding()).quantize_fp4(x, number, global_scale, *held)
    if out is None:
        return Fp4Tensor(codes, scales, format, global_scale)
    out.global_scale = global_scale
    return out


def dequantize_fp4(q: Fp4Tensor, dtype: torch.dtype = torch.bfloat16, *,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The values ``q`` stands for, in ``dtype`` (fp32, bf16 or fp16)."""
    if not isinstance(q, Fp4Tensor):
        raise ValueError("q must be an Fp4Tensor")
    return (router._module or binding()).dequantize_fp4(
        q.codes, q.scales, q.global_scale, code(FORMATS, q.format, "format"), dtype, out)


def matmul_fp4(a: Fp4Tensor, b: Fp4Tensor, *, dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None, check: bool = False) -> torch.Tensor:
    """``a`` [M, K] times the transpose of ``b`` [N, K], summed in fp32, in ``dtype``. ``check`` as
    in ``kernel``; a device error of an earlier call raises ``DeviceError``."""
    for name, m in (("a", a), ("b", b)):
        if not isinstance(m, Fp4Tensor):
            raise ValueError(f"{name} must be an Fp4Tensor")
    return (router._module or binding()).matmul_fp4(
        a.codes, a.scales, a.global_scale, code(FORMATS, a.format, "format"), b.codes, b.scales,
        b.global_scale, code(FORMATS, b.format, "format"), dtype, out, check)


def fp4_workspace_bytes(prob: FmoeFp4Problem) -> int:
    """Scratch bytes of a forward_fp4 call with these sizes (fmoe_fp4_workspace_size)."""
    lib = load_library()
    n = ctypes.c_size_t(0)
    rc = lib.fmoe_fp4_workspace_size(ctypes.byref(prob), ctypes.byref(n))
    if rc != FMOE_OK:
        _raise(lib, rc, "fp4_workspace_bytes")
    return int(n.value)


def forward_fp4(hidden_states: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor,
                w13: Fp4Tensor, w2: Fp4Tensor, local_expert_offset: int = 0, *,
                input_scale: torch.Tensor | None = None,
                intermediate_scale: torch.Tensor | None = None, out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None, check: bool = False) -> torch.Tensor:
    """The expert layer on 4-bit weights; returns bf16 [T, H] (fmoe_fp4_forward).

    ``hidden_states`` [T, H] (fp32, bf16 or fp16) are quantised by the call, ``topk_idx`` int32 /
    ``topk_w`` fp32 [T, K] come from ``route_experts`` or ``route``. ``w13`` [E_local, 2I, H] (gate
    rows, then up rows; the SiLU is on the up half, as in ``kernel``) and ``w2`` [E_local, H, I]
    hold experts [offset, offset + E_local); picks outside take no part. ``input_scale`` and
    ``intermediate_scale`` (nvfp4, fp32 [1] on the device) are the activations' global scales.
    There is no backward pass: ``hidden_states`` or ``topk_w`` that require a gradient are refused
    outside ``torch.no_grad()``.
    ``workspace`` is the caller's scratch (``fp4_workspace_bytes``; one call at a time), ``check``
    as in ``kernel``; a device error of an earlier call raises ``DeviceError``."""
    for name, m in (("w13", w13), ("w2", w2)):
        if not isinstance(m, Fp4Tensor):
            raise ValueError(f"{name} must be an Fp4Tensor")
    return (router._module or binding()).forward_fp4(
        hidden_states, topk_idx, topk_w, w13.codes, w13.scales, w13.global_scale,
        code(FORMATS, w13.format, "format"), w2.codes, w2.scales, w2.global_scale,
        code(FORMATS, w2.format, "format"), local_expert_offset, input_scale, intermediate_scale,
        out, workspace, check)
