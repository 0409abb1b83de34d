"""Matrices of 4-bit blocks: quantisation, products (include/fmoe.h, fmoe_fp4_*).

``"mxfp4"``: 32 values share a power of two. ``"nvfp4"``: 16 values share an e4m3 scale, and a
matrix may have an fp32 global scale ``g`` beside them, which lets the e4m3 scales cover the
matrix's range: ``g = x.abs().amax() / (6 * 448)`` puts the largest block at the top of it.
"""
from __future__ import annotations

import ctypes
import dataclasses
import functools

import torch

from . import FMOE_OK, _raise, _raise_device_error, load_library
from .router import DTYPE_CODES, _call, _expect

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}


class FmoeFp4Matrix(ctypes.Structure):
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


def _check_format(format):
    if format not in FORMATS:
        raise ValueError(f"format must be one of {', '.join(FORMATS)}, got {format!r}")


def _scale_shape(lead, rows, cols, format):
    return (*lead, -(-rows // 128), -(-cols // (4 * BLOCK[format])), 512)


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
        _check_format(format)
        if scales.element_size() != 1:
            raise TypeError(f"scales dtype mismatch: expected 8 bits, got {scales.dtype}")
        if tuple(scales.shape) != (*codes.shape[:-1], codes.shape[-1] * 2 // BLOCK[format]):
            raise ValueError("scales must be [..., rows, cols / block]")
        return cls(codes, cls.tile_scales(scales.view(torch.uint8)), format, global_scale)

    def _matrix(self, name, dims):
        """Checked argument block of the C entry points."""
        _check_format(self.format)
        if not isinstance(self.codes, torch.Tensor) or self.codes.dim() not in dims:
            raise ValueError(f"{name}.codes must be {' or '.join(f'{d}D' for d in dims)}")
        codes, dev = self.codes, self.codes.device
        if dev.type != "cuda":
            raise ValueError(f"{name}.codes must be a CUDA tensor")
        *lead, rows, half = codes.shape
        _expect(codes, f"{name}.codes", codes.shape, torch.uint8, dev)
        _expect(self.scales, f"{name}.scales", _scale_shape(lead, rows, 2 * half, self.format),
                torch.uint8, dev)
        g = self.global_scale
        if g is not None:
            g = _global_scale(g, lead, dev, f"{name}.global_scale", self.format)
        return FmoeFp4Matrix(codes.data_ptr(), self.scales.data_ptr(), g, rows, 2 * half,
                             lead[0] if lead else 1, FORMATS[self.format])


def _global_scale(g, lead, dev, name, format):
    if format == "mxfp4":
        raise ValueError(f"{name}: mxfp4 has no global scale")
    if not isinstance(g, torch.Tensor) or g.device != dev:
        raise ValueError(f"{name} must be a tensor on {dev}")
    if g.numel() != (lead[0] if lead else 1) or not g.is_contiguous():
        raise ValueError(f"{name} must have one contiguous element per matrix")
    if g.dtype is not torch.float32:
        raise TypeError(f"{name} dtype mismatch: expected torch.float32, got {g.dtype}")
    return g.data_ptr()


def _out(out, shape, dtype, dev):
    if dtype not in DTYPE_CODES:
        raise TypeError(f"output dtype mismatch: expected float32, bfloat16 or float16, got {dtype}")
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    _expect(out, "out", shape, dtype, dev)
    return out


def quantize_fp4(x: torch.Tensor, format: str, *, global_scale: torch.Tensor | None = None,
                 out: Fp4Tensor | None = None) -> Fp4Tensor:
    """Quantises ``x`` [rows, cols] or [batch, rows, cols] (fp32, bf16 or fp16; cols a multiple
    of 32) to ``format``. ``global_scale`` (nvfp4; fp32 on the device, one element per matrix) is
    used and kept in the result; ``out`` is filled instead of new tensors."""
    _check_format(format)
    if not isinstance(x, torch.Tensor) or x.dim() not in (2, 3):
        raise ValueError("x must be 2D or 3D")
    if x.device.type != "cuda":
        raise ValueError("x must be a CUDA tensor")
    if x.dtype not in DTYPE_CODES:
        raise TypeError(f"x dtype mismatch: expected float32, bfloat16 or float16, got {x.dtype}")
    *lead, rows, cols = x.shape
    if cols % 32 or cols == 0:
        raise ValueError(f"x must have a multiple of 32 columns, got {cols}")
    if x.stride(-1) != 1:
        x = x.contiguous()
    dev = x.device
    if out is None:
        out = Fp4Tensor(torch.empty(*lead, rows, cols // 2, dtype=torch.uint8, device=dev),
                        torch.empty(_scale_shape(lead, rows, cols, format), dtype=torch.uint8,
                                    device=dev), format, global_scale)
    elif out.format != format or tuple(out.shape) != tuple(x.shape) or out.device != dev:
        raise ValueError("out must have the format, shape and device of the result")
    else:
        out.global_scale = global_scale
    if lead and lead[0] == 0:
        return out
    q = out._matrix("out", (x.dim(),))
    _call("quantize_fp4", dev, "fmoe_fp4_quantize", ctypes.byref(q), x.data_ptr(),
          DTYPE_CODES[x.dtype], x.stride(-2), x.stride(0) if lead else 0)
    return out


def dequantize_fp4(q: Fp4Tensor, dtype: torch.dtype = torch.bfloat16, *,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The values ``q`` stands for, in ``dtype`` (fp32, bf16 or fp16)."""
    if not isinstance(q, Fp4Tensor):
        raise ValueError("q must be an Fp4Tensor")
    m = q._matrix("q", (2, 3))
    out = _out(out, q.shape, dtype, q.device)
    if out.numel() == 0:
        return out
    _call("dequantize_fp4", q.device, "fmoe_fp4_dequantize", ctypes.byref(m), out.data_ptr(),
          DTYPE_CODES[dtype])
    return out


def matmul_fp4(a: Fp4Tensor, b: Fp4Tensor, *, dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``a`` [M, K] times the transpose of ``b`` [N, K], summed in fp32, in ``dtype``."""
    for name, m in (("a", a), ("b", b)):
        if not isinstance(m, Fp4Tensor):
            raise ValueError(f"{name} must be an Fp4Tensor")
    ma, mb = a._matrix("a", (2,)), b._matrix("b", (2,))
    if a.codes.device != b.codes.device:
        raise ValueError("a and b must be on the same device")
    out = _out(out, (ma.rows, mb.rows), dtype, a.codes.device)
    _call("matmul_fp4", a.device, "fmoe_fp4_matmul", ctypes.byref(ma), ctypes.byref(mb),
          out.data_ptr(), DTYPE_CODES[dtype])
    return out


def fp4_workspace_bytes(prob: FmoeFp4Problem) -> int:
    """Scratch bytes of a forward_fp4 call with these sizes (fmoe_fp4_workspace_size)."""
    lib = load_library()
    n = ctypes.c_size_t(0)
    rc = lib.fmoe_fp4_workspace_size(ctypes.byref(prob), ctypes.byref(n))
    if rc != FMOE_OK:
        _raise(lib, rc, "fp4_workspace_bytes")
    return int(n.value)


@functools.lru_cache(maxsize=64)
def _workspace_bytes(*sizes):
    return fp4_workspace_bytes(FmoeFp4Problem(*sizes))


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
    ``workspace`` is the caller's scratch (``fp4_workspace_bytes``; one call at a time), ``check``
    as in ``kernel``; a device error of an earlier call raises ``DeviceError``."""
    for name, m in (("w13", w13), ("w2", w2)):
        if not isinstance(m, Fp4Tensor):
            raise ValueError(f"{name} must be an Fp4Tensor")
    if w13.format != w2.format:
        raise ValueError("w13 and w2 must have the same format")
    if not isinstance(hidden_states, torch.Tensor) or hidden_states.dim() != 2:
        raise ValueError("hidden_states must be 2D")
    if not isinstance(topk_idx, torch.Tensor) or topk_idx.dim() != 2:
        raise ValueError("topk_idx must be 2D")
    if hidden_states.dtype not in DTYPE_CODES:
        raise TypeError(f"hidden_states dtype mismatch: expected float32, bfloat16 or float16, got "
                        f"{hidden_states.dtype}")
    m13, m2 = w13._matrix("w13", (3,)), w2._matrix("w2", (3,))
    dev = w13.codes.device
    T, K = topk_idx.shape
    E, H, I = m13.batch, m13.cols, m13.rows // 2
    if m13.rows % 2 or (m2.batch, m2.rows, m2.cols) != (E, H, I):
        raise ValueError(f"w13 must be [E, 2I, H] and w2 [E, H, I], got {w13.shape} and {w2.shape}")
    if w2.codes.device != dev:
        raise ValueError("w13 and w2 must be on the same device")
    _expect(hidden_states, "hidden_states", (T, H), hidden_states.dtype, dev)
    _expect(topk_idx, "topk_idx", (T, K), torch.int32, dev)
    _expect(topk_w, "topk_w", (T, K), torch.float32, dev)
    scales = [None if g is None else _global_scale(g, [], dev, name, w13.format)
              for name, g in (("input_scale", input_scale),
                              ("intermediate_scale", intermediate_scale))]
    sizes = (T, H, I, E, K, int(local_expert_offset), m13.format, DTYPE_CODES[hidden_states.dtype])
    prob = FmoeFp4Problem(*sizes)
    nbytes = _workspace_bytes(*sizes)
    _raise_device_error(dev, "an earlier call on this device")
    out = _out(out, (T, H), torch.bfloat16, dev)
    if T == 0:
        return out
    if workspace is None:
        # from the allocator, which orders it with this stream and keeps it for a capturing graph
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    elif workspace.device != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous on {dev}")
    t = FmoeFp4Tensors(hidden_states.data_ptr(), topk_idx.data_ptr(), topk_w.data_ptr(),
                       m13.codes, m13.scales, m13.global_scale, m2.codes, m2.scales,
                       m2.global_scale, *scales, out.data_ptr())
    _call("forward_fp4", dev, "fmoe_fp4_forward", ctypes.byref(prob), ctypes.byref(t),
          workspace.data_ptr(), workspace.numel() * workspace.element_size())
    if check:
        torch.cuda.current_stream(dev).synchronize()
        _raise_device_error(dev, "this call")
    return out
