"""Matrices of 4-bit blocks: quantisation, products (include/fmoe.h, fmoe_fp4_*).

``"mxfp4"``: 32 values share a power of two. ``"nvfp4"``: 16 values share an e4m3 scale, and a
matrix may have an fp32 global scale ``g`` beside them, which lets the e4m3 scales cover the
matrix's range: ``g = x.abs().amax() / (6 * 448)`` puts the largest block at the top of it.
"""
from __future__ import annotations

import ctypes
import dataclasses

import torch

from . import FMOE_OK, _check_tensor, _raise, load_library
from .router import DTYPE_CODES

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}


class FmoeFp4Matrix(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("global_scale", ctypes.c_void_p), ("rows", ctypes.c_int64),
                ("cols", ctypes.c_int64), ("batch", ctypes.c_int32), ("format", ctypes.c_int32)]


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
        *lead, rows, half = self.codes.shape
        _check_tensor(self.codes, f"{name}.codes", tuple(self.codes.shape), torch.uint8)
        _check_tensor(self.scales, f"{name}.scales",
                      _scale_shape(lead, rows, 2 * half, self.format), torch.uint8)
        g = _global_scale(self.global_scale, lead, self.codes.device, f"{name}.global_scale",
                          self.format)
        if self.scales.device != self.codes.device:
            raise ValueError(f"{name}.codes and {name}.scales must be on the same device")
        return FmoeFp4Matrix(self.codes.data_ptr(), self.scales.data_ptr(), g, rows, 2 * half,
                             lead[0] if lead else 1, FORMATS[self.format])


def _global_scale(g, lead, device, name, format):
    if g is None:
        return None
    if format == "mxfp4":
        raise ValueError(f"{name}: mxfp4 has no global scale")
    if not isinstance(g, torch.Tensor) or g.device != device:
        raise ValueError(f"{name} must be a tensor on {device}")
    if g.numel() != (lead[0] if lead else 1) or not g.is_contiguous():
        raise ValueError(f"{name} must have one contiguous element per matrix")
    if g.dtype != torch.float32:
        raise TypeError(f"{name} dtype mismatch: expected torch.float32, got {g.dtype}")
    return g.data_ptr()


def _call(lib, where, dev, fn, *args):
    with torch.cuda.device(dev):
        rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    if rc != FMOE_OK:
        _raise(lib, rc, where)


def _out(out, shape, dtype, dev):
    if dtype not in DTYPE_CODES:
        raise TypeError(f"output dtype mismatch: expected float32, bfloat16 or float16, got {dtype}")
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    _check_tensor(out, "out", tuple(shape), dtype)
    if out.device != dev:
        raise ValueError(f"out must be on {dev}")
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
    lib = load_library()
    _call(lib, "quantize_fp4", dev, lib.fmoe_fp4_quantize, ctypes.byref(q), x.data_ptr(),
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
    lib = load_library()
    _call(lib, "dequantize_fp4", q.device, lib.fmoe_fp4_dequantize, ctypes.byref(m),
          out.data_ptr(), DTYPE_CODES[dtype])
    return out


def matmul_fp4(a: Fp4Tensor, b: Fp4Tensor, *, dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """``a`` [M, K] times the transpose of ``b`` [N, K], summed in fp32, in ``dtype``."""
    for name, m in (("a", a), ("b", b)):
        if not isinstance(m, Fp4Tensor):
            raise ValueError(f"{name} must be an Fp4Tensor")
    ma, mb = a._matrix("a", (2,)), b._matrix("b", (2,))
    if a.device != b.device:
        raise ValueError("a and b must be on the same device")
    out = _out(out, (a.shape[0], b.shape[0]), dtype, a.device)
    lib = load_library()
    _call(lib, "matmul_fp4", a.device, lib.fmoe_fp4_matmul, ctypes.byref(ma), ctypes.byref(mb),
          out.data_ptr(), DTYPE_CODES[dtype])
    return out
