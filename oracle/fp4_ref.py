"""The 4-bit block formats on the CPU, from the definition in include/fmoe.h, for the tests."""
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def nearest_code(a):
    """The code of the grid value nearest to a >= 0 (float64), ties to the even code."""
    # (from 2^53 on a float64 difference would not tell 4 from 6)
    d = (a.clamp(max=8.0)[..., None] - GRID).abs()
    best = d.amin(-1, keepdim=True)
    tie = d == best
    order = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7])  # even codes first
    return torch.where(tie, order, 8).argmin(-1)


def quantize(x, fmt, g=None):
    """(codes uint8 [..., K], scale bytes uint8 [..., K / block]) of x; g is a float or None."""
    block = BLOCK[fmt]
    v = x.float().unflatten(-1, (-1, block))
    top = v.abs().amax(-1)
    top = torch.where(torch.isnan(v).any(-1), float("nan"), top)
    bad = ~torch.isfinite(top)
    fine = torch.where(bad, 1.0, top)
    if fmt == "mxfp4":
        e = torch.frexp(fine.double()).exponent - 1 - 2
        e = torch.where(fine == 0, -127, e).clamp(min=-127)
        scale = torch.where(bad, 255, e + 127).to(torch.uint8)
        q = torch.ldexp(v.double(), -e[..., None])
    else:
        g32 = torch.tensor(1.0 if g is None else g, dtype=torch.float32)
        s = (fine / (torch.tensor(6.0) * g32)).clamp(max=448.0).to(torch.float8_e4m3fn)
        scale = torch.where(bad, 127, s.view(torch.uint8))
        d = s.float() * g32
        q = torch.where(d[..., None] > 0, v / d[..., None], 0.0).double()
    q = torch.where(torch.isfinite(q), q, 0.0)
    code = nearest_code(q.abs()) + 8 * torch.signbit(v)
    return code.to(torch.uint8).flatten(-2), scale


def scale_values(scale, fmt):
    if fmt == "mxfp4":
        return torch.where(scale == 255, float("nan"), torch.exp2(scale.double() - 127))
    return scale.view(torch.float8_e4m3fn).double()


def values(codes, scale, fmt):
    """float64 values without the global scale."""
    v = GRID[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)
    return v * scale_values(scale, fmt).repeat_interleave(BLOCK[fmt], -1)


def unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def pack(codes):
    c = codes.unflatten(-1, (-1, 2))
    return c[..., 0] | (c[..., 1] << 4)


def untile(tiles, rows, blocks):
    """Scale bytes [..., rows, blocks] from the tile layout, byte by byte."""
    r, b = torch.arange(rows)[:, None], torch.arange(blocks)[None, :]
    return tiles[..., r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4]
