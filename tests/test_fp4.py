"""quantize_fp4, dequantize_fp4 and matmul_fp4 against the definition on the CPU.

Codes, scales and dequantised values are compared exactly. Product tolerance: the operands'
products are exact in fp32 (4 significant bits of codes times 8 of two e4m3 scales); a sum of K
of them rounds at most once per step, in the tensor core to the alignment of the largest term:
below K 2^-23 of the sum of magnitudes sum |a||b|, and the result's own rounding (eps / 2).
"""
import ctypes

import pytest
import torch

from oracle import fp4_ref as ref

FORMATS = ["mxfp4", "nvfp4"]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _values(rows, cols, kind, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if kind == "ties":  # multiples of 1/4 with a block maximum of 6: every midpoint of the grid
        x = torch.randint(-24, 25, (rows, cols), generator=g) / 4.0
        x[:, ::16] = 6.0
    elif kind == "range":  # magnitudes from the smallest to the largest
        x = x * torch.exp2(torch.randint(-60, 60, (rows, cols // 16), generator=g).float()
                           ).repeat_interleave(16, 1)
    elif kind == "special":
        x[0, :16] = 0.0
        x[-1, 5] = float("inf")
        x[rows // 2, cols - 1] = float("nan")
        x[rows // 3, 16:32] = -0.0
        x[rows // 3, 0] = 1e-38
    return x


def _check(q, x, fmt, g=None):
    codes, scale = ref.quantize(x, fmt, g)
    rows, cols = x.shape
    got = ref.untile(q.scales.cpu(), rows, cols // ref.BLOCK[fmt])
    assert torch.equal(got, scale)
    nan = scale.eq(255 if fmt == "mxfp4" else 127).repeat_interleave(ref.BLOCK[fmt], -1)
    assert torch.equal(ref.unpack(q.codes.cpu())[~nan], codes[~nan])
    # every byte past the edge is zero
    edge = q.scales.cpu().clone()
    r, b = torch.arange(rows)[:, None], torch.arange(cols // ref.BLOCK[fmt])[None, :]
    edge[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4] = 0
    assert not edge.any()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("g", [None, 2.0 ** -9, 2.0 ** 110])
def test_zeros_keep_their_sign(fmoe, fmt, dtype, g):
    """Zeros of both signs among other values, and alone; a global scale that takes the other way
    to the quotients."""
    if fmt == "mxfp4" and g is not None:
        pytest.skip("mxfp4 has no global scale")
    x = _values(40, 96, "normal", 1)
    x = x * torch.randint(0, 2, x.shape, generator=torch.Generator().manual_seed(2))
    x[3] = -0.0
    x = x.to(dtype)
    assert (torch.signbit(x) & (x == 0)).sum() > 500
    gd = None if g is None else torch.tensor(g, device="cuda")
    _check(fmoe.quantize_fp4(x.cuda(), fmt, global_scale=gd), x, fmt, g)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["normal", "ties", "range", "special"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (128, 256), (129, 288), (257, 1056)])
def test_quantize_and_back(fmoe, fmt, dtype, kind, rows, cols):
    x = _values(rows, cols, kind, rows + cols)
    if dtype == torch.float16 and kind == "range":
        x = x.clamp(-60000.0, 60000.0)
    x = x.to(dtype)
    for g in ([None] if fmt == "mxfp4" else [None, 0.0123]):
        gd = None if g is None else torch.tensor(g, device="cuda")
        q = fmoe.quantize_fp4(x.cuda(), fmt, global_scale=gd)
        assert q.shape == (rows, cols)
        _check(q, x, fmt, g)
        codes, scale = ref.quantize(x, fmt, g)
        codes = ref.unpack(q.codes.cpu())  # a NaN block's codes are free
        scales = ref.scale_values(scale, fmt).float()
        if g is not None:
            scales = scales * torch.tensor(g)
        want = ref.values(codes, torch.full_like(scale, 127 if fmt == "mxfp4" else 0x38), fmt
                          ).float() * scales.repeat_interleave(ref.BLOCK[fmt], -1)
        for to in TYPES:
            got = fmoe.dequantize_fp4(q, to)
            assert got.dtype == to
            assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=-7.0),
                               torch.nan_to_num(want.to(to).float(), nan=-7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_batches_and_strides(fmoe, fmt):
    """Stacks with a global scale each; rows inside a wider matrix, at odd offsets, transposed."""
    x = torch.randn(3, 70, 96, generator=torch.Generator().manual_seed(0)).cuda()
    gs = [0.01, 0.5, 3.0]
    g = torch.tensor(gs, device="cuda") if fmt == "nvfp4" else None
    q = fmoe.quantize_fp4(x, fmt, global_scale=g)
    back = fmoe.dequantize_fp4(q, torch.float32)
    for e in range(3):
        one = fmoe.Fp4Tensor(q.codes[e], q.scales[e], fmt, None if g is None else g[e:e + 1])
        _check(one, x[e].cpu(), fmt, gs[e] if g is not None else None)
        assert torch.equal(fmoe.dequantize_fp4(one, torch.float32), back[e])
    wide = torch.randn(40, 333, generator=torch.Generator().manual_seed(1)).cuda()
    for y in (wide[:, 5:5 + 64], wide[::3, 1:33], wide.bfloat16()[:, 3:67], wide.t()[:64, :32],
              wide[:1, :64].expand(9, 64), wide.half()[:, :320]):
        _check(fmoe.quantize_fp4(y, fmt), y.cpu(), fmt)


@pytest.mark.gpu
def test_quantize_into_given_tensors(fmoe):
    x = torch.randn(130, 64, device="cuda")
    q = fmoe.quantize_fp4(x, "nvfp4")
    held = fmoe.Fp4Tensor(torch.empty_like(q.codes), torch.empty_like(q.scales), "nvfp4")
    assert fmoe.quantize_fp4(x, "nvfp4", out=held) is held
    assert torch.equal(held.codes, q.codes) and torch.equal(held.scales, q.scales)
    empty = fmoe.quantize_fp4(x[:0], "mxfp4")
    assert empty.shape == (0, 64) and fmoe.dequantize_fp4(empty).shape == (0, 64)
    b = fmoe.quantize_fp4(x, "mxfp4")
    assert fmoe.matmul_fp4(empty, b).shape == (0, 130)
    assert fmoe.matmul_fp4(b, empty).shape == (130, 0)


def _operand(rows, cols, fmt, g, seed):
    """A matrix of every code and scales over a range, and its values."""
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (rows, cols), generator=gen, dtype=torch.uint8)
    low, high = (120, 135) if fmt == "mxfp4" else (0x20, 0x48)
    scale = torch.randint(low, high, (rows, cols // ref.BLOCK[fmt]), generator=gen,
                          dtype=torch.uint8)
    return codes, scale, ref.values(codes, scale, fmt) * (1.0 if g is None else g)


def _held(fmoe, codes, scale, fmt, g=None):
    return fmoe.Fp4Tensor.from_rows(ref.pack(codes).cuda(), scale.cuda(), fmt,
                                    None if g is None else torch.tensor(g, device="cuda"))


def _close(got, a, b, dtype):
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    half = torch.finfo(dtype).eps / 2
    bound = want.abs() * half + size * a.shape[1] * 2.0 ** -23 * (1 + half)
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), (off / bound.clamp(min=1e-300)).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 32), (1, 128, 256), (7, 40, 64), (16, 4096, 512), (33, 129, 96), (128, 256, 1024),
    (129, 255, 2080), (300, 300, 288), (1, 5000, 7168), (257, 1, 160), (64, 520, 4128),
    (1500, 3400, 1056), (4999, 1057, 288), (200, 19000, 544),
    (16, 300, 2080), (7, 4096, 1024), (32, 1000, 4128), (1, 8, 1056), (31, 9000, 2048)])
def test_matmul(fmoe, fmt, M, N, K):
    ca, sa, a = _operand(M, K, fmt, None, M + K)
    cb, sb, b = _operand(N, K, fmt, None, N + K + 1)
    qa, qb = _held(fmoe, ca, sa, fmt), _held(fmoe, cb, sb, fmt)
    for dtype in TYPES:
        if dtype == torch.float16 and (a @ b.t()).abs().max() > 60000:
            continue
        got = fmoe.matmul_fp4(qa, qb, dtype=dtype)
        assert got.dtype == dtype and got.shape == (M, N)
        _close(got, a, b, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("ga,gb", [(0.25, None), (None, 3.0), (0.0123, 7.7)])
def test_matmul_global_scales(fmoe, ga, gb):
    ca, sa, a = _operand(40, 320, "nvfp4", None, 1)
    cb, sb, b = _operand(72, 320, "nvfp4", None, 2)
    got = fmoe.matmul_fp4(_held(fmoe, ca, sa, "nvfp4", ga), _held(fmoe, cb, sb, "nvfp4", gb),
                          dtype=torch.float32)
    f = torch.tensor(1.0 if ga is None else ga) * torch.tensor(1.0 if gb is None else gb)
    _close(got / f.cuda(), a, b, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_matmul_single_elements(fmoe, fmt):
    """One nonzero value a row: every (row, column) of the operands and of their scales is read
    from its own place."""
    for M, N, K in ((200, 96, 544), (130, 300, 288)):
        gen = torch.Generator().manual_seed(M)
        ca, cb = (torch.zeros(r, K, dtype=torch.uint8) for r in (M, N))
        k = torch.randint(0, K, (N,), generator=gen)
        cb[torch.arange(N), k] = torch.randint(1, 8, (N,), generator=gen, dtype=torch.uint8)
        ca = torch.randint(0, 16, (M, K), generator=gen, dtype=torch.uint8)
        _, sa, _ = _operand(M, K, fmt, None, 3)
        _, sb, _ = _operand(N, K, fmt, None, 4)
        got = fmoe.matmul_fp4(_held(fmoe, ca, sa, fmt), _held(fmoe, cb, sb, fmt),
                              dtype=torch.float32)
        want = ref.values(ca, sa, fmt) @ ref.values(cb, sb, fmt).t()
        assert torch.equal(got.cpu().double(), want)  # single products are exact


@pytest.mark.gpu
def test_matmul_nan_blocks_reach_their_rows_only(fmoe):
    x = torch.randn(140, 256, generator=torch.Generator().manual_seed(0))
    x[133, 70] = float("nan")
    w = torch.randn(50, 256, generator=torch.Generator().manual_seed(1))
    w[3, 0] = float("inf")
    for fmt in FORMATS:
        y = fmoe.matmul_fp4(fmoe.quantize_fp4(x.cuda(), fmt), fmoe.quantize_fp4(w.cuda(), fmt))
        nan = torch.isnan(y).cpu()
        want = torch.zeros(140, 50, dtype=torch.bool)
        want[133] = True
        want[:, 3] = True
        assert torch.equal(nan, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_then_multiply(fmoe, fmt):
    """The operators together: activations and weights quantised, multiplied, against the values
    that they stand for; captured and replayed on other inputs; on a side stream; twice alike."""
    x = torch.randn(77, 512, generator=torch.Generator().manual_seed(0)).cuda()
    w = (torch.randn(200, 512, generator=torch.Generator().manual_seed(1)) / 20).cuda()
    g = w.abs().amax() / 2688 if fmt == "nvfp4" else None
    qw = fmoe.quantize_fp4(w, fmt, global_scale=g)
    call = lambda: fmoe.matmul_fp4(fmoe.quantize_fp4(x, fmt), qw, dtype=torch.float32)  # noqa: E731
    first = call()
    assert torch.equal(first, call())
    a = fmoe.dequantize_fp4(fmoe.quantize_fp4(x, fmt), torch.float32).cpu().double()
    b = fmoe.dequantize_fp4(qw, torch.float32).cpu().double()
    # b's fp32 values are the code times a rounded scale: 2^-24, as is the product's factor
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    assert ((first.cpu().double() - want).abs() <= size * (512 * 2.0 ** -23 + 2.0 ** -22)).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert torch.equal(got, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for seed in (5, 6):
        x.copy_(torch.randn(77, 512, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        assert torch.equal(held, call())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(7, 300, 2080), (32, 9000, 2048), (300, 300, 288),
                                   (1000, 4000, 288), (33, 129, 96)])
@pytest.mark.parametrize("ga,gb", [(2.6e-23, 2.6e-23), (3e-22, 4e-22), (1e-30, 1e-9),
                                   (1e-45, 1e30), (1e-30, 1e33), (3e20, 4e18), (1e30, 1e35),
                                   (1e-38, 1e-38)])
def test_matmul_global_scales_of_any_size(fmoe, M, N, K, ga, gb):
    """Global scales whose product leaves the range of normal fp32 numbers while the results are
    in it, results that leave it, and zeros. The factor is applied in fp32 to the fp32 sum: at most
    three more roundings (2^-24 each), and 2^-150 (fp32) or 2^-134 (bf16) where the result is below
    the normal range, twice."""
    ca, sa, a = _operand(M, K, "nvfp4", None, 11)
    cb, sb, b = _operand(N, K, "nvfp4", None, 12)
    ca[M // 2], a[M // 2] = 0, 0.0
    qa, qb = _held(fmoe, ca, sa, "nvfp4", ga), _held(fmoe, cb, sb, "nvfp4", gb)
    f = qa.global_scale.double().item() * qb.global_scale.double().item()
    want, size = a @ b.t() * f, a.abs() @ b.abs().t() * f
    for dtype, least in ((torch.float32, 2.0 ** -149), (torch.bfloat16, 2.0 ** -133)):
        got = fmoe.matmul_fp4(qa, qb, dtype=dtype).cpu().double()
        half, most = torch.finfo(dtype).eps / 2, torch.finfo(dtype).max
        bound = want.abs() * (half + 3 * 2.0 ** -24) + size * K * 2.0 ** -23 * (1 + half) + least
        assert (got[M // 2] == 0).all()
        below, above = want.abs() + bound < most, want.abs() - bound > most * (1 + half)
        off = (got - want).abs()
        assert (off[below] <= bound[below]).all(), (off / bound)[below].max().item()
        assert (got[above] == want[above].sign() * float("inf")).all()


@pytest.mark.gpu
def test_matmul_fp4_reports_device_errors(fmoe):
    """An error that an earlier call left (planted on the host) is raised by a product too, once;
    check=True waits for the call itself."""
    from fmoe_b200 import workloads as W

    geo = W.TINY
    inp = W.make_inputs(geo, 16, seed=3)
    gpu = {k: v.cuda() for k, v in inp.items() if isinstance(v, torch.Tensor)}
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(0)).cuda()
    q = fmoe.quantize_fp4(x, "nvfp4")
    want = fmoe.matmul_fp4(q, q)
    assert fmoe.poll_device_error() == 0
    fmoe.inject_device_error(1 << 1)
    fmoe.kernel(*W.operator_args(gpu), 0, 2.5)
    torch.cuda.synchronize()
    with pytest.raises(fmoe.DeviceError, match="device error 0x2"):
        fmoe.matmul_fp4(q, q)
    assert torch.equal(fmoe.matmul_fp4(q, q, check=True), want)
    assert fmoe.poll_device_error() == 0


# ------------------------------------------------------------------------------ refusals
def _matrix(**kw):
    from fmoe_b200.fp4 import FmoeFp4Matrix

    base = dict(codes=16, scales=16, global_scale=None, rows=4, cols=64, batch=1, format=1)
    base.update(kw)
    return FmoeFp4Matrix(**base)


@pytest.mark.parametrize("bad", [
    dict(format=2), dict(rows=-1), dict(rows=2 ** 30 + 1), dict(cols=0), dict(cols=48),
    dict(cols=65568), dict(batch=0), dict(batch=1025), dict(codes=None), dict(scales=None),
    dict(codes=8), dict(scales=4), dict(format=0, global_scale=16)])
def test_fp4_matrix_rejects(fmoe, bad):
    lib = fmoe.load_library()
    q, ok = _matrix(**bad), _matrix()
    for rc in (lib.fmoe_fp4_quantize(ctypes.byref(q), 16, 0, 64, 0, None),
               lib.fmoe_fp4_dequantize(ctypes.byref(q), 16, 0, None),
               lib.fmoe_fp4_matmul(ctypes.byref(q), ctypes.byref(ok), 16, 0, None),
               lib.fmoe_fp4_matmul(ctypes.byref(ok), ctypes.byref(q), 16, 0, None)):
        assert rc == fmoe.FMOE_ERR_VALUE
        assert len(lib.fmoe_last_error()) > 0


def test_fp4_calls_reject_arguments(fmoe):
    lib = fmoe.load_library()
    q = _matrix()
    p = ctypes.byref(q)
    assert lib.fmoe_fp4_quantize(p, 16, 3, 64, 0, None) == fmoe.FMOE_ERR_TYPE
    assert lib.fmoe_fp4_quantize(p, None, 0, 64, 0, None) == fmoe.FMOE_ERR_VALUE
    assert lib.fmoe_fp4_quantize(p, 16, 0, -1, 0, None) == fmoe.FMOE_ERR_VALUE
    assert lib.fmoe_fp4_dequantize(p, 8, 0, None) == fmoe.FMOE_ERR_VALUE
    assert lib.fmoe_fp4_dequantize(p, 16, -1, None) == fmoe.FMOE_ERR_TYPE
    assert lib.fmoe_fp4_matmul(p, p, 16, 7, None) == fmoe.FMOE_ERR_TYPE
    assert lib.fmoe_fp4_matmul(p, p, None, 0, None) == fmoe.FMOE_ERR_VALUE
    for other in (dict(cols=128), dict(format=0), dict(batch=2), dict(rows=2 ** 22 + 1)):
        assert lib.fmoe_fp4_matmul(p, ctypes.byref(_matrix(**other)), 16, 0,
                                   None) == fmoe.FMOE_ERR_VALUE
    for rows in (dict(rows=0),):
        e = ctypes.byref(_matrix(codes=None, scales=None, **rows))
        assert lib.fmoe_fp4_quantize(e, None, 0, 64, 0, None) == fmoe.FMOE_OK
        assert lib.fmoe_fp4_matmul(e, p, None, 0, None) == fmoe.FMOE_OK


def test_fp4_scale_bytes(fmoe):
    lib = fmoe.load_library()
    n = ctypes.c_size_t(0)
    for kw, want in ((dict(rows=1, cols=32, format=1), 512), (dict(rows=129, cols=96), 2 * 2 * 512),
                     (dict(rows=128, cols=160, format=0), 2 * 512),
                     (dict(rows=256, cols=7168, batch=3), 3 * 2 * 112 * 512)):
        assert lib.fmoe_fp4_scale_bytes(ctypes.byref(_matrix(**kw)), ctypes.byref(n)) == fmoe.FMOE_OK
        assert n.value == want
    assert lib.fmoe_fp4_scale_bytes(ctypes.byref(_matrix(cols=33)),
                                    ctypes.byref(n)) == fmoe.FMOE_ERR_VALUE


def test_fp4_tensor_layout(fmoe):
    """Scales given row by row land where the layout says, on any device."""
    s = torch.arange(300 * 6, dtype=torch.int64).remainder(251).to(torch.uint8).view(300, 6)
    tiles = fmoe.Fp4Tensor.tile_scales(s)
    assert tiles.shape == (3, 2, 512)
    assert torch.equal(ref.untile(tiles, 300, 6), s)
    both = fmoe.Fp4Tensor.tile_scales(torch.stack([s, s + 1]))
    assert torch.equal(ref.untile(both, 300, 6)[1], s + 1)
    codes = torch.zeros(300, 48, dtype=torch.uint8)
    q = fmoe.Fp4Tensor.from_rows(codes, s, "nvfp4")
    assert q.shape == (300, 96) and torch.equal(q.scales, tiles)
    with pytest.raises(ValueError, match="scales"):
        fmoe.Fp4Tensor.from_rows(codes, s, "mxfp4")
    with pytest.raises(TypeError, match="scales"):
        fmoe.Fp4Tensor.from_rows(codes, s.int(), "nvfp4")


def test_fp4_rejects_tensors(fmoe):
    with pytest.raises(ValueError, match="format"):
        fmoe.quantize_fp4(torch.zeros(4, 64), "fp4")
    with pytest.raises(ValueError, match="CUDA"):
        fmoe.quantize_fp4(torch.zeros(4, 64), "mxfp4")
    with pytest.raises(ValueError, match="2D or 3D"):
        fmoe.quantize_fp4(torch.zeros(64), "mxfp4")
    q = fmoe.Fp4Tensor(torch.zeros(4, 32, dtype=torch.uint8),
                       torch.zeros(1, 1, 512, dtype=torch.uint8), "nvfp4")
    with pytest.raises(ValueError, match="CUDA"):
        fmoe.dequantize_fp4(q)
    with pytest.raises(ValueError, match="CUDA"):
        fmoe.matmul_fp4(q, q)


@pytest.mark.gpu
def test_fp4_rejects_arguments(fmoe):
    x = torch.zeros(4, 64, device="cuda")
    with pytest.raises(TypeError, match="x dtype"):
        fmoe.quantize_fp4(x.double(), "mxfp4")
    with pytest.raises(ValueError, match="32 columns"):
        fmoe.quantize_fp4(x[:, :48], "mxfp4")
    with pytest.raises(ValueError, match="global scale"):
        fmoe.quantize_fp4(x, "mxfp4", global_scale=torch.ones(1, device="cuda"))
    with pytest.raises(ValueError, match="global_scale"):
        fmoe.quantize_fp4(x, "nvfp4", global_scale=torch.ones(1))
    with pytest.raises(ValueError, match="global_scale"):
        fmoe.quantize_fp4(x, "nvfp4", global_scale=torch.ones(2, device="cuda"))
    with pytest.raises(TypeError, match="global_scale"):
        fmoe.quantize_fp4(x, "nvfp4", global_scale=torch.ones(1, device="cuda").half())
    q, m = fmoe.quantize_fp4(x, "nvfp4"), fmoe.quantize_fp4(x, "mxfp4")
    with pytest.raises(ValueError, match="out"):
        fmoe.quantize_fp4(x[:2], "nvfp4", out=q)
    with pytest.raises(ValueError, match="format"):
        fmoe.matmul_fp4(q, m)
    with pytest.raises(ValueError, match="columns"):
        fmoe.matmul_fp4(q, fmoe.quantize_fp4(x[:, :32], "nvfp4"))
    with pytest.raises(TypeError, match="output dtype"):
        fmoe.matmul_fp4(q, q, dtype=torch.float64)
    with pytest.raises(ValueError, match="out"):
        fmoe.matmul_fp4(q, q, out=torch.empty(4, 5, dtype=torch.bfloat16, device="cuda"))
    short = fmoe.Fp4Tensor(q.codes, q.scales[:, :0], "nvfp4")
    with pytest.raises(ValueError, match="scales"):
        fmoe.dequantize_fp4(short)


def test_fp4_rejects_addresses_between_elements(fmoe):
    """Refused on the host: the kernels would fault on them."""
    lib = fmoe.load_library()
    ok, off = _matrix(), _matrix(global_scale=18)
    for dtype, x in ((0, 18), (1, 17), (2, 33)):
        assert lib.fmoe_fp4_quantize(ctypes.byref(ok), x, dtype, 64, 0,
                                     None) == fmoe.FMOE_ERR_VALUE
        assert b"aligned" in lib.fmoe_last_error()
    for rc in (lib.fmoe_fp4_quantize(ctypes.byref(off), 16, 0, 64, 0, None),
               lib.fmoe_fp4_dequantize(ctypes.byref(off), 16, 0, None),
               lib.fmoe_fp4_matmul(ctypes.byref(off), ctypes.byref(ok), 16, 0, None),
               lib.fmoe_fp4_matmul(ctypes.byref(ok), ctypes.byref(off), 16, 0, None)):
        assert rc == fmoe.FMOE_ERR_VALUE
        assert b"global_scale" in lib.fmoe_last_error()
