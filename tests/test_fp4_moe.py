"""forward_fp4, alone and behind route_experts, against the definition in 64 bits.

Tolerance. The quantised hidden states are exact. The first product sums H exact terms in fp32:
off by dg = H 2^-23 sum |x||w|, the SwiGLU adds 2^-20 of its value (fast exponential and division,
a few units in the last place each). A value of h nearer to a rounding border of its block than
that may be rounded either way: it is allowed one step of the grid, and where the scale itself is
at a border the block's values may move by half of the block's largest. Everything else is
rounded as in 64 bits. The second product, the weight and the sum over the picks: I 2^-23 of the
magnitudes, each row rounded to bf16 (2^-9... eps / 2 = 2^-8 of the magnitudes), the sum again.
"""
import ctypes
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from oracle import fp4_ref as ref
from oracle import router_ref

BF16 = 2.0 ** -8


def _weights(E, N, K, fmt, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(E, N, K, generator=g) * K ** -0.5
    scale = w.abs().amax((1, 2)) / 2688 if fmt == "nvfp4" else None
    codes, s = [], []
    for e in range(E):
        c, b = ref.quantize(w[e], fmt, None if scale is None else scale[e].item())
        codes.append(c)
        s.append(b)
    codes, s = torch.stack(codes), torch.stack(s)
    v = ref.values(codes, s, fmt)
    if scale is not None:
        v = v * scale.double()[:, None, None]
    return dict(codes=ref.pack(codes), scales=s, g=scale, values=v)


def _held(fmoe, m, fmt):
    return fmoe.Fp4Tensor.from_rows(m["codes"].cuda(), m["scales"].cuda(), fmt,
                                    None if m["g"] is None else m["g"].cuda())


def _quantize_with_doubt(h, dh, fmt, g):
    """The values h is quantised to, and how far they may be off if h is off by dh."""
    codes, scale = ref.quantize(h, fmt, g)
    f = 1.0 if g is None else g
    v = ref.values(codes, scale, fmt) * f
    block = ref.BLOCK[fmt]
    top = h.abs().unflatten(-1, (-1, block)).amax(-1)
    # the scale for the block's largest value at either end of its doubt
    ends = []
    for t in ((h.abs() - dh).unflatten(-1, (-1, block)).amax(-1),
              (h.abs() + dh).unflatten(-1, (-1, block)).amax(-1)):
        one = torch.zeros(*top.shape, block, dtype=torch.float64)
        one[..., 0] = t.clamp(min=0.0)
        ends.append(ref.quantize(one.flatten(-2), fmt, g)[1])
    moved = (ends[0] != ends[1]).repeat_interleave(block, -1)
    d = (ref.scale_values(scale, fmt) * f).repeat_interleave(block, -1)
    q = h.abs() / d.clamp(min=1e-300)
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    gap = (q[..., None] - mid).abs()
    near, at = gap.min(-1)
    step = torch.tensor([0.5, 0.5, 0.5, 0.5, 1.0, 1.0, 2.0], dtype=torch.float64)[at]
    doubt = torch.where(near * d <= dh + q * d * 2.0 ** -22, step * d, 0.0)
    doubt = torch.where(moved, 0.5 * top.repeat_interleave(block, -1) + doubt, doubt)
    return v, doubt


def _expected(x, idx, w, w13, w2, offset, fmt, gx, gc):
    """(out float64 [T, H], bound)."""
    T, H = x.shape
    E, I = w13["values"].shape[0], w2["values"].shape[2]
    codes, scale = ref.quantize(x, fmt, gx)
    v = ref.values(codes, scale, fmt) * (1.0 if gx is None else gx)
    out, bound = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    rows = torch.zeros_like(out)
    for e in range(E):
        t, k = torch.nonzero(idx == e + offset, as_tuple=True)
        if not len(t):
            continue
        a, b = v[t], w13["values"][e]
        g1, size = a @ b.t(), a.abs() @ b.abs().t()
        d1 = size * (H + 4) * 2.0 ** -23
        gate, up, dg, du = g1[:, :I], g1[:, I:], d1[:, :I], d1[:, I:]
        silu = up * torch.sigmoid(up)
        h = gate * silu
        dh = silu.abs() * dg + gate.abs() * 1.1 * du + dg * du + h.abs() * 2.0 ** -20
        hq, doubt = _quantize_with_doubt(h, dh, fmt, gc)
        c = w2["values"][e]
        o, osize, odoubt = hq @ c.t(), hq.abs() @ c.abs().t(), doubt @ c.abs().t()
        f = w[t, k].double()[:, None]
        out.index_add_(0, t, o * f)
        mag = (o.abs() + odoubt) * f.abs()
        rows.index_add_(0, t, mag)
        bound.index_add_(0, t, (odoubt + (osize + odoubt) * (I + 8) * 2.0 ** -23) * f.abs())
    return out, bound + rows * BF16 * 1.01 + (out.abs() + bound) * BF16 * 1.01 + 1e-30


def _case(fmoe, T, H, I, E, E_local, K, fmt, dtype, seed, offset=0, route="random"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g).to(dtype)
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(max(T, 1))])[:T]
    idx = idx.to(torch.int32).view(T, K)
    if route == "holes":
        idx[torch.rand(T, K, generator=g) < 0.4] = -1
    elif route == "one":
        idx[:] = offset + 1
    elif route == "skewed":
        idx[: T * 2 // 3, 0] = offset + 2
    elif route == "none":
        idx[:] = -1
    w = torch.rand(T, K, generator=g) - 0.2
    w13, w2 = _weights(E_local, 2 * I, H, fmt, seed + 1), _weights(E_local, H, I, fmt, seed + 2)
    gx, gc = (0.0021713, 0.0031237) if fmt == "nvfp4" else (None, None)
    args = [x.cuda(), idx.cuda(), w.cuda(), _held(fmoe, w13, fmt), _held(fmoe, w2, fmt), offset]
    kw = {} if gx is None else dict(input_scale=torch.tensor(gx, device="cuda"),
                                    intermediate_scale=torch.tensor([gc], device="cuda"))
    if gx is not None:  # the fp32 values that the device sees
        gx, gc = kw["input_scale"].item(), kw["intermediate_scale"].item()
    return args, kw, (x.float(), idx, w, w13, w2, offset, fmt, gx, gc)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("T,H,I,E,E_local,K,offset,route,dtype", [
    (1, 256, 128, 16, 16, 4, 0, "random", torch.bfloat16),
    (7, 256, 128, 16, 16, 4, 0, "random", torch.float32),
    (64, 512, 256, 32, 8, 8, 8, "random", torch.bfloat16),
    (300, 256, 128, 16, 4, 4, 12, "holes", torch.float16),
    (33, 96, 96, 8, 8, 2, 0, "random", torch.bfloat16),
    (150, 544, 160, 8, 8, 3, 0, "random", torch.float16),
    (40, 128, 32, 4, 4, 1, 0, "random", torch.bfloat16),
    (140, 256, 128, 8, 2, 2, 3, "one", torch.bfloat16),
    (9, 256, 128, 8, 8, 2, 0, "none", torch.bfloat16),
    (2000, 128, 128, 256, 256, 8, 0, "random", torch.bfloat16),
    (50, 1056, 384, 5, 3, 5, 1, "random", torch.float32),
    # few rows an expert and long sums: tiles shared by two CTAs, next to an expert of more rows
    (16, 1056, 1152, 16, 16, 4, 0, "random", torch.bfloat16),
    (1, 2048, 1024, 8, 8, 2, 0, "random", torch.bfloat16),
    (60, 1280, 1152, 16, 8, 2, 3, "skewed", torch.bfloat16),
    (33, 1024, 1056, 64, 64, 8, 0, "holes", torch.float16),
    # fewer tiles than SMs and long sums, of few rows and of many
    (3, 4096, 2304, 4, 4, 2, 0, "random", torch.bfloat16),
    (200, 2560, 2176, 2, 2, 1, 0, "random", torch.bfloat16),
    (140, 2080, 2080, 3, 3, 2, 0, "holes", torch.float32),
    (500, 2048, 2048, 8, 8, 2, 0, "skewed", torch.bfloat16),
])
def test_forward_fp4(fmoe, fmt, T, H, I, E, E_local, K, offset, route, dtype):
    args, kw, state = _case(fmoe, T, H, I, E, E_local, K, fmt, dtype, T + H, offset, route)
    out = fmoe.forward_fp4(*args, **kw)
    assert out.dtype == torch.bfloat16 and out.shape == (T, H)
    want, bound = _expected(*state)
    off = (out.cpu().double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()
    # The bound takes every value in doubt at its worst, and all of one sign. As a whole the
    # result is nearer: bf16 twice (2^-8 each at most), and of the values of h at most about one
    # in a thousand (2 dg over the mean distance of two borders) takes the other of two
    # neighbours, at most a third of itself away: 0.8 % + 0.33 sqrt(1e-3) = 1.9 %.
    assert off.pow(2).sum().sqrt() <= 0.02 * want.pow(2).sum().sqrt()
    assert torch.equal(out, fmoe.forward_fp4(*args, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_route_and_forward_together(fmoe, fmt):
    """Router and experts as a layer runs them: eagerly, captured and replayed on new inputs, on a
    side stream beside another call, with the slices of two devices' experts summing to the whole."""
    T, H, I, E, K = 50, 256, 128, 16, 4
    args, kw, state = _case(fmoe, T, H, I, E, E, K, fmt, torch.bfloat16, 5)
    x, w13, w2 = args[0], args[3], args[4]
    logits = torch.randn(T, E, generator=torch.Generator().manual_seed(9)).cuda()
    bias = (torch.rand(E, generator=torch.Generator().manual_seed(10)) * 0.2).cuda()

    def layer():
        idx, w = fmoe.route_experts(logits, K, score="sigmoid", bias=bias, n_group=4, topk_group=2,
                                    scale=2.5)
        return idx, w, fmoe.forward_fp4(x, idx, w, w13, w2, **kw)

    idx, w, out = layer()
    want_idx, _ = router_ref.route(logits.cpu(), bias.cpu(), K, "sigmoid", 4, 2, "top2", True, 2.5)
    assert torch.equal(idx.cpu(), want_idx)
    want, bound = _expected(state[0], idx.cpu(), w.cpu(), *state[3:])
    assert ((out.cpu().double() - want).abs() <= bound).all()

    # two slices of the experts
    parts = [fmoe.forward_fp4(
        x, idx, w, fmoe.Fp4Tensor(w13.codes[s], w13.scales[s], fmt,
                                  None if w13.global_scale is None else w13.global_scale[s]),
        fmoe.Fp4Tensor(w2.codes[s], w2.scales[s], fmt,
                       None if w2.global_scale is None else w2.global_scale[s]),
        s.start, **kw) for s in (slice(0, 10), slice(10, 16))]
    for part, lo, hi in zip(parts, (0, 10), (10, 16)):
        mine = torch.where((idx >= lo) & (idx < hi), idx, -1).cpu()
        want, bound = _expected(state[0], mine, w.cpu(), *state[3:])
        assert ((part.cpu().double() - want).abs() <= bound).all()

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        held2 = layer()
    side = torch.cuda.Stream()
    for seed in (11, 12):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(T, H, generator=g))
        logits.copy_(torch.randn(T, E, generator=g))
        # both graphs at once on two streams, and an eager call between them
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            second.replay()
        got = layer()
        torch.cuda.current_stream().wait_stream(side)
        for a, b, c in zip(held, held2, got):
            assert torch.equal(a, c) and torch.equal(b, c)


@pytest.mark.gpu
def test_forward_fp4_agrees_with_its_parts(fmoe):
    """One expert and weight 1: the layer is quantise, multiply, SwiGLU, quantise, multiply."""
    T, H, I = 200, 512, 256
    for fmt in ("mxfp4", "nvfp4"):
        w13 = fmoe.quantize_fp4(torch.randn(1, 2 * I, H, device="cuda") / H ** 0.5, fmt)
        w2 = fmoe.quantize_fp4(torch.randn(1, H, I, device="cuda") / I ** 0.5, fmt)
        x = torch.randn(T, H, device="cuda").bfloat16()
        idx = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
        got = fmoe.forward_fp4(x, idx, torch.ones(T, 1, device="cuda"), w13, w2)
        one = lambda q: fmoe.Fp4Tensor(q.codes[0], q.scales[0], fmt)  # noqa: E731
        h = fmoe.matmul_fp4(fmoe.quantize_fp4(x, fmt), one(w13), dtype=torch.float32)
        h = h[:, :I] * torch.nn.functional.silu(h[:, I:])
        want = fmoe.matmul_fp4(fmoe.quantize_fp4(h, fmt), one(w2))
        # equal but where a value of h sat on a rounding border (2^-20 of it: 8 borders an octave,
        # 256 values a row)
        same = (got == want).all(1).float().mean().item()
        assert same > 0.9
        assert (got.float() - want.float()).norm() < 0.02 * want.float().norm()


@pytest.mark.gpu
def test_forward_fp4_workspace_and_out(fmoe):
    from fmoe_b200.fp4 import FmoeFp4Problem, fp4_workspace_bytes

    args, kw, _ = _case(fmoe, 30, 256, 128, 16, 16, 4, "nvfp4", torch.bfloat16, 1)
    want = fmoe.forward_fp4(*args, **kw)
    n = fp4_workspace_bytes(FmoeFp4Problem(30, 256, 128, 16, 4, 0, 1, 1))
    ws = torch.full((n + 256,), 255, dtype=torch.uint8, device="cuda")  # NaN wherever it is read
    out = torch.full((31, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    got = fmoe.forward_fp4(*args, **kw, workspace=ws[:n], out=out[:30], check=True)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
    assert (out[30] == 7.0).all() and (ws[n:] == 255).all()
    with pytest.raises(ValueError, match="workspace"):
        fmoe.forward_fp4(*args, **kw, workspace=ws[:n - 256])
    with pytest.raises(ValueError, match="workspace"):
        fmoe.forward_fp4(*args, **kw, workspace=torch.empty(n, dtype=torch.uint8))
    empty = fmoe.forward_fp4(args[0][:0], args[1][:0], args[2][:0], *args[3:], **kw)
    assert empty.shape == (0, 256)


@pytest.mark.gpu
def test_forward_fp4_rejects_arguments(fmoe):
    args, kw, _ = _case(fmoe, 6, 256, 128, 16, 16, 4, "nvfp4", torch.bfloat16, 1)
    x, idx, w, w13, w2, _ = args
    other = fmoe.quantize_fp4(torch.zeros(16, 256, 128, device="cuda"), "mxfp4")
    for bad, err, match in (
            ((x.double(), idx, w, w13, w2), TypeError, "hidden_states"),
            ((x[:, :128], idx, w, w13, w2), ValueError, "hidden_states"),
            ((x[:5], idx, w, w13, w2), ValueError, "hidden_states"),
            ((x.cpu(), idx, w, w13, w2), ValueError, "hidden_states"),
            ((x, idx.long(), w, w13, w2), TypeError, "topk_idx"),
            ((x, idx, w.half(), w13, w2), TypeError, "topk_w"),
            ((x, idx, w[:, :3], w13, w2), ValueError, "topk_w"),
            ((x, idx, w, w13, other), ValueError, "format"),
            ((x, idx, w, w2, w13), ValueError, "w13 must be"),
            ((x, idx, w, w13, x), ValueError, "Fp4Tensor")):
        with pytest.raises(err, match=match):
            fmoe.forward_fp4(*bad)
    with pytest.raises(ValueError, match="input_scale"):
        fmoe.forward_fp4(*args, input_scale=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="intermediate_scale"):
        fmoe.forward_fp4(*args, intermediate_scale=torch.ones(1))
    with pytest.raises(ValueError, match="out"):
        fmoe.forward_fp4(*args, out=torch.empty(5, 256, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("T,H,I,E,E_local,K,offset,route,dtype", [
    (300, 7168, 128, 16, 16, 8, 0, "random", torch.bfloat16),
    (1100, 2048, 128, 8, 8, 8, 0, "random", torch.bfloat16),
    (1100, 2048, 160, 32, 8, 8, 8, "holes", torch.float16),
    # a batch that just fits in 2^24 values of all picks' rows, and one that just does not
    (512, 4096, 128, 16, 4, 8, 4, "random", torch.float32),
    (513, 4096, 128, 16, 4, 8, 4, "random", torch.bfloat16),
])
def test_forward_fp4_large_batches(fmoe, fmt, T, H, I, E, E_local, K, offset, route, dtype):
    """A token's result is that of the definition in large batches too, and bit for bit the one it
    has in a small batch: every sum has an order of its own, whatever lies beside it."""
    args, kw, state = _case(fmoe, T, H, I, E, E_local, K, fmt, dtype, T + H, offset, route)
    out = fmoe.forward_fp4(*args, **kw)
    assert torch.equal(out, fmoe.forward_fp4(*args, **kw))
    x, idx, w = args[:3]
    for part in (slice(0, 40), slice(T // 2, T // 2 + 1), slice(T - 24, T)):
        some = fmoe.forward_fp4(x[part].clone(), idx[part].clone(), w[part].clone(), *args[3:],
                                **kw)
        assert torch.equal(some, out[part])
        want, bound = _expected(*(v[part] for v in state[:3]), *state[3:])
        assert ((some.cpu().double() - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("T,H,K", [(20, 1024, 2), (300, 7168, 8), (2100, 4096, 2)])
def test_forward_fp4_rounds_once(fmoe, fmt, T, H, K):
    """Picks that nearly cancel. With the same expert picked with weights 1 and 2^-7 - 1, a row r
    of fp32 gives r - r (1 - 2^-7): its roundings (the factor, two rows, the sum: 2^-24 |r| each)
    are below 2^-14 of the result r 2^-7. One rounding to bf16 follows, as for the pick of weight
    2^-7 alone: each is within half a step (2^-8) of its number, 2^-7 (1 + 2^-8) together."""
    args, kw, _ = _case(fmoe, T, H, 128, 4, 4, 1, fmt, torch.bfloat16, 3)
    x, one, _, w13, w2, _ = args
    idx = torch.full((T, K), -1, dtype=torch.int32, device="cuda")
    w = torch.zeros(T, K, device="cuda")
    idx[:, 0] = idx[:, K - 1] = one[:, 0]
    w[:, 0], w[:, K - 1] = 1.0, 2.0 ** -7 - 1.0
    got = fmoe.forward_fp4(x, idx, w, w13, w2, **kw).double()
    want = fmoe.forward_fp4(x, one, torch.full((T, 1), 2.0 ** -7, device="cuda"), w13, w2,
                            **kw).double()
    assert want.abs().max() > 0
    assert ((got - want).abs() <= want.abs() * (2.0 ** -7 + 2.0 ** -13)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("I", [128, 160])
def test_forward_fp4_small_scales(fmoe, I):
    """Global scales of the second product that multiply to less than fp32 holds, under routing
    weights that bring the result back; and of the first that multiply to more, over zeros."""
    T, H, E, K = 40, 256, 4, 2
    g = torch.Generator().manual_seed(I)
    x = torch.randn(T, H, generator=g) * 2.0 ** -33
    x[5] = 0.0
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).to(torch.int32)
    w = (torch.rand(T, K, generator=g) + 0.1) * 2.0 ** 50
    w13, w2 = _weights(E, 2 * I, H, "nvfp4", 1), _weights(E, H, I, "nvfp4", 2)
    w2["g"], w2["values"] = w2["g"] * 2.0 ** -70, w2["values"] * 2.0 ** -70
    gx = (x.abs().amax() / 2688).item()
    v = ref.values(*ref.quantize(x, "nvfp4", gx), "nvfp4") * gx
    h = torch.cat([v @ e[:I].t() * torch.nn.functional.silu(v @ e[I:].t()) for e in w13["values"]])
    gc = torch.tensor(h.abs().amax().item() / 2688).item()
    assert gc * w2["g"].max().item() < 2.0 ** -149  # nothing is left of the factor in fp32
    call = lambda x, gx, gc, w13, w: fmoe.forward_fp4(  # noqa: E731
        x.cuda(), idx.cuda(), w.cuda(), _held(fmoe, w13, "nvfp4"), _held(fmoe, w2, "nvfp4"),
        input_scale=torch.tensor(gx, device="cuda"),
        intermediate_scale=torch.tensor(gc, device="cuda"))
    out = call(x, gx, gc, w13, w)
    want, bound = _expected(x, idx, w, w13, w2, 0, "nvfp4", gx, gc)
    off = (out.cpu().double() - want).abs()
    assert (out[5] == 0).all() and 2.0 ** -90 < want.abs().max() < 2.0 ** -40
    assert (off <= bound).all(), (off / bound).max().item()
    assert off.pow(2).sum().sqrt() <= 0.02 * want.pow(2).sum().sqrt()  # as in test_forward_fp4
    # 2^100 times 2^100 is an infinity; a row of zeros stays one
    big = dict(w13, g=w13["g"] * 0 + 2.0 ** 100)
    out = call(torch.zeros(T, H), 2.0 ** 100, 1.0, big, w)
    assert (out == 0).all()


@pytest.mark.gpu
def test_forward_fp4_takes_slices_of_a_routing(fmoe):
    """Picks and weights of some of a batch's tokens, at addresses of no more than 4 bytes'
    alignment, also where a captured graph replays on new ones."""
    args, kw, _ = _case(fmoe, 30, 256, 128, 16, 16, 3, "nvfp4", torch.bfloat16, 1)
    x, idx, w = args[:3]
    whole = fmoe.forward_fp4(*args, **kw)
    for first, last in ((1, 30), (2, 11), (29, 30)):
        part = slice(first, last)
        assert idx[part].data_ptr() % 16
        assert torch.equal(fmoe.forward_fp4(x[part], idx[part], w[part], *args[3:], **kw),
                           whole[part])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = fmoe.forward_fp4(x[1:], idx[1:], w[1:], *args[3:], **kw)
    for _ in range(2):
        idx.copy_(idx.roll(3, 0))
        w.copy_(w.flip(0))
        graph.replay()
        assert torch.equal(held, fmoe.forward_fp4(*args, **kw)[1:])


@pytest.mark.gpu
def test_fp4_first_call_of_a_process_can_be_captured(fmoe):
    """Nothing that a call makes for later calls (the device's error word) may break a capture.
    In a process of its own, where no call came before."""
    program = """
import torch
import fmoe_b200 as f
x = torch.randn(40, 256, device="cuda")
w13, w2 = torch.randn(4, 256, 256, device="cuda") / 16, torch.randn(4, 256, 128, device="cuda") / 11
idx = torch.arange(80, device="cuda", dtype=torch.int32).view(40, 2) % 4
w = torch.full((40, 2), 0.5, device="cuda")
f.load_library()
torch.cuda.synchronize()
def call():
    q = f.quantize_fp4(x, "nvfp4")
    return f.matmul_fp4(q, q), f.forward_fp4(x, idx, w, f.quantize_fp4(w13, "nvfp4"),
                                             f.quantize_fp4(w2, "nvfp4"))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    held = call()
graph.replay()
for a, b in zip(held, call()):
    assert torch.equal(a, b)
print("captured")
"""
    root = Path(fmoe.__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=str(root)))
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("field,value", [
    ("num_tokens", -1), ("num_tokens", 2 ** 20 + 1), ("hidden_size", 48), ("hidden_size", 0),
    ("hidden_size", 16416), ("intermediate_size", 100), ("num_local_experts", 0),
    ("num_local_experts", 257), ("local_expert_offset", -1), ("top_k", 0), ("top_k", 33), ("format", 2), ("dtype", 3)])
def test_fp4_forward_rejects(fmoe, field, value):
    from fmoe_b200.fp4 import FmoeFp4Problem, FmoeFp4Tensors

    lib = fmoe.load_library()
    p = FmoeFp4Problem(4, 256, 128, 8, 2, 0, 1, 1)
    n = ctypes.c_size_t(0)
    assert lib.fmoe_fp4_workspace_size(ctypes.byref(p), ctypes.byref(n)) == fmoe.FMOE_OK
    assert n.value > 4 * 2 * 256
    setattr(p, field, value)
    t = FmoeFp4Tensors(*[256] * 12)
    want = fmoe.FMOE_ERR_TYPE if field == "dtype" else fmoe.FMOE_ERR_VALUE
    assert lib.fmoe_fp4_workspace_size(ctypes.byref(p), ctypes.byref(n)) == want
    assert lib.fmoe_fp4_forward(ctypes.byref(p), ctypes.byref(t), 256, 1 << 40, None) == want


def test_fp4_forward_rejects_pointers(fmoe):
    from fmoe_b200.fp4 import FmoeFp4Problem, FmoeFp4Tensors

    lib = fmoe.load_library()
    p = FmoeFp4Problem(4, 256, 128, 8, 2, 0, 1, 1)
    call = lambda t, ws=256, n=1 << 40: lib.fmoe_fp4_forward(  # noqa: E731
        ctypes.byref(p), ctypes.byref(t), ws, n, None)
    fields = [f for f, _ in FmoeFp4Tensors._fields_ if "global" not in f and "_scale" != f[-6:]]
    for f in fields:
        for bad in (None, 8):
            t = FmoeFp4Tensors(*[256] * 12)
            setattr(t, f, bad)
            assert call(t) == fmoe.FMOE_ERR_VALUE, f
    t = FmoeFp4Tensors(*[256] * 12)
    assert call(t, ws=None) == fmoe.FMOE_ERR_WORKSPACE
    assert call(t, ws=128) == fmoe.FMOE_ERR_WORKSPACE
    assert call(t, n=100) == fmoe.FMOE_ERR_WORKSPACE
    p.format = 0  # mxfp4 takes no global scale
    assert call(t) == fmoe.FMOE_ERR_VALUE
    p.num_tokens = 0
    assert call(FmoeFp4Tensors()) == fmoe.FMOE_OK


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [-1, -2 ** 31, -2 ** 32, -2 ** 40 - 1, 2 ** 31,
                                    2 ** 32])
def test_forward_fp4_rejects_offsets(fmoe, offset):
    """Offsets that no expert id reaches, also where their low 32 bits are a valid one."""
    args, kw, _ = _case(fmoe, 6, 256, 128, 16, 16, 4, "nvfp4", torch.bfloat16, 1)
    with pytest.raises(ValueError, match="local_expert_offset"):
        fmoe.forward_fp4(*args[:5], offset, **kw)


@pytest.mark.gpu
def test_forward_fp4_takes_large_offsets(fmoe):
    """Ids up to the largest int32, told apart from those beside the slice."""
    args, kw, _ = _case(fmoe, 9, 256, 128, 16, 16, 4, "nvfp4", torch.bfloat16, 1)
    x, idx, w, w13, w2, _ = args
    want = fmoe.forward_fp4(*args, **kw)
    for offset in (2 ** 30 + 5, 2 ** 31 - 16):
        far = idx + offset
        assert torch.equal(fmoe.forward_fp4(x, far, w, w13, w2, offset, **kw), want)
        assert (fmoe.forward_fp4(x, idx, w, w13, w2, offset, **kw) == 0).all()
        assert (fmoe.forward_fp4(x, far, w, w13, w2, 2 ** 30 - 16, **kw) == 0).all()


@pytest.mark.gpu
def test_forward_fp4_refuses_to_drop_a_gradient(fmoe):
    """The layer has no backward pass: what would ask it for one is refused, not cut off."""
    args, kw, _ = _case(fmoe, 6, 256, 128, 16, 16, 4, "nvfp4", torch.bfloat16, 1)
    x, idx, w, w13, w2, _ = args
    want = fmoe.forward_fp4(*args, **kw)
    logits = torch.randn(6, 16, device="cuda", requires_grad=True)
    idx2, w2_ = fmoe.route_experts(logits, 4)
    for xx, ii, ww in ((x.clone().requires_grad_(True), idx, w), (x, idx2, w2_)):
        with pytest.raises(ValueError, match="no gradient"):
            fmoe.forward_fp4(xx, ii, ww, w13, w2, **kw)
    # without a graph to lose, the same tensors are taken
    with torch.no_grad():
        assert torch.equal(fmoe.forward_fp4(x.clone().requires_grad_(True), idx, w, w13, w2, **kw),
                           want)
    assert fmoe.forward_fp4(x, idx2, w2_.detach(), w13, w2, **kw).shape == x.shape
    with torch.autograd.forward_ad.dual_level():
        for name, (xx, ww) in {"hidden_states": (torch.autograd.forward_ad.make_dual(x, x), w),
                               "topk_w": (x, torch.autograd.forward_ad.make_dual(w, w))}.items():
            with pytest.raises(ValueError, match=name + ".*tangent"):
                fmoe.forward_fp4(xx, idx, ww, w13, w2, **kw)


def test_fp4_forward_rejects_scales_between_elements(fmoe):
    from fmoe_b200.fp4 import FmoeFp4Problem, FmoeFp4Tensors

    lib = fmoe.load_library()
    p = FmoeFp4Problem(4, 256, 128, 8, 2, 0, 1, 1)
    for f in ("w13_global", "w2_global", "input_scale", "intermediate_scale"):
        t = FmoeFp4Tensors(*[256] * 12)
        setattr(t, f, 258)
        assert lib.fmoe_fp4_forward(ctypes.byref(p), ctypes.byref(t), 256, 1 << 40,
                                    None) == fmoe.FMOE_ERR_VALUE
        assert b"global scales" in lib.fmoe_last_error()
