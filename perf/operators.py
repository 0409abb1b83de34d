"""The router, the 4-bit quantisation, the 4-bit product and the 4-bit expert layer as measured
cases: what each is called with, its plain form in elementary torch operations, and its work.

Kinds of cases
  route    expert routing (softmax or sigmoid scores, balance bias, groups, top-k), forward;
           with ``grad`` also the gradient of the logits, as a training step needs it
  quant    quantisation of a matrix to 4-bit blocks and back
  matmul   a 4-bit matrix times the transpose of another
  moe      a layer's step: routing, then the experts' two 4-bit products with the SwiGLU between
"""
import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BLOCK = {"mxfp4": 32, "nvfp4": 16}  # values that share one scale


def _fmoe():
    if "fmoe_b200" not in sys.modules:  # once: a program imports the package before its first step
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "fused-moe-yws_b200"))
    import fmoe_b200

    return fmoe_b200


# ------------------------------------------------------------------------------- the cases
def listed():
    group8 = dict(score="sigmoid", bias=True, n_group=8, topk_group=4, group_score="top2",
                  renormalize=True, scale=2.5, top_k=8, E=256)
    return [
        # one token of the 256-expert layer: what a decode step pays for its routing
        dict(name="route decode 1x256", kind="route", T=1, dtype="fp32", grad=False, masked=False,
             **group8),
        # a prefill chunk of the same layer
        dict(name="route prefill 16384x256", kind="route", T=16384, dtype="fp32", grad=False,
             masked=False, **group8),
        # training step of a small softmax router with plain (not renormalised) weights; an odd
        # batch with padded tokens, whose logits are all masked
        dict(name="route train softmax 8191x60", kind="route", T=8191, E=60, top_k=4,
             score="softmax", bias=False, n_group=1, topk_group=1, group_score="top2",
             renormalize=False, scale=1.0, dtype="bf16", grad=True, masked=True),
        # training step of the 256-expert router, gradients through the renormalised weights
        dict(name="route train sigmoid 16384x256", kind="route", T=16384, dtype="bf16", grad=True,
             masked=False, **group8),
        # the hidden states of a prefill chunk
        dict(name="quant nvfp4 4096x7168", kind="quant", M=4096, K=7168, format="nvfp4",
             dtype="bf16"),
        # an odd number of rows in the other format
        dict(name="quant mxfp4 1003x2048", kind="quant", M=1003, K=2048, format="mxfp4",
             dtype="fp16"),
        # one weight matrix of an expert against a decode batch: bound by reading the weights
        dict(name="matmul nvfp4 16x4096x7168", kind="matmul", M=16, N=4096, K=7168,
             format="nvfp4"),
        # ragged in every size
        dict(name="matmul mxfp4 333x1000x2080", kind="matmul", M=333, N=1000, K=2080,
             format="mxfp4"),
        # a large product: bound by the tensor cores
        dict(name="matmul nvfp4 8192x4096x7168", kind="matmul", M=8192, N=4096, K=7168,
             format="nvfp4"),
        # the small 16-expert layer, an odd number of tokens
        dict(name="moe mxfp4 tiny T=7", kind="moe", T=7, H=256, I=128, E=16, E_local=16, top_k=4,
             score="softmax", bias=False, n_group=1, topk_group=1, group_score="top2",
             renormalize=True, scale=1.0, dtype="bf16", format="mxfp4"),
        # a 32-expert slice of the 256-expert layer: decode and prefill
        dict(name="moe nvfp4 slice T=16", kind="moe", T=16, H=7168, I=2048, E_local=32,
             dtype="bf16", format="nvfp4", **group8),
        dict(name="moe nvfp4 slice T=4096", kind="moe", T=4096, H=7168, I=2048, E_local=32,
             dtype="bf16", format="nvfp4", **group8),
    ]


def _spread(rng, low, high, step=1):
    """A multiple of `step` in [low, high], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step or step))


def _draw_router(rng):
    E = rng.choice([8, 16, 32, 60, 64, 72, 96, 128, 160, 256, 384, 512])
    n_group = rng.choice([1, 1] + [g for g in (2, 4, 8) if E % g == 0 and E // g >= 4])
    topk_group = rng.randint(1, n_group)
    score = rng.choice(["softmax", "sigmoid"])
    top_k = rng.randint(1, min(16, topk_group * (E // n_group)))
    # a single renormalised weight is constant: nobody trains through it
    return dict(E=E, n_group=n_group, topk_group=topk_group, score=score, top_k=top_k,
                bias=rng.random() < 0.5, group_score=rng.choice(["top2", "max"]),
                renormalize=top_k > 1 and rng.random() < 0.6, scale=rng.choice([1.0, 2.5]))


def draw(rng):
    kind = rng.choice(["route", "route", "quant", "matmul", "moe"])
    fmt = rng.choice(["mxfp4", "nvfp4"])
    if kind == "route":
        c = _draw_router(rng)
        return dict(kind=kind, T=_spread(rng, 1, min(32768, 16384 * 256 // c["E"])),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), grad=rng.random() < 0.5,
                    masked=rng.random() < 0.3, **c)
    if kind == "quant":
        K = _spread(rng, 64, 8192, 32)
        return dict(kind=kind, M=_spread(rng, 1, min(8192, 4096 * 7168 // K)), K=K, format=fmt,
                    dtype=rng.choice(["fp32", "bf16", "fp16"]))
    if kind == "matmul":
        N, K = _spread(rng, 24, 8192), _spread(rng, 64, 8192, 32)
        return dict(kind=kind, M=_spread(rng, 1, 8192), N=N, K=K, format=fmt)
    c = _draw_router(rng)
    E_local = c["E"] if c["E"] <= 32 else rng.choice([8, 16, 32])
    return dict(kind=kind, T=_spread(rng, 1, 2048), H=_spread(rng, 256, 4096, 32),
                I=_spread(rng, 128, 2048, 32), E_local=min(E_local, c["E"]),
                dtype=rng.choice(["bf16", "fp16"]), format=fmt, **c)


# ------------------------------------------------------------------------------- the inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _tiles(scales):
    """Scale bytes [..., M, B] as the products read them: [..., ceil(M/128), ceil(B/4), 512],
    the byte of row r and block b at (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4 of its tile."""
    *lead, M, B = scales.shape
    m, b = -(-M // 128), -(-B // 4)
    full = torch.zeros(*lead, m * 128, b * 4, dtype=torch.uint8, device=scales.device)
    full[..., :M, :B] = scales
    full = full.view(*lead, m, 4, 32, b, 4)
    n = len(lead)
    order = list(range(n)) + [n, n + 3, n + 2, n + 1, n + 4]
    return full.permute(order).reshape(*lead, m, b, 512).contiguous()


def _matrix(gen, M, K, fmt, spread=1.0):
    """A 4-bit matrix as a program has it in hand: codes, scale bytes, the global scale."""
    x = _randn(gen, M, K) * spread
    g = x.abs().amax() / (6.0 * 448.0) if fmt == "nvfp4" else None
    codes, scales = _encode(x, fmt, g)
    return dict(codes=codes, scales=scales, tiles=_tiles(scales), g=g)


def _experts(gen, E, N, K, fmt):
    """E weight matrices [N, K] of one layer, each with its own global scale."""
    parts = [_matrix(gen, N, K, fmt, K ** -0.5) for _ in range(E)]
    stack = lambda key: torch.stack([p[key] for p in parts])  # noqa: E731
    return dict(codes=stack("codes"), scales=stack("scales"), tiles=stack("tiles"),
                g=stack("g") if fmt == "nvfp4" else None)


def prepare(case, seed):
    gen = _gen(seed)
    state = dict(case=case)
    kind = case["kind"]
    if kind in ("route", "moe"):
        T, E = case["T"], case["E"]
        x = _randn(gen, T, E) * 1.5
        if case.get("masked"):
            # experts that a token may not use, and padded tokens that may use none
            off = torch.rand(T, E, generator=gen, device="cuda") < 0.05
            off |= torch.rand(T, 1, generator=gen, device="cuda") < 0.05
            x = x.masked_fill(off, -math.inf)
        dtype = torch.float32 if kind == "moe" else _DTYPES[case["dtype"]]
        state["logits"] = x.to(dtype)
        state["bias"] = (torch.rand(E, generator=gen, device="cuda") * 0.2 - 0.1
                         if case["bias"] else None)
        if case.get("grad"):
            state["grad"] = _randn(gen, T, case["top_k"])
    if kind == "quant":
        # activations: a few channels are much larger than the others; the last row is empty
        x = _randn(gen, case["M"], case["K"])
        x = x * torch.where(torch.rand(case["K"], generator=gen, device="cuda") < 0.01, 20.0, 1.0)
        if case["M"] > 1:
            x[-1] = 0.0
        state["x"] = x.to(_DTYPES[case["dtype"]])
        state["g"] = x.abs().amax() / (6.0 * 448.0) if case["format"] == "nvfp4" else None
    if kind == "matmul":
        state["a"] = _matrix(gen, case["M"], case["K"], case["format"])
        state["b"] = _matrix(gen, case["N"], case["K"], case["format"], case["K"] ** -0.5)
    if kind == "moe":
        fmt = case["format"]
        state["x"] = _randn(gen, case["T"], case["H"]).to(_DTYPES[case["dtype"]])
        state["w13"] = _experts(gen, case["E_local"], 2 * case["I"], case["H"], fmt)
        state["w2"] = _experts(gen, case["E_local"], case["H"], case["I"], fmt)
        state["first"] = (case["E"] - case["E_local"]) // 2
        # the activations' global scales, from a calibration: largest magnitudes of about 5.8
        # and 14 over 6 * 448
        state["g_x"] = torch.full((), 2.1713e-3, device="cuda") if fmt == "nvfp4" else None
        state["g_c"] = torch.full((), 5.2371e-3, device="cuda") if fmt == "nvfp4" else None
    return state


# ------------------------------------------------------------------------------- plain forms
def _encode(x, fmt, g):
    """Codes (two a byte, the first value in the low half) and scale bytes of fp32 values.

    mxfp4: 32 values share 2^e, e = floor(log2 of the largest magnitude) - 2.
    nvfp4: 16 values share an e4m3 scale of (largest magnitude / (6 g)); g is fp32.
    A value is rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even code. A block
    with an infinity or a NaN has the scale NaN."""
    *lead, K = x.shape
    block = _BLOCK[fmt]
    v = x.reshape(*lead, K // block, block)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(top)
    if fmt == "mxfp4":
        e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
        e = torch.where(top == 0, -127, e)
        scales = torch.where(bad, 255, e + 127).to(torch.uint8)
        q = torch.ldexp(v, -e[..., None])
    else:
        g = torch.ones((), device=x.device) if g is None else g
        s = (top / (6.0 * g)).clamp(max=448.0).to(torch.float8_e4m3fn)
        scales = torch.where(bad, 127, s.view(torch.uint8))
        d = s.float() * g
        q = torch.where(d[..., None] > 0, v / d[..., None], torch.zeros_like(v))
    a = q.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5.0))
    code = code + torch.signbit(v).to(torch.uint8) * 8
    code = code.reshape(*lead, K // 2, 2)
    return code[..., 0] + code[..., 1] * 16, scales


def _scale_values(scales, fmt):
    if fmt == "mxfp4":
        e = scales.to(torch.int32) - 127
        return torch.where(scales == 255, math.nan, torch.ldexp(torch.ones((), device=e.device), e))
    return scales.view(torch.float8_e4m3fn).float()


def _decode(codes, scales, fmt, g=None):
    """The fp32 values that codes and scale bytes stand for."""
    value = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    value = torch.cat([value, -value])
    byte = torch.arange(256, device=codes.device)
    pairs = torch.stack([value[byte % 16], value[byte // 16]], -1)
    v = pairs[codes.to(torch.int32)]
    s = _scale_values(scales, fmt)
    if g is not None:
        s = s * g
    v = v.reshape(*scales.shape, _BLOCK[fmt]) * s[..., None]
    return v.reshape(*codes.shape[:-1], -1)


def _route(logits, bias, c):
    """(indices, scores in 64 bits, chosen scores, weights in 64 bits). Decided in 64 bits: the
    order of two experts may hang on the last bit. Without a bias the order of the scores is that
    of the logits. A logit of -inf or NaN takes an expert out."""
    x = logits.double()
    out = torch.isnan(x) | (x == -math.inf)
    if c["score"] == "softmax":
        y = x.masked_fill(out, -math.inf)
        top = y.amax(-1, keepdim=True)
        e = torch.where(y == top, 1.0, torch.exp(y - top)).masked_fill(out, 0.0)
        s = e / e.sum(-1, keepdim=True).clamp(min=1.0)
    else:
        s = (1.0 / (1.0 + torch.exp(-x))).masked_fill(out, 0.0)
    choice = x if bias is None else s + bias.double()
    choice = choice.masked_fill(out, -math.inf)
    T, E = x.shape
    n = c["n_group"]
    if n > 1:
        if c["group_score"] == "max":
            of_group = choice.view(T, n, E // n).amax(-1)
        else:
            worth = (s if bias is None else s + bias.double()).masked_fill(out, -math.inf)
            best = torch.sort(worth.view(T, n, E // n), dim=-1, descending=True).values
            of_group = best[..., 0] + best[..., 1]
        order = torch.sort(of_group, dim=-1, descending=True, stable=True).indices
        kept = torch.zeros(T, n, dtype=torch.bool, device=x.device)
        kept.scatter_(1, order[:, :c["topk_group"]], True)
        choice = choice.masked_fill(~kept.repeat_interleave(E // n, dim=1), -math.inf)
    best = torch.sort(choice, dim=-1, descending=True, stable=True)
    idx = best.indices[:, :c["top_k"]]
    live = best.values[:, :c["top_k"]] > -math.inf
    picked = torch.where(live, s.gather(1, idx), 0.0)
    w = picked * c["scale"]
    if c["renormalize"]:
        if c["score"] == "softmax":
            # the softmax over the chosen experts alone
            z = torch.where(live, x.gather(1, idx), -math.inf)
            top = z.amax(-1, keepdim=True)
            e = torch.where(z == top, 1.0, torch.exp(z - top)).masked_fill(~live, 0.0)
            w = e / e.sum(-1, keepdim=True).clamp(min=1.0) * c["scale"]
        else:
            w = picked / (picked.sum(-1, keepdim=True) + 1e-20) * c["scale"]
    return torch.where(live, idx, -1), s, picked, w


def _route_grad(logits, c, idx, s, picked, w, grad):
    """The gradient of the logits: through the renormalisation, then the scores."""
    g = torch.where(idx >= 0, grad.double(), 0.0)
    at = idx.clamp(min=0)
    if c["renormalize"] and c["score"] == "softmax":
        p = w / c["scale"]
        d = w * (g - (g * p).sum(-1, keepdim=True))
    elif c["renormalize"]:
        total = picked.sum(-1, keepdim=True) + 1e-20
        ds = c["scale"] / total * (g - (g * picked).sum(-1, keepdim=True) / total)
        d = ds * picked * (1.0 - picked)
    elif c["score"] == "sigmoid":
        d = c["scale"] * g * picked * (1.0 - picked)
    else:
        d = c["scale"] * g * picked
    d = torch.where(idx >= 0, d, 0.0)
    out = torch.zeros_like(s).scatter_add_(1, at, d)
    if c["score"] == "softmax" and not c["renormalize"]:
        out = out - s * d.sum(-1, keepdim=True)
    return out.to(logits.dtype)


def _plain_moe(state):
    c = state["case"]
    fmt, n = c["format"], c["E_local"]
    idx, _, _, w = _route(state["logits"], state["bias"], c)
    T, k = idx.shape
    x = _decode(*_encode(state["x"].float(), fmt, state["g_x"]), fmt, state["g_x"])
    # the (token, expert) pairs of this slice, in expert order, padded to the fullest expert
    e = (idx - state["first"]).flatten()
    e = torch.where((idx.flatten() < 0) | (e < 0) | (e >= n), n, e)
    order = torch.argsort(e, stable=True)
    count = torch.bincount(e, minlength=n + 1)
    start = count.cumsum(0) - count
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device=x.device) - start[e[order]]
    most = max(1, int(count[:n].max()))
    row = torch.where(e < n, e * most + place, n * most)  # the last row takes the others' pairs
    rows = torch.zeros(n * most + 1, x.shape[1], device=x.device)
    rows[row] = x.repeat_interleave(k, dim=0)
    of = lambda m: _decode(m["codes"], m["scales"], fmt,  # noqa: E731
                           None if m["g"] is None else m["g"][:, None, None])
    g1 = torch.bmm(rows[:-1].view(n, most, -1), of(state["w13"]).transpose(1, 2))
    gate, up = g1[..., :c["I"]], g1[..., c["I"]:]
    h = gate * (up / (1.0 + torch.exp(-up)))
    h = _decode(*_encode(h, fmt, state["g_c"]), fmt, state["g_c"])
    o = torch.bmm(h, of(state["w2"]).transpose(1, 2)).reshape(n * most, -1)
    o = torch.cat([o, o.new_zeros(1, o.shape[1])])[row].view(T, k, -1)
    return (o * w.float()[..., None]).sum(1).to(torch.bfloat16)


def _plain(state):
    c = state["case"]
    kind = c["kind"]
    if kind == "route":
        idx, s, picked, w = _route(state["logits"], state["bias"], c)
        got = dict(idx=idx.to(torch.int32), w=w.float())
        if c["grad"]:
            got["grad"] = _route_grad(state["logits"], c, idx, s, picked, w, state["grad"])
        return got
    if kind == "quant":
        codes, scales = _encode(state["x"].float(), c["format"], state["g"])
        return _decode(codes, scales, c["format"], state["g"]).to(torch.bfloat16)
    if kind == "matmul":
        a, b = state["a"], state["b"]
        y = _decode(a["codes"], a["scales"], c["format"], a["g"]) @ _decode(
            b["codes"], b["scales"], c["format"], b["g"]).t()
        return y.to(torch.bfloat16)
    return _plain_moe(state)


def _own(state):
    f = _fmoe()
    c = state["case"]
    kind = c["kind"]
    held = lambda m: f.Fp4Tensor(m["codes"], m["tiles"], c["format"], m["g"])  # noqa: E731
    how = {k: c[k] for k in ("score", "n_group", "topk_group", "group_score", "renormalize",
                             "scale") if k in c}
    if kind == "route":
        idx, w = f.route_experts(state["logits"], c["top_k"], bias=state["bias"], **how)
        got = dict(idx=idx, w=w)
        if c["grad"]:
            got["grad"] = f.route_experts_backward(
                state["grad"], state["logits"], idx, score=c["score"],
                renormalize=c["renormalize"], scale=c["scale"])
        return got
    if kind == "quant":
        q = f.quantize_fp4(state["x"], c["format"], global_scale=state["g"])
        return f.dequantize_fp4(q, torch.bfloat16)
    if kind == "matmul":
        return f.matmul_fp4(held(state["a"]), held(state["b"]))
    idx, w = f.route_experts(state["logits"], c["top_k"], bias=state["bias"], **how)
    return f.forward_fp4(state["x"], idx, w, held(state["w13"]), held(state["w2"]),
                         state["first"], input_scale=state["g_x"],
                         intermediate_scale=state["g_c"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------- the work
def work(case):
    c = case
    kind = c["kind"]
    if kind in ("route", "moe"):
        size = 4 if kind == "moe" or c["dtype"] == "fp32" else 2
        pairs = c["T"] * c["top_k"]
        nbytes = c["T"] * c["E"] * size + pairs * 8
        flops = c["T"] * c["E"] * 4  # the scores: an exponential, an addition, a division, a compare
        if c.get("grad"):
            nbytes += c["T"] * c["E"] * size + pairs * 4
            flops += c["T"] * c["E"] * 2 + pairs * 4
    if kind == "route":
        return dict(bytes=nbytes, flops=flops)
    held = lambda rows, K: rows * (K // 2 + -(-K // _BLOCK[c["format"]]))  # noqa: E731
    if kind == "quant":
        size = 4 if c["dtype"] == "fp32" else 2
        n = c["M"] * c["K"]
        # read, written as 4-bit blocks, those read, the values written
        return dict(bytes=n * size + 2 * held(c["M"], c["K"]) + n * 2, flops=n * 4)
    if kind == "matmul":
        return dict(bytes=held(c["M"], c["K"]) + held(c["N"], c["K"]) + c["M"] * c["N"] * 2,
                    flops=2 * c["M"] * c["N"] * c["K"])
    T, H, I = c["T"], c["H"], c["I"]
    share = c["top_k"] / c["E"]
    active = c["E_local"] * (1.0 - (1.0 - share) ** T)  # experts that get a token
    rows = T * c["E_local"] * share
    return dict(bytes=nbytes + active * (held(2 * I, H) + held(H, I)) + T * H * 4,
                flops=flops + rows * 6 * H * I)


# ------------------------------------------------------------------------------- 64 bits
def _fp4_64(x, fmt, g):
    """The values that x (64 bits) is quantised to, from the definition: the nearest value of the
    4-bit grid times the block's scale."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64,
                        device=x.device)
    b = x.unflatten(-1, (-1, _BLOCK[fmt]))
    top = b.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        # the largest power of two that is not above the largest magnitude (frexp is exact)
        power = torch.frexp(top.clamp(min=2.0 ** -140)).exponent.double() - 1
        d = torch.round(torch.exp2(power + 140)) * 2.0 ** -142
        d = d.clamp(2.0 ** -127, 2.0 ** 127)
    else:
        g = 1.0 if g is None else g.double()
        d = (top / (6.0 * g)).clamp(max=448.0).float().to(torch.float8_e4m3fn).double() * g
    q = torch.where(d > 0, b / torch.where(d > 0, d, 1.0), 0.0)
    low = (torch.bucketize(q.abs(), grid, right=True) - 1).clamp(0, 7)
    high = (low + 1).clamp(max=7)
    to_low, to_high = q.abs() - grid[low], grid[high] - q.abs()
    up = (to_high < to_low) | ((to_high == to_low) & (low % 2 == 1))
    return (grid[torch.where(up & (high > low), high, low)] * q.sign() * d).flatten(-2)


def _held_64(m, fmt):
    """A 4-bit matrix's values in 64 bits."""
    low, high = m["codes"] & 15, m["codes"] >> 4
    code = torch.stack([low, high], -1).flatten(-2)
    mag, exp = (code & 1).double(), ((code >> 1) & 3).double()
    v = torch.where(exp == 0, mag * 0.5, (1.0 + mag * 0.5) * torch.exp2(exp - 1.0))
    v = torch.where(code >= 8, -v, v)
    if fmt == "mxfp4":
        s = torch.exp2(m["scales"].double() - 127.0)
    else:
        s = m["scales"].view(torch.float8_e4m3fn).double()
    return v * s.repeat_interleave(_BLOCK[fmt], dim=-1)


def _route_64(logits, bias, c):
    """The scores and, by repeated maxima, the chosen experts of each token."""
    x = logits.double()
    never = ~(x > -math.inf)
    if c["score"] == "softmax":
        s = torch.softmax(x.masked_fill(never, -math.inf), -1).masked_fill(never, 0.0)
        s = torch.nan_to_num(s)
    else:
        s = torch.sigmoid(x).masked_fill(never, 0.0)
    worth = (s if bias is None else s + bias.double()).masked_fill(never, -math.inf)
    rank = (x if bias is None else worth).masked_fill(never, -math.inf)
    T, E = x.shape
    n = c["n_group"]
    if n > 1:
        groups = (rank if c["group_score"] == "max" else worth).reshape(T, n, E // n)
        value = (groups.amax(-1) if c["group_score"] == "max"
                 else groups.topk(2, dim=-1).values.sum(-1))
        better = (value[:, None] > value[..., None]) | (
            (value[:, None] == value[..., None])
            & (torch.arange(n, device=x.device)[None, None] < torch.arange(n, device=x.device)[None, :, None]))
        kept = better.sum(-1) < c["topk_group"]
        rank = torch.where(kept[..., None], rank.reshape(T, n, E // n), -math.inf).reshape(T, E)
    idx = []
    for _ in range(c["top_k"]):
        top = rank.amax(-1, keepdim=True)
        at = (rank == top).to(torch.int8).argmax(-1, keepdim=True)
        idx.append(torch.where(top > -math.inf, at, -1))
        rank = rank.scatter(1, at, -math.inf)
    return torch.cat(idx, 1), s


def _weights_64(x, s, idx, c):
    """Weights from scores, differentiable in x for the gradient."""
    live = idx >= 0
    p = torch.where(live, s.gather(1, idx.clamp(min=0)), 0.0)
    if c["renormalize"] and c["score"] == "softmax":
        z = torch.where(live, x.gather(1, idx.clamp(min=0)), -1e300)
        p = torch.where(live, torch.softmax(z, -1), 0.0)
    elif c["renormalize"]:
        p = p / (p.sum(-1, keepdim=True) + 1e-20)
    return p * c["scale"]


def exact(case, seed):
    c, st = case, prepare(case, seed)
    kind = c["kind"]
    if kind == "route":
        idx, _ = _route_64(st["logits"], st["bias"], c)
        x = st["logits"].double()
        x = torch.where(x > -math.inf, x, -1e4).requires_grad_(c["grad"])
        s = torch.softmax(x, -1) if c["score"] == "softmax" else torch.sigmoid(x)
        w = _weights_64(x, s, idx, c)
        got = dict(idx=None, w=w.detach())
        if c["grad"]:
            w.backward(st["grad"].double())
            got["grad"] = x.grad
        return got
    fmt = c["format"]
    if kind == "quant":
        return _fp4_64(st["x"].double(), fmt, st["g"])
    scaled = lambda m: _held_64(m, fmt) * (1.0 if m["g"] is None else m["g"].double())  # noqa: E731
    if kind == "matmul":
        return scaled(st["a"]) @ scaled(st["b"]).t()
    idx, s = _route_64(st["logits"], st["bias"], c)
    w = _weights_64(st["logits"].double(), s, idx, c)
    x = _fp4_64(st["x"].double(), fmt, st["g_x"])
    y = torch.zeros(c["T"], c["H"], dtype=torch.float64, device="cuda")
    one = lambda m, e: {k: None if v is None else v[e] for k, v in m.items()}  # noqa: E731
    for e in range(c["E_local"]):
        token, k = torch.nonzero(idx == e + st["first"], as_tuple=True)
        if not len(token):
            continue
        g = x[token] @ scaled(one(st["w13"], e)).t()
        h = g[:, :c["I"]] * g[:, c["I"]:] * torch.sigmoid(g[:, c["I"]:])
        o = _fp4_64(h, fmt, st["g_c"]) @ scaled(one(st["w2"], e)).t()
        y.index_add_(0, token, o * w[token, k][:, None])
    return y
