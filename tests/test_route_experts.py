"""route_experts and its gradient against the definition in 64 bits.

Tolerances. Weights are fp32: an exponential (2 units in the last place, 2^-22), a sum of at
most 32 positive terms (each addition 2^-24), two divisions and a product (2^-24 each): below
2^-19 relative. The argument of the exponential is rounded once, which adds 2^-24 |x - max|
(|x| <= 64 below: 2^-18). Sum: 2^-17. A gradient adds the difference g - mean of terms of that
accuracy: 2^-16 of the largest |g| * scale, then the rounding of its own type (eps / 2).
"""
import ctypes
import math

import pytest
import torch

from oracle import router_ref as ref

REL = 2.0 ** -17
GRAD = 2.0 ** -16


def _inputs(T, E, dtype, kind, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E, generator=g) * 2.0
    if kind == "ties":
        x = torch.round(x)
    elif kind == "wide":
        x = (x * 12.0).clamp(-60.0, 60.0)
    elif kind == "masked":
        x[torch.rand(T, E, generator=g) < 0.5] = -math.inf
        x[torch.rand(T, E, generator=g) < 0.02] = math.nan
        x[:: 3] = -math.inf  # rows with nothing left
        x[1:2, 1:] = -math.inf  # a row with one expert
    return x.to(dtype)


def _bias(E, kind, dtype, seed):
    if kind == "none":
        return None
    g = torch.Generator().manual_seed(seed + 1)
    b = torch.zeros(E) if kind == "zero" else (torch.rand(E, generator=g) - 0.5) * 0.2
    if kind == "closed":
        b[0] = -math.inf
    return b.to(dtype)


RULES = [
    # E, top_k, n_group, topk_group, group_score
    (256, 8, 8, 4, "top2"), (256, 8, 8, 4, "max"), (60, 4, 1, 1, "top2"), (60, 6, 4, 2, "top2"),
    (1, 1, 1, 1, "top2"), (8, 2, 1, 1, "max"), (16, 4, 4, 2, "top2"), (72, 8, 3, 1, "max"),
    (160, 6, 8, 3, "max"), (512, 16, 32, 7, "top2"), (1000, 32, 4, 2, "top2"), (33, 32, 1, 1, "max"),
    (64, 6, 2, 1, "top2"), (128, 8, 4, 2, "max"), (32, 4, 16, 5, "max"), (512, 8, 2, 1, "max"),
    (1024, 8, 4, 3, "top2"), (384, 15, 2, 1, "top2"), (96, 7, 4, 3, "top2"), (72, 4, 8, 6, "max"),
    (40, 4, 8, 2, "top2"), (640, 8, 4, 2, "top2"), (384, 8, 1, 1, "max"), (66, 5, 2, 2, "top2"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rule", RULES, ids=lambda r: "-".join(map(str, r)))
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("kind,bias,dtype", [
    ("normal", "none", torch.float32), ("normal", "some", torch.float32),
    ("ties", "zero", torch.bfloat16), ("ties", "none", torch.float16),
    ("masked", "some", torch.bfloat16), ("masked", "none", torch.float32),
    ("wide", "closed", torch.float16)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_experts_matches_definition(fmoe, rule, score, kind, bias, dtype, renormalize):
    E, K, n, kg, how = rule
    T = 37
    x = _inputs(T, E, dtype, kind, seed=E + K)
    b = _bias(E, bias, torch.bfloat16 if dtype == torch.bfloat16 else torch.float32, E)
    idx, w = fmoe.route_experts(x.cuda(), K, score=score, bias=None if b is None else b.cuda(),
                                n_group=n, topk_group=kg, group_score=how,
                                renormalize=renormalize, scale=2.5)
    want_idx, want_w = ref.route(x, b, K, score, n, kg, how, renormalize, 2.5)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(idx.cpu(), want_idx)
    # weights below 2^-100 may be flushed by the exponential
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=REL, atol=2.0 ** -100)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0, 1, 2, 7, 8, 9, 1000])
def test_route_experts_lengths(fmoe, T):
    x = _inputs(T, 256, torch.float32, "normal", T)
    b = _bias(256, "some", torch.float32, T)
    idx, w = fmoe.route_experts(x.cuda(), 8, score="sigmoid", bias=b.cuda(), n_group=8,
                                topk_group=4, scale=2.5)
    want_idx, want_w = ref.route(x, b, 8, "sigmoid", 8, 4, "top2", True, 2.5)
    assert torch.equal(idx.cpu(), want_idx)
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=REL, atol=0.0)


@pytest.mark.gpu
def test_route_experts_many_tokens_match_the_bit_exact_router(fmoe):
    """The rule of `route` gives the picks of `route` wherever that one's single precision
    decides the order (ties aside, the two differ only by scores below its resolution)."""
    x = torch.randn(70000, 256, generator=torch.Generator().manual_seed(5)).cuda()
    b = (torch.randn(256, generator=torch.Generator().manual_seed(6)) * 0.1).bfloat16().cuda()
    idx, w = fmoe.route_experts(x, 8, score="sigmoid", bias=b, n_group=8, topk_group=4, scale=2.5)
    idx0, w0 = fmoe.route(x, b, 8, 4, 8, 2.5)
    same = (idx == idx0).all(1)
    # a gap below 2^-22 between two neighbours of the order: about 256 * 9 * 2^-21 of the tokens
    assert (~same).float().mean().item() < 5e-3
    torch.testing.assert_close(w[same], w0[same], rtol=2 * REL, atol=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_experts_decides_below_single_precision(fmoe, score):
    """Scores that round to the same fp32 value but differ: the larger one is picked first."""
    E = 64
    x = torch.full((3, E), -4.0)
    b = torch.zeros(E)
    # expert 40 and 3 differ by one unit in the last place of a logit near 8, where both scores
    # are equal in fp32; with a bias the order is that of the scores
    x[:, 3] = 12.0
    x[:, 40] = torch.nextafter(torch.tensor(12.0), torch.tensor(13.0))
    x[1, 3], x[1, 40] = x[1, 40].clone(), x[1, 3].clone()
    x[2, 3] = x[2, 40]
    for bias in (None, b, b + 0.25):
        want, _ = ref.route(x, bias, 2, score)
        assert want[:, 0].tolist() == [40, 3, 3]
        got, _ = fmoe.route_experts(x.cuda(), 2, score=score,
                                    bias=None if bias is None else bias.cuda())
        assert torch.equal(got.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,K,n,kg,how", [(256, 8, 8, 4, "top2"), (256, 8, 8, 3, "max"),
                                          (64, 6, 2, 1, "top2"), (32, 4, 1, 1, "max"),
                                          (256, 32, 1, 1, "max"), (1024, 8, 4, 2, "top2")])
def test_route_experts_crowded_scores(fmoe, score, E, K, n, kg, how):
    """Logits a few units in the last place apart, so that many scores, group sums and runners-up
    round alike, in ones, twos and threes; and scores that a bias brings that close."""
    g = torch.Generator().manual_seed(E + K)
    T = 60
    base = torch.randn(T, E, generator=g)
    x = (base * 2).round() / 2 + torch.randint(-3, 4, (T, E), generator=g) * 2.0 ** -22
    b = torch.randint(-2, 3, (E,), generator=g) * 2.0 ** -24 + 0.125
    # expert e + E/2 gets a bias that evens out its score's distance to expert e's
    far = torch.randn(T, E, generator=g)
    c = torch.zeros(E)
    s = torch.sigmoid(far.double())
    c[E // 2:] = (s[0, :E // 2] - s[0, E // 2:]).float()
    for logits, bias in ((x, b), (x, None), (far, c)):
        idx, _ = fmoe.route_experts(logits.cuda(), K, score=score, n_group=n, topk_group=kg,
                                    group_score=how, bias=None if bias is None else bias.cuda())
        want, _ = ref.route(logits, bias, K, score, n, kg, how)
        assert torch.equal(idx.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,K,n,kg", [(256, 8, 8, 4), (160, 6, 8, 3), (64, 6, 2, 1), (32, 4, 16, 5),
                                      (60, 6, 6, 2)])
def test_route_experts_groups_without_bias(fmoe, score, dtype, E, K, n, kg):
    """Groups whose two best scores tie, or differ by less than single precision resolves (large
    negative logits), or of which one or none may be used."""
    g = torch.Generator().manual_seed(E + n)
    x = torch.randint(-6, 7, (80, E), generator=g) / 2 + 0.125
    x[20:40] -= 40
    x[40:60] = 9 + torch.randint(0, 8, (20, E), generator=g) / 16  # sigmoids close to 1
    x[60:] = x[60:].masked_fill(torch.rand(20, E, generator=g) < 0.9, -math.inf)
    x[79] = -math.inf
    x = x.to(dtype)
    idx, w = fmoe.route_experts(x.cuda(), K, score=score, n_group=n, topk_group=kg)
    want_idx, want_w = ref.route(x, None, K, score, n, kg, "top2")
    assert torch.equal(idx.cpu(), want_idx)
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=REL, atol=2.0 ** -100)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,K,n,kg,how", [(256, 8, 1, 1, "max"), (64, 32, 1, 1, "max"),
                                          (160, 6, 8, 3, "top2"), (128, 8, 4, 2, "max"),
                                          (384, 9, 2, 1, "top2"), (1024, 12, 32, 9, "max")])
def test_route_experts_logits_that_share_their_upper_bits(fmoe, score, E, K, n, kg, how):
    """fp32 logits without a bias: equal ones, ones a unit in the last place apart, and most of a
    row at the type's lowest value."""
    g = torch.Generator().manual_seed(E + K)
    x = torch.randn(90, E, generator=g)
    x[:30] = (x[:30] * 4).round() / 4
    x[30:60] = (x[30:60] * 4).round() / 4
    x[30:60] *= 1 + torch.randint(0, 3, (30, E), generator=g) * 2.0 ** -23
    x[60:].masked_fill_(torch.rand(30, E, generator=g) < 0.95, torch.finfo(torch.float32).min)
    idx, w = fmoe.route_experts(x.cuda(), K, score=score, n_group=n, topk_group=kg, group_score=how)
    want_idx, want_w = ref.route(x, None, K, score, n, kg, how)
    assert torch.equal(idx.cpu(), want_idx)
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=REL, atol=2.0 ** -100)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_experts_infinite_logits(fmoe, score):
    x = torch.randn(4, 32, generator=torch.Generator().manual_seed(0))
    x[0, 7] = math.inf
    x[1, 7] = x[1, 20] = math.inf
    x[2, 5] = -0.0
    x[2, 4] = 0.0
    x[2, :4] = x[2, 6:] = -1.0
    for renormalize in (True, False):
        idx, w = fmoe.route_experts(x.cuda(), 2, score=score, renormalize=renormalize)
        want_idx, want_w = ref.route(x, None, 2, score, renormalize=renormalize)
        assert torch.equal(idx.cpu(), want_idx)
        torch.testing.assert_close(w.cpu().double(), want_w, rtol=REL, atol=0.0)
    assert want_idx[2].tolist() == [4, 5]


@pytest.mark.gpu
def test_route_experts_strided_logits(fmoe):
    """Rows inside a wider matrix, an odd offset, a transposed and a broadcast matrix."""
    wide = torch.randn(50, 301, generator=torch.Generator().manual_seed(1)).cuda()
    for x in (wide[:, 3:131], wide[::2, :64], wide.t()[:96], wide[:1, :64].expand(9, 64),
              wide.bfloat16()[:, 1:65]):
        idx, w = fmoe.route_experts(x, 4, score="softmax")
        want_idx, want_w = ref.route(x.float().cpu(), None, 4, "softmax")
        assert torch.equal(idx.cpu(), want_idx)
        torch.testing.assert_close(w.cpu().double(), want_w, rtol=REL, atol=0.0)
        gw = torch.randn(w.shape, generator=torch.Generator().manual_seed(2)).cuda()
        got = fmoe.route_experts_backward(gw, x, idx)
        same = fmoe.route_experts_backward(gw, x.contiguous(), idx)
        assert torch.equal(got, same)


def _grad_of(x, idx, gw, score, renormalize, scale):
    x = x.double().clone().requires_grad_(True)
    ref.weights(x, idx, score, renormalize, scale).backward(gw.double())
    return torch.where(x.detach() > -math.inf, x.grad, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("E,K", [(256, 8), (60, 4), (1, 1), (8, 8), (1000, 32), (33, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["normal", "masked"])
def test_gradient_matches_definition(fmoe, E, K, score, renormalize, dtype, kind):
    T = 19
    x = _inputs(T, E, dtype, kind, seed=E)
    gw = torch.randn(T, K, generator=torch.Generator().manual_seed(7))
    leaf = x.cuda().requires_grad_(True)
    idx, w = fmoe.route_experts(leaf, K, score=score, renormalize=renormalize, scale=1.5)
    w.backward(gw.cuda())
    want = _grad_of(x, idx.cpu(), gw, score, renormalize, 1.5)
    assert leaf.grad.dtype == dtype
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    # a value below fp16's normal range is rounded to a multiple of 2^-24
    atol = GRAD * 1.5 * gw.abs().max().item() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    torch.testing.assert_close(leaf.grad.cpu().double(), want, rtol=half + REL, atol=atol)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_matches_differences(fmoe, score, renormalize):
    """Central differences of the forward pass itself, along random directions. The step h leaves
    h^2 of the third derivative (below 1, scaled by |v|^3) and 2^-24 / h of rounding."""
    T, E, K, h = 5, 24, 4, 2.0 ** -8
    x = _inputs(T, E, torch.float32, "normal", 3).cuda()
    gw = torch.randn(T, K, generator=torch.Generator().manual_seed(4)).cuda()
    idx, _ = fmoe.route_experts(x, K, score=score, renormalize=renormalize)
    grad = fmoe.route_experts_backward(gw, x, idx, score=score, renormalize=renormalize)
    for seed in range(4):
        v = torch.randn(T, E, generator=torch.Generator().manual_seed(seed)).cuda()
        f = []
        for step in (h, -h):
            i, w = fmoe.route_experts(x + step * v, K, score=score, renormalize=renormalize)
            # the picks may swap places: bring the weights into the order of `idx`
            dense = torch.zeros(T, E, device="cuda").scatter_(1, i.long(), w)
            f.append((dense.gather(1, idx.long()) * gw).sum().item())
        want = (f[0] - f[1]) / (2 * h)
        bound = h * h * v.abs().pow(3).sum().item() * gw.abs().max().item() + T * K * 2.0 ** -23 / h
        assert abs((grad * v).sum().item() - want) < bound


@pytest.mark.gpu
def test_gradient_of_repeated_and_foreign_indices(fmoe):
    """An expert named twice gets both terms; indices outside the experts take no part."""
    x = torch.randn(3, 40, generator=torch.Generator().manual_seed(0))
    idx = torch.tensor([[5, 5, 7, 0], [39, -1, 40, 39], [1, 2, 3, -7]], dtype=torch.int32)
    gw = torch.randn(3, 4, generator=torch.Generator().manual_seed(1))
    known = torch.where((idx >= 0) & (idx < 40), idx, -1)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            got = fmoe.route_experts_backward(gw.cuda(), x.cuda(), idx.cuda(), score=score,
                                              renormalize=renormalize)
            want = _grad_of(x, known, gw, score, renormalize, 1.0)
            torch.testing.assert_close(got.cpu().double(), want, rtol=REL,
                                       atol=GRAD * gw.abs().max().item())


@pytest.mark.gpu
def test_gradient_of_a_broadcast_sum(fmoe):
    """A gradient that arrives broadcast (of a sum) equals the laid-out one."""
    x = torch.randn(6, 16, generator=torch.Generator().manual_seed(0)).cuda().requires_grad_(True)
    idx, w = fmoe.route_experts(x, 4, renormalize=False)
    w.sum().backward()
    want = fmoe.route_experts_backward(torch.ones_like(w), x.detach(), idx, renormalize=False)
    assert torch.equal(x.grad, want)
    assert not idx.requires_grad


@pytest.mark.gpu
def test_route_experts_graph_and_streams(fmoe):
    """A captured pass replays on new inputs; a call on another stream orders with that stream."""
    x = torch.randn(100, 128, generator=torch.Generator().manual_seed(0)).cuda()
    gw = torch.randn(100, 6, generator=torch.Generator().manual_seed(1)).cuda()
    call = lambda: (lambda i, w: (i, w, fmoe.route_experts_backward(gw, x, i)))(  # noqa: E731
        *fmoe.route_experts(x, 6))
    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for seed in (2, 3):
        x.copy_(torch.randn(100, 128, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        for got, want in zip(held, call()):
            assert torch.equal(got, want)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        got = call()
    side.synchronize()
    for a, b in zip(got, call()):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,n,kg", [(32, 4, 1), (32, 4, 2), (30, 3, 1), (60, 6, 2), (256, 8, 4),
                                    (24, 12, 5)])
@pytest.mark.parametrize("how", ["top2", "max"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_experts_bias_of_infinity(fmoe, score, E, n, kg, how, dtype):
    """A bias of +inf puts its expert first; a group with no other usable expert is below all
    others by "top2" all the same. The others are out by their logits or by a bias of -inf."""
    G = E // n
    g = torch.Generator().manual_seed(E + n)
    x = torch.randn(12, E, generator=g).to(dtype)
    b = (torch.rand(E, generator=g) - 0.5) * 0.2
    b[1] = math.inf
    x[0, :G] = x[3, :G] = -math.inf
    x[0, 1] = x[3, 1] = 0.5
    x[4, :G] = -math.inf
    x[5, 2 * G:] = -math.inf  # fewer usable experts than picks
    x[5, 0] = math.nan
    second = b.clone()
    second[0:G] = -math.inf
    second[1] = math.inf
    second[E - 1] = math.inf
    for bias in (b, second):
        idx, w = fmoe.route_experts(x.cuda(), 2, score=score, bias=bias.cuda(), n_group=n,
                                    topk_group=kg, group_score=how)
        want_idx, want_w = ref.route(x, bias, 2, score, n, kg, how)
        assert torch.equal(idx.cpu(), want_idx)
        torch.testing.assert_close(w.cpu().double(), want_w, rtol=REL, atol=2.0 ** -100)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,n,kg", [(64, 8, 1), (64, 8, 3), (256, 8, 4), (128, 2, 1), (60, 6, 2)])
@pytest.mark.parametrize("base", [2.0 ** 22, 2.0 ** 17, 2.0 ** 14, -2.0 ** 20])
def test_route_experts_large_logits_that_share_their_upper_bits(fmoe, score, E, n, kg, base):
    """Groups whose two best logits agree in all but their last bits, the larger one at the higher
    index, so far from zero that their difference is large."""
    G = E // n
    g = torch.Generator().manual_seed(E + n)
    # the other experts: out of use, or far below and each with upper bits of its own
    x = torch.full((64, E), -math.inf)
    x[1::2] = -2.0 ** 30 * (1 + torch.arange(E) / 1024)
    step = max(0.25, abs(base) * 2.0 ** -23)
    low = base + torch.randint(0, 8, (64, n), generator=g) * step
    up = torch.randint(0, 40, (64, n), generator=g) * step
    up[:16] += 80.0
    at = torch.randint(0, G // 2, (64, n), generator=g) + torch.arange(n) * G
    x.scatter_(1, at, low)
    x.scatter_(1, at + G // 2, low + up)
    # two groups a step apart, the better one behind the other
    x[0] = -math.inf
    x[0, 0], x[0, G - 1], x[0, G], x[0, 2 * G - 1] = base, base + 100, base, base + 100 + 2 * step
    idx, w = fmoe.route_experts(x.cuda(), 2, score=score, n_group=n, topk_group=kg)
    want_idx, want_w = ref.route(x, None, 2, score, n, kg, "top2")
    assert torch.equal(idx.cpu(), want_idx)
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=REL, atol=2.0 ** -100)


@pytest.mark.gpu
@pytest.mark.parametrize("n,kg", [(1, 1), (4, 4), (3, 3)])
def test_route_experts_scores_that_64_bits_do_not_tell_apart(fmoe, n, kg):
    """Biased scores are compared as 64 bits hold them: sigmoids of 40 and 41 are both 1, and a
    share of 2^-60 is nothing beside a bias of 1. Without a bias the logits themselves decide."""
    E = 48
    x = torch.full((2, E), -3.0)
    x[0, 3], x[0, 40] = 40.0, 41.0
    x[1, 5], x[1, 44] = -44.0, -43.0
    b = torch.zeros(E)
    b[5] = b[44] = 1.0
    for bias, first in ((None, [[40, 3], None]), (b * 0, [[3, 40], None]), (b, [None, [5, 44]])):
        idx, _ = fmoe.route_experts(x.cuda(), 2, score="sigmoid", n_group=n, topk_group=kg,
                                    bias=None if bias is None else bias.cuda())
        want, _ = ref.route(x, bias, 2, "sigmoid", n, kg)
        assert torch.equal(idx.cpu(), want)
        for row, pair in enumerate(first):
            assert pair is None or want[row].tolist() == pair


# ------------------------------------------------------------------------------ refusals
def _router(fmoe, **kw):
    from fmoe_b200.router import FmoeRouter

    base = dict(num_tokens=4, logits_stride=64, num_experts=64, top_k=4, n_group=4, topk_group=2,
                score=0, group_score=0, renormalize=1, logits_dtype=0, bias_dtype=0, scale=1.0)
    base.update(kw)
    return FmoeRouter(**base)


@pytest.mark.parametrize("field,value,code", [
    ("num_tokens", -1, "value"), ("num_experts", 0, "value"), ("num_experts", 1025, "value"),
    ("top_k", 0, "value"), ("top_k", 33, "value"), ("n_group", 0, "value"), ("n_group", 5, "value"),
    ("n_group", 64, "value"), ("topk_group", 0, "value"), ("topk_group", 5, "value"),
    ("score", 2, "value"), ("group_score", -1, "value"), ("logits_stride", 63, "value"),
    ("logits_dtype", 3, "type"), ("bias_dtype", 2, "type")])
def test_router_rejects(fmoe, field, value, code):
    lib = fmoe.load_library()
    out = fmoe.FmoeRouteOut(0, 0)
    r = _router(fmoe, **{field: value})
    rc = lib.fmoe_route_experts(ctypes.byref(r), None, None, ctypes.byref(out), None)
    assert rc == (fmoe.FMOE_ERR_TYPE if code == "type" else fmoe.FMOE_ERR_VALUE)
    assert len(lib.fmoe_last_error()) > 0
    assert lib.fmoe_route_experts_backward(ctypes.byref(r), None, None, None, None, None) == rc


def test_router_rejects_null_and_takes_no_tokens(fmoe):
    lib = fmoe.load_library()
    r, out = _router(fmoe), fmoe.FmoeRouteOut(0, 0)
    assert lib.fmoe_route_experts(ctypes.byref(r), None, None, ctypes.byref(out),
                                  None) == fmoe.FMOE_ERR_VALUE
    assert b"must not be NULL" in lib.fmoe_last_error()
    r = _router(fmoe, num_tokens=0)
    assert lib.fmoe_route_experts(ctypes.byref(r), None, None, ctypes.byref(out),
                                  None) == fmoe.FMOE_OK
    assert lib.fmoe_route_experts(None, None, None, ctypes.byref(out),
                                  None) == fmoe.FMOE_ERR_VALUE


def test_route_experts_rejects_tensors(fmoe):
    with pytest.raises(ValueError, match="2D"):
        fmoe.route_experts(torch.zeros(4), 2)
    with pytest.raises(ValueError, match="CUDA"):
        fmoe.route_experts(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="CUDA"):
        fmoe.route_experts_backward(torch.zeros(4, 2), torch.zeros(4, 8),
                                    torch.zeros(4, 2, dtype=torch.int32))


@pytest.mark.gpu
def test_route_experts_rejects_arguments(fmoe):
    x = torch.zeros(4, 8, device="cuda")
    idx = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError, match="dtype"):
        fmoe.route_experts(x.double(), 2)
    with pytest.raises(ValueError, match="score"):
        fmoe.route_experts(x, 2, score="relu")
    with pytest.raises(ValueError, match="group_score"):
        fmoe.route_experts(x, 2, group_score="sum")
    with pytest.raises(ValueError, match="top_k"):
        fmoe.route_experts(x, 9)
    with pytest.raises(ValueError, match="n_group"):
        fmoe.route_experts(x, 2, n_group=3)
    with pytest.raises(ValueError, match="bias"):
        fmoe.route_experts(x, 2, bias=torch.zeros(7, device="cuda"))
    with pytest.raises(TypeError, match="bias"):
        fmoe.route_experts(x, 2, bias=torch.zeros(8, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="bias must be a CUDA"):
        fmoe.route_experts(x, 2, bias=torch.zeros(8))
    with pytest.raises(TypeError, match="topk_idx"):
        fmoe.route_experts_backward(torch.zeros(4, 2, device="cuda"), x, idx.long())
    with pytest.raises(ValueError, match="grad_w"):
        fmoe.route_experts_backward(torch.zeros(4, 3, device="cuda"), x, idx)
    with pytest.raises(TypeError, match="grad_w"):
        fmoe.route_experts_backward(torch.zeros(4, 2, device="cuda").half(), x, idx)


def test_route_experts_refuses_forward_mode(fmoe):
    """A tangent would be lost without a word: there is no forward-mode derivative."""
    x = torch.randn(4, 8)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="logits.*tangent"):
            fmoe.route_experts(torch.autograd.forward_ad.make_dual(x, x), 2)
    with pytest.raises(ValueError, match="CUDA"):
        fmoe.route_experts(x, 2)


@pytest.mark.gpu
def test_route_experts_refuses_forward_mode_on_the_device(fmoe):
    """Also with a reverse-mode leaf (torch refuses that one itself); the same tensors without
    their tangents are taken."""
    x = torch.randn(4, 8, device="cuda")
    idx, w = fmoe.route_experts(x, 2)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        leaf = torch.autograd.forward_ad.make_dual(x.clone().requires_grad_(True), x)
        for logits in (dual, leaf):
            with pytest.raises((ValueError, RuntimeError)):
                fmoe.route_experts(logits, 2)
        with pytest.raises(ValueError, match="grad_w.*tangent"):
            fmoe.route_experts_backward(torch.autograd.forward_ad.make_dual(w, w), x, idx)
        primal = torch.autograd.forward_ad.unpack_dual(dual).primal
        assert torch.equal(fmoe.route_experts(primal, 2)[0], idx)


def test_router_rejects_addresses_between_elements(fmoe):
    """Refused on the host: the kernels would fault on them."""
    lib = fmoe.load_library()
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        r = _router(fmoe, logits_dtype=dtype, bias_dtype=min(dtype, 1))
        p = ctypes.byref(r)
        for logits, bias, idx, w in ((64 + size // 2, 64, 64, 64), (64, 64 + size // 2, 64, 64),
                                     (64, None, 66, 64), (64, None, 64, 65)):
            out = fmoe.FmoeRouteOut(idx, w)
            assert lib.fmoe_route_experts(p, logits, bias, ctypes.byref(out),
                                          None) == fmoe.FMOE_ERR_VALUE
            assert b"aligned" in lib.fmoe_last_error()
        for grad_w, logits, idx, out in ((66, 64, 64, 64), (64, 64 + size // 2, 64, 64),
                                         (64, 64, 62, 64), (64, 64, 64, 64 + size // 2)):
            assert lib.fmoe_route_experts_backward(p, grad_w, logits, idx, out,
                                                   None) == fmoe.FMOE_ERR_VALUE
            assert b"aligned" in lib.fmoe_last_error()
