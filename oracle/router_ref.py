"""Expert routing in 64 bits on the CPU: the definition of include/fmoe.h fmoe_route_experts,
token by token, for the tests."""
import math

import torch


def scores(x, score):
    """s of one token's logits (float64 list), None where an expert may not be used."""
    usable = [v > -math.inf for v in x]  # False for NaN too
    if score == "sigmoid":
        return [(1.0 / (1.0 + math.exp(-v)) if v > -700.0 else math.exp(v)) if u else None
                for v, u in zip(x, usable)]
    top = max((v for v, u in zip(x, usable) if u), default=0.0)
    e = [(1.0 if v == top else math.exp(v - top)) if u else None for v, u in zip(x, usable)]
    total = sum(v for v in e if v is not None)
    return [None if v is None else v / total for v in e]


def route(logits, bias, top_k, score, n_group=1, topk_group=1, group_score="top2",
          renormalize=True, scale=1.0):
    """(idx int32 [T, K], w float64 [T, K])."""
    T, E = logits.shape
    idx = torch.full((T, top_k), -1, dtype=torch.int32)
    w = torch.zeros(T, top_k, dtype=torch.float64)
    b = None if bias is None else bias.double().tolist()
    G = E // n_group
    for t, x in enumerate(logits.double().tolist()):
        s = scores(x, score)
        worth = [None if v is None else v + (0.0 if b is None else b[e]) for e, v in enumerate(s)]
        worth = [None if v is None or not v > -math.inf else v for v in worth]
        order = [None if v is None else (x[e] if b is None else v) for e, v in enumerate(worth)]
        left = [e for e in range(E) if order[e] is not None]
        if n_group > 1:
            value = []
            for g in range(n_group):
                of = sorted(((order if group_score == "max" else worth)[e]
                             for e in left if e // G == g), reverse=True)
                if group_score == "max":
                    value.append(of[0] if of else -math.inf)
                else:
                    value.append(of[0] + of[1] if len(of) > 1 else -math.inf)
            kept = sorted(range(n_group), key=lambda g: (-value[g], g))[:topk_group]
            left = [e for e in left if e // G in kept]
        picks = sorted(left, key=lambda e: (-order[e], e))[:top_k]
        if not picks:
            continue
        p = [s[e] for e in picks]
        if renormalize and score == "softmax":
            top = max(x[e] for e in picks)
            p = [1.0 if x[e] == top else math.exp(x[e] - top) for e in picks]
            p = [v / sum(p) for v in p]
        elif renormalize:
            total = sum(p) + 1e-20
            p = [v / total for v in p]
        idx[t, :len(picks)] = torch.tensor(picks, dtype=torch.int32)
        w[t, :len(picks)] = torch.tensor(p, dtype=torch.float64) * scale
    return idx, w


def weights(x, idx, score, renormalize, scale):
    """The weights of given picks as a differentiable function of float64 logits; -inf and NaN
    logits take no part."""
    dead = ~(x > -math.inf)
    x = torch.where(dead, torch.full_like(x, -1e5), x)
    at = idx.long().clamp(min=0)
    live = (idx >= 0) & ~dead.gather(1, at)
    if score == "softmax":
        s = torch.softmax(x, -1)
    else:
        s = torch.sigmoid(x)
    p = torch.where(live, s.gather(1, at), 0.0)
    if renormalize and score == "softmax":
        z = torch.where(live, x.gather(1, at), -1e6)
        p = torch.where(live, torch.softmax(z, -1), 0.0)
    elif renormalize:
        p = p / (p.sum(-1, keepdim=True) + 1e-20)
    return p * scale
