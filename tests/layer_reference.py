"""Norm, scored router, gate and gradient clipping (include/hccl/hccl_amd_experts.h) in 64 bits on the CPU, from their formulas, each with the
magnitude that its rounding errors are relative to.

U = 2^-24 is half a unit in the last place of 32 bits; bounds count roundings (experts_reference.close adds half a unit of the output's type).
"""
import numpy as np


def norm(x, residual, gain, eps):
    """s and y."""
    s = x if residual is None else x + residual
    with np.errstate(all="ignore"):
        r = 1 / np.sqrt((s * s).mean(1, keepdims=True) + eps)
        return s, s * r * (1 if gain is None else gain)


def norm_grad(dy, s, gain, eps, dsum):
    """dx, dgain and their magnitudes."""
    g = np.ones(s.shape[1]) if gain is None else gain
    with np.errstate(all="ignore"):
        r = 1 / np.sqrt((s * s).mean(1, keepdims=True) + eps)
        n, d = s * r, dy * g
        mean, size = (d * n).mean(1, keepdims=True), np.abs(d * n).mean(1, keepdims=True)
        dx = r * (d - n * mean) + (0 if dsum is None else dsum)
        dx_size = r * (np.abs(d) + np.abs(n) * size) + (0 if dsum is None else np.abs(dsum))
        return dx, (dy * n).sum(0), dx_size, np.abs(dy * n).sum(0)


def sigmoid(g):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-g))


def gate(g, u):
    return g * sigmoid(g) * u


def gate_grad(da, g, u):
    """dg, du and their magnitudes."""
    t, rest = sigmoid(g), sigmoid(-g)
    return da * u * t * (1 + g * rest), da * g * t, np.abs(da * u) * t * (1 + np.abs(g) * rest), np.abs(da * g * t)


def scores(x, kind):
    """Rows of scores; a softmax leaves NaN out, and +inf takes all."""
    if kind == "sigmoid":
        with np.errstate(invalid="ignore"):
            return sigmoid(x)
    top = np.fmax.reduce(x, axis=1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.where(x == top, 1.0, np.where(x < top, np.exp(x - top), 0.0))
        return e / e.sum(1, keepdims=True)


def route(x, kind, bias, groups, kept, group_top, topk, renorm, scale, mask):
    """x: logits in 64 bits [tokens, experts]."""
    T, E = x.shape
    size = E // groups
    s = scores(x, kind) if T else x
    expert, weights = np.full((T, topk), -1, np.int32), np.zeros((T, topk))
    for t in range(T):
        if mask is not None and mask[t] == 0:
            continue
        key = s[t] + (0 if bias is None else bias)
        can = (x[t] > -np.inf) & (key > -np.inf)
        of = {}
        for g in range(groups):
            best = sorted((key[e] for e in range(g * size, (g + 1) * size) if can[e]), reverse=True)[:group_top]
            if best:
                of[g] = sum(best)
        use = sorted(of, key=lambda g: (-of[g], g))[:kept]
        order = sorted((e for e in range(E) if can[e] and e // size in use), key=lambda e: (-key[e], e))[:topk]
        if not order:
            continue
        expert[t, :len(order)] = order
        bad = kind == "softmax" and not (np.where(np.isnan(x[t]), np.inf, x[t]) < np.inf).all()
        if not renorm:
            w = s[t][order]
        else:
            log = x[t][order] if kind == "softmax" else np.minimum(x[t][order], 0) - np.log1p(np.exp(-np.abs(x[t][order])))
            with np.errstate(invalid="ignore"):
                w = np.exp(log - log.max())
            w = w / w.sum()
        weights[t, :len(order)] = np.nan if bad else scale * w
    counts = np.array([(expert == e).sum() for e in range(E)] + [(expert[:, 0] >= 0).sum()])
    offsets = np.concatenate([[0], np.cumsum(counts[:E])])
    flat = expert.reshape(-1)
    row_of = np.full(flat.shape, -1, np.int32)
    order = np.argsort(np.where(flat < 0, E, flat), kind="stable")[:int((flat >= 0).sum())]
    row_of[order] = np.arange(len(order))
    return {"expert": expert, "weights": weights, "row_of": row_of.reshape(expert.shape), "counts": counts, "offsets": offsets, "scores": s}


def route_grad(x, r, kind, topk, renorm, scale, dw):
    """Gradient of the logits and its magnitude, from route()'s result."""
    T, E = x.shape
    out, size = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        n = int((r["expert"][t] >= 0).sum())
        if n == 0:
            continue
        e, w, d, s = r["expert"][t, :n], r["weights"][t, :n], dw[t, :n], r["scores"][t]
        if renorm:
            mean, about = (w / scale * d).sum(), (w / scale * np.abs(d)).sum()
            up, big = w * (d - mean), np.abs(w) * (np.abs(d) + about)
        else:
            up, big = w * d, np.abs(w * d)
        if kind == "sigmoid":
            rest = sigmoid(-x[t][e])
            up, big = up * rest, big * rest
        out[t, e], size[t, e] = up, big
        if kind == "softmax" and not renorm:
            out[t] -= s * up.sum()
            size[t] += s * big.sum()
    return out, size


def bias_step(counts, rate, bias):
    n = counts.astype(np.int64)
    return (bias + np.float32(rate) * np.sign(n.sum() - len(n) * n).astype(np.float32)).astype(np.float32)


def route_many(x, kind, bias, groups, kept, group_top, topk, renorm, scale):
    """route() for finite logits of many tokens, all tokens at once."""
    T, E = x.shape
    s = scores(x, kind)
    key = s + (0 if bias is None else bias)
    of = -np.sort(-key.reshape(T, groups, -1), axis=2)[:, :, :group_top]
    of = of[:, :, 0] + (of[:, :, 1] if of.shape[2] > 1 else 0)
    use = np.argsort(-of, axis=1, kind="stable")[:, :kept]                 # (of equal ones the lowest stays in front)
    keep = np.zeros((T, groups), bool)
    np.put_along_axis(keep, use, True, 1)
    key = np.where(np.repeat(keep, E // groups, 1), key, -np.inf)
    expert = np.argsort(-key, axis=1, kind="stable")[:, :topk]
    p = np.take_along_axis(s, expert, 1)
    counts = np.concatenate([np.bincount(expert.reshape(-1), minlength=E), [T]])
    order = np.argsort(expert.reshape(-1), kind="stable")
    row_of = np.empty(T * topk, np.int32)
    row_of[order] = np.arange(T * topk)
    return {"expert": expert, "weights": scale * p / (p.sum(1, keepdims=True) if renorm else 1), "row_of": row_of.reshape(T, topk), "counts": counts,
            "offsets": np.concatenate([[0], np.cumsum(counts[:E])]), "scores": s}
