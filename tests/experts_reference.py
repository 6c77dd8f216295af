"""The experts' operators (include/hccl/hccl_amd_experts.h) in 64 bits on the CPU, from their formulas, and the bounds their
32-bit results are held to.

Bounds: U = 2^-24 is half a unit in the last place of 32 bits, and a sum of n products in 32 bits is off by at most
(n + 1) U times the sum of the products' magnitudes, whatever its order.  A result of fewer bits adds half a unit of its own.
"""
import numpy as np
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a unit, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
FP32, E8M0 = 1, 2


def up128(n):
    return (n + 127) // 128 * 128


# ---- 8-bit blocks: exact, the definition says where it rounds ---------------------------------------------------------------

def block_scale(top, kind):
    """(what is stored, what values are multiplied by, the scale's value) of blocks with these maxima (numpy float32)."""
    top = np.maximum(top.astype(np.float32), np.float32(2.0 ** -96))
    if kind == FP32:
        stored = top * (np.float32(1) / np.float32(448))
        return stored, np.float32(1) / top * np.float32(448), stored.astype(np.float64)
    m, p = np.frexp(top.astype(np.float64))               # m in [1/2, 1)
    power = p - 9 + (m > 0.875)
    return (power + 127).astype(np.uint8), np.exp2(-power.astype(np.float64)).astype(np.float32), np.exp2(power.astype(np.float64))


def to_fp8(v):
    """float32 -> codes; infinities and NaN become 0x7f."""
    q = torch.from_numpy(np.ascontiguousarray(np.where(np.isfinite(v), v, 0).astype(np.float32))).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    return np.where(np.isfinite(v), q, np.uint8(0x7f)).astype(np.uint8)


def from_fp8(q):
    return torch.from_numpy(np.ascontiguousarray(q)).view(torch.float8_e4m3fn).to(torch.float32).numpy().astype(np.float64)


def same_codes(got, want):
    """NaN has two codes: its sign says nothing."""
    return np.array_equal(np.where((got & 0x7f) == 0x7f, 0x7f, got), want)


def tops(v, axis):
    a = np.abs(v)
    return np.max(np.where(np.isfinite(a), a, 0), axis=axis)


def quant_rows(x, kind):
    """x float32 [rows, width] -> codes [rows, padded], stored scales, scale values [rows, blocks]."""
    rows, width = x.shape
    x = np.pad(x, ((0, 0), (0, up128(width) - width))).reshape(rows, -1, 128)
    stored, times, value = block_scale(tops(x, 2), kind)
    with np.errstate(invalid="ignore", over="ignore"):
        return to_fp8((x * times[..., None]).reshape(rows, -1)), stored, value


def quant_weights(w, kind):
    """w float32 [experts, n, k] -> codes [experts, n, padded k], stored scales, scale values [experts, nb, kb]."""
    e, n, k = w.shape
    blocks = np.pad(w, ((0, 0), (0, up128(n) - n), (0, up128(k) - k))).reshape(e, up128(n) // 128, 128, up128(k) // 128, 128)
    stored, times, value = block_scale(tops(blocks, (2, 4)), kind)
    with np.errstate(invalid="ignore", over="ignore"):
        q = to_fp8(blocks * times[:, :, None, :, None])
    return q.reshape(e, up128(n), up128(k))[:, :n], stored, value


def quant_columns(x, offsets, kind):
    """x float32 [rows, width] -> codes [width, columns in use], stored scales, scale values [blocks in use, width]."""
    q, stored, value = [], [], []
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        if hi > lo:
            a, s, v = quant_rows(np.ascontiguousarray(x[lo:hi].T), kind)
            q.append(a)
            stored.append(s.T)
            value.append(v.T)
    if not q:
        return np.zeros((x.shape[1], 0), np.uint8), np.zeros((0, x.shape[1])), np.zeros((0, x.shape[1]))
    return np.concatenate(q, 1), np.concatenate(stored), np.concatenate(value)


def rows_values(q, scale):
    return from_fp8(q) * np.repeat(scale, 128, -1)


def weights_values(q, scale):
    n = q.shape[1]
    return from_fp8(q) * np.repeat(np.repeat(scale, 128, 1)[:, :n], 128, 2)


# ---- router ------------------------------------------------------------------------------------------------------------------

def route(logits, topk, renorm, mask, loss_scale):
    """logits float64 [tokens, experts] (numpy).  Returns a dict of numpy arrays; weights and loss in 64 bits."""
    T, E = logits.shape
    live = np.ones(T, bool) if mask is None else mask != 0
    expert = np.full((T, topk), -1, np.int32)
    weights = np.zeros((T, topk))
    p = np.zeros((T, E))
    for t in range(T):
        if not live[t]:
            continue
        x = logits[t]
        can = [e for e in range(E) if x[e] > -np.inf]     # (a comparison with NaN is false)
        order = sorted(can, key=lambda e: (-x[e], e))[:topk]
        if not order:
            continue
        expert[t, :len(order)] = order
        with np.errstate(invalid="ignore"):
            z = np.exp(x - x[order[0]])
            p[t] = z / z.sum()
        chosen = p[t][order]
        weights[t, :len(order)] = chosen if not renorm else (z[order] / z[order].sum() if np.isfinite(z.sum()) else np.nan)
    counts = np.array([(expert == e).sum() for e in range(E)] + [(expert[:, 0] >= 0).sum() if topk else 0])
    rows, tokens = counts[:E].sum(), counts[E]
    offsets = np.concatenate([[0], np.cumsum(counts[:E])])
    row_of = np.full((T, topk), -1, np.int32)
    at = offsets[:E].copy()
    for t in range(T):
        for j in range(topk):
            if expert[t, j] >= 0:
                row_of[t, j] = at[expert[t, j]]
                at[expert[t, j]] += 1
    loss = 0.0 if rows == 0 else loss_scale * E * float(np.sum(counts[:E] / rows * (p.sum(0) / tokens)))
    return {"expert": expert, "weights": weights, "row_of": row_of, "counts": counts, "offsets": offsets, "loss": loss, "p": p}


def route_grad(r, topk, renorm, loss_scale, weight_grad, loss_grad):
    """Gradient of <weight_grad, weights> + loss_grad * loss, by the formula, from route()'s result."""
    p, expert, counts = r["p"], r["expert"], r["counts"]
    T, E = p.shape
    rows, tokens = counts[:E].sum(), counts[E]
    g = np.zeros((T, E))
    if loss_grad is not None and rows:
        g[:] = loss_grad * loss_scale * E * counts[:E] / rows / tokens
    out = np.zeros((T, E))
    size = np.zeros((T, E))     # magnitudes that were added up, for the bounds
    for t in range(T):
        n = int((expert[t] >= 0).sum())
        if n == 0:
            continue
        e, gt = expert[t, :n], g[t].copy()
        if weight_grad is not None and not renorm:
            gt[e] += weight_grad[t, :n]
        out[t] = p[t] * (gt - (p[t] * gt).sum())
        size[t] = p[t] * (np.abs(gt) + (p[t] * np.abs(gt)).sum())
        if weight_grad is not None and renorm:
            w = r["weights"][t, :n]
            out[t, e] += w * (weight_grad[t, :n] - (w * weight_grad[t, :n]).sum())
            size[t, e] += w * (np.abs(weight_grad[t, :n]) + (w * np.abs(weight_grad[t, :n])).sum())
    return out, size


def route_finite(logits, topk, renorm, mask, loss_scale, weight_grad, loss_grad):
    """route() and route_grad() for finite logits of many tokens, all tokens at once."""
    T, E = logits.shape
    live = np.ones((T, 1), bool) if mask is None else (mask != 0)[:, None]
    pick = np.argsort(-logits, axis=1, kind="stable")[:, :topk]      # (of equal ones the lowest expert stays in front)
    z = np.exp(logits - logits.max(1, keepdims=True))
    p = np.where(live, z / z.sum(1, keepdims=True), 0)
    chosen = np.take_along_axis(p, pick, 1)
    inside = np.where(live, chosen.sum(1, keepdims=True), 1)
    weights = chosen / inside if renorm else chosen
    expert = np.where(live, pick, -1).astype(np.int32)
    counts = np.concatenate([np.bincount(pick[live[:, 0]].reshape(-1), minlength=E), [live.sum()]])
    rows, tokens = counts[:E].sum(), counts[E]
    order = np.argsort(np.where(live, pick, E).reshape(-1), kind="stable")
    row_of = np.empty(T * topk, np.int32)
    row_of[order] = np.arange(T * topk)
    row_of = np.where(live, row_of.reshape(T, topk), -1)
    loss = loss_scale * E * float(np.sum(counts[:E] / rows * (p.sum(0) / tokens)))
    g = np.broadcast_to(loss_grad * loss_scale * E * counts[:E] / rows / tokens, (T, E)).copy()
    dw = np.where(live, weight_grad, 0)
    if not renorm:
        np.put_along_axis(g, pick, np.take_along_axis(g, pick, 1) + dw, 1)
    grad = p * (g - (p * g).sum(1, keepdims=True))
    size = p * (np.abs(g) + (p * np.abs(g)).sum(1, keepdims=True))
    if renorm:
        for to, d in ((grad, weights * (dw - (weights * dw).sum(1, keepdims=True))), (size, weights * (np.abs(dw) + (weights * np.abs(dw)).sum(1, keepdims=True)))):
            np.put_along_axis(to, pick, np.take_along_axis(to, pick, 1) + d, 1)
    return {"expert": expert, "weights": weights, "row_of": row_of, "counts": counts, "offsets": np.concatenate([[0], np.cumsum(counts[:E])]), "loss": loss}, grad, size


# ---- bounds ------------------------------------------------------------------------------------------------------------------

def close(got, want, bound, dtype=torch.float32):
    """got within bound of want, half a unit of its type added (a bound, so nothing is tuned to a result)."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    both = np.isnan(got) & np.isnan(want)
    room = np.broadcast_to(bound, want.shape) + HALF[dtype] * np.abs(want) * (1 + 2.0 ** -7) + TINY[dtype]
    bad = ~both & ~(np.abs(got - want) <= room)
    return not bad.any()
