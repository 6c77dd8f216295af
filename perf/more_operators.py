"""Timed operators: what a layer with experts and its training step do besides its products and its all-to-all-v.

Rows are added to their residual and normed, for a router in their type and for a product in 8 bits (`norm`); a router scores
experts, with a bias that balances them and in groups (`route`); between an expert's two products a gate multiplies (`gate`); and the
gradients of all of it are held to a norm over all tensors (`clip`).  Cases with `train` run the gradients too.

Shapes: x[rows, width]; h[rows, 2 * width] (gate, then what it multiplies); logits[tokens, experts], row_of[tokens, topk] (the row
in expert order, -1: none).  8-bit rows are padded with zeros to a multiple of 128 and have a scale per 128 values.
"""
import math
import os
import sys

import torch

own = False

_TYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_CODE = {"fp32": 4, "bf16": 11, "fp16": 3}      # HcclDataType
_F8, _F8_SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu
_LEAST = 2.0 ** -96     # the smallest block maximum a scale is made from
_LARGEST = 448.0        # the largest value of the 8-bit type
_EPSILON = 1e-6
_RATE = 1e-3            # step of the balancing bias


def _up(n):
    return (n + 127) // 128 * 128


# ---- cases --------------------------------------------------------------------------------------------------------------


def _norm(name, rows, width, dtype, residual, scale, plain, train):
    """`scale`: 8-bit rows with such scales ("none": not); `plain`: rows in their own type."""
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual, "scale": scale, "plain": plain, "train": train}


def _route(name, tokens, experts, topk, dtype, score, bias, groups, kept, group_top, renorm, masked, train):
    """`kept` of `groups` groups, by the sum of their `group_top` largest; `masked`: the share of tokens that are padding."""
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "topk": topk, "dtype": dtype, "score": score, "bias": bias,
            "groups": groups, "kept": kept, "group_top": group_top, "renorm": renorm, "masked": masked, "train": train}


def _gate(name, rows, width, dtype, scale, used, train):
    """`used`: the share of the rows that are there, known to the device alone."""
    return {"name": name, "op": "gate", "rows": rows, "width": width, "dtype": dtype, "scale": scale, "used": used, "train": train}


def _clip(name, layers, width, hidden, dtype, vectors):
    """`vectors`: the type of the one-dimensional tensors' gradients."""
    return {"name": name, "op": "clip", "layers": layers, "width": width, "hidden": hidden, "dtype": dtype, "vectors": vectors}


def listed():
    return [
        # one token of one decoding step, on its way into an 8-bit product and a router
        _norm("norm_token", 1, 8192, "bf16", True, "fp32", True, False),
        # a training step whose width and rows are no multiple of anything, without a residual
        _norm("norm_odd_train", 5003, 2001, "fp16", False, "none", True, True),
        # a prompt batch, straight into an 8-bit product
        _norm("norm_prompt", 8192, 4096, "bf16", True, "e8m0", False, False),
        # a large training batch
        _norm("norm_large_train", 16384, 8192, "bf16", True, "none", True, True),
        # 64 decoding tokens over 256 experts in eight groups
        _route("route_decode", 64, 256, 8, "bf16", "sigmoid", True, 8, 4, 2, True, 0.0, False),
        # a ragged batch, an odd number of experts in groups of the largest alone, padded sequences
        _route("route_ragged_train", 5003, 60, 6, "fp32", "softmax", False, 4, 2, 1, False, 0.1, True),
        # a large batch
        _route("route_large_train", 65536, 256, 8, "bf16", "sigmoid", True, 8, 4, 2, True, 0.0, True),
        # a decoding step's rows at their experts, in a receive buffer for more of them
        _gate("gate_decode", 512, 2048, "bf16", "fp32", 0.5, False),
        # a prompt batch at its experts
        _gate("gate_prompt", 65536, 2048, "bf16", "e8m0", 1.0, False),
        # a training step's, of an odd number of rows and an odd width
        _gate("gate_odd_train", 16411, 4095, "bf16", "fp32", 0.9, True),
        # two layers of a small model: many short tensors
        _clip("clip_small", 2, 64, 130, "fp32", "fp32"),
        # a large model's gradients, matrices in 16 bits, vectors in 32
        _clip("clip_large", 16, 2048, 8192, "bf16", "fp32"),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n if rng.random() < 0.5 else max(1, n // 64) * 64))


def draw(rng):
    op = rng.choice(["norm", "route", "gate", "clip"])
    if op == "norm":
        width = _log(rng, 64, 16384)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        scale = rng.choice(["none", "fp32", "e8m0"])
        rows = _log(rng, 1, max(1, min(65536, (16384 * 8192) // (width * (2 if dtype == "fp32" else 1)))))
        c = _norm("", rows, width, dtype, rng.random() < 0.7, scale, scale == "none" or rng.random() < 0.5, rng.random() < 0.5)
    elif op == "route":
        experts, groups = rng.choice([(8, 1), (16, 4), (60, 4), (64, 8), (126, 9), (128, 1), (160, 8), (256, 8), (256, 1), (384, 1)])
        kept = rng.randint(1, groups)
        score = rng.choice(["sigmoid", "sigmoid", "softmax"])
        topk = rng.randint(1, min(10, kept * (experts // groups)))
        c = _route("", _log(rng, 1, 65536 * 256 // max(experts, 256)), experts, topk, rng.choice(["fp32", "bf16", "fp16"]), score, rng.random() < 0.7, groups,
                   kept, rng.randint(1, 2), rng.random() < 0.7, rng.choice([0.0, 0.0, 0.1, 0.5]), rng.random() < 0.6)
    elif op == "gate":
        width = _log(rng, 64, 8192)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        rows = _log(rng, 1, max(1, min(65536, (16384 * 4096) // (width * (2 if dtype == "fp32" else 1)))))
        c = _gate("", rows, width, dtype, rng.choice(["none", "fp32", "fp32", "e8m0"]), rng.choice([1.0, 1.0, 0.9, 0.5]), rng.random() < 0.5)
    else:
        width = _log(rng, 32, 4096)
        hidden = _log(rng, width, 4 * width)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        layers = rng.randint(1, max(1, min(40, (1 << (29 if dtype == "fp32" else 30)) // (4 * width * width + 3 * width * hidden))))
        c = _clip("", layers, width, hidden, dtype, rng.choice(["fp32", "bf16"]))
    del c["name"]
    return c


# ---- what a program has in hand --------------------------------------------------------------------------------------------


def _package():
    root = os.getcwd()
    if root not in sys.path:
        sys.path.insert(0, root)
    from __graft_entry__ import load_package
    return load_package()


class _State(dict):
    __getattr__ = dict.__getitem__


_stream = None


def prepare(case, seed):
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()          # the library takes no null stream
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = _State(case, stream=_stream.cuda_stream)
    return globals()["_prepare_" + case["op"]](s, g)


def _rand(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _bytes(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def _rows8(rows, width, scale):
    """Room for 8-bit rows and their scales."""
    W = _up(width)
    return {"q": _bytes(rows * W).view(_F8).reshape(rows, W),
            "scales": torch.empty(rows, W // 128, device="cuda") if scale == "fp32" else _bytes(rows * W // 128).view(_F8_SCALE).reshape(rows, W // 128)}


def _prepare_norm(s, g):
    t, shape = _TYPE[s.dtype], (s.rows, s.width)
    s["x"] = _rand(shape, g).to(t)
    s["r"] = (_rand(shape, g) * torch.exp(0.5 * _rand((s.rows, 1), g))).to(t) if s.residual else None
    s["gain"] = (1 + 0.2 * _rand((s.width,), g)).to(t)
    s["out"] = o = {}
    if s.residual:
        o["sum"] = torch.empty(shape, dtype=t, device="cuda")
    if s.plain:
        o["y"] = torch.empty(shape, dtype=t, device="cuda")
    if s.scale != "none":
        o |= _rows8(s.rows, s.width, s.scale)
    if s.train:
        s["y_grad"], s["sum_grad"] = _rand(shape, g).to(t), _rand(shape, g).to(t)
        o["x_grad"], o["gain_grad"] = torch.empty(shape, dtype=t, device="cuda"), torch.empty(s.width, device="cuda")
        s["workspace"] = _bytes(4 * 2048 * _up(s.width))
    return s


def _prepare_route(s, g):
    T, E, k = s.tokens, s.experts, s.topk
    t = _TYPE[s.dtype]
    s["logits"] = (1.5 * _rand((T, E), g) + 0.5 * _rand((E,), g)).to(t)
    s["mask"] = (torch.rand(T, generator=g, device="cuda") >= s.masked).to(torch.uint8) if s.masked else None
    # the bias has moved by whole steps
    s["b"] = torch.round(40 * _rand((E,), g)) * _RATE if s.bias else None
    s["weight_grad"] = _rand((T, k), g)
    new = lambda n, dtype: torch.empty(n, dtype=dtype, device="cuda")  # noqa: E731
    s["out"] = {"expert": new((T, k), torch.int32), "weights": new((T, k), torch.float32), "row_of": new((T, k), torch.int32),
                "counts": new(E + 1, torch.int32), "offsets": new(E + 1, torch.int32)}
    if s.train:
        s.out["logit_grad"] = new((T, E), t)
        if s.bias:
            s.out["new_bias"] = new(E, torch.float32)
    s["workspace"] = _bytes((T // 4 + 1024) * (E + 8) * 8)
    return s


def _prepare_gate(s, g):
    t = _TYPE[s.dtype]
    s["h"] = (1.5 * _rand((s.rows, 2 * s.width), g)).to(t)
    s["n"] = n = max(1, int(s.rows * s.used))
    s["rows_used"] = torch.tensor([n], dtype=torch.int32, device="cuda")
    zeros = lambda shape: torch.zeros(shape, dtype=t, device="cuda")  # noqa: E731
    s["out"] = o = {"a": zeros((s.rows, s.width))} if s.scale == "none" else {k: v.zero_() if v.dtype == torch.float32 else v for k, v in _rows8(s.rows, s.width, s.scale).items()}
    for v in o.values():                      # rows that are not there stay as they are
        if v.element_size() == 1:
            v.view(torch.uint8).zero_()
    if s.train:
        s["a_grad"] = _rand((s.rows, s.width), g).to(t)
        o["h_grad"], o["a_again"] = zeros((s.rows, 2 * s.width)), zeros((s.rows, s.width))
    return s


def _prepare_clip(s, g):
    W, F = s.width, s.hidden
    matrices, vectors = [W * W] * 4 * s.layers + [W * F] * 3 * s.layers, [W] * 2 * s.layers + [F] * s.layers
    # each kind's gradients lie in one buffer one behind the other, as a reduction of them wants it
    of = {}
    for name, dtype, counts in (("matrices", s.dtype, matrices), ("vectors", s.vectors, vectors)):
        n = sum(counts)
        flat = torch.empty(n, dtype=_TYPE[dtype], device="cuda")
        size = 3.0 * (1 + torch.rand(1, generator=g, device="cuda")) * (sum(matrices) + sum(vectors)) ** -0.5
        for at in range(0, n, 1 << 27):
            part = flat[at:at + (1 << 27)]
            part.copy_(_rand(part.shape, g) * size)
        of[name] = (flat, torch.empty_like(flat), counts, dtype)
    s["out"] = {"clipped_" + name: v[1] for name, v in of.items()}
    s["flat"] = {name: v[0] for name, v in of.items()}
    s["counts"] = {name: v[2] for name, v in of.items()}
    # from, to, how many, of which type: 32 bytes for each tensor
    table, s["n"] = [], len(matrices) + len(vectors)
    for flat, to, counts, dtype in of.values():
        at = 0
        for n in counts:
            table.append([flat.data_ptr() + at * _SIZE[dtype], to.data_ptr() + at * _SIZE[dtype], n, _CODE[dtype]])
            at += n
    s["table"] = torch.tensor(table, dtype=torch.int64)
    s.out |= {"squares": torch.empty(1, dtype=torch.float64, device="cuda"), "norm": torch.empty(1, device="cuda")}
    s["workspace"] = _bytes(8 * 2048 * (1 + s.n // 16))
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------


def run(state):
    return globals()[("_own_" if own else "_plain_") + state.op](state)


def _types(H):
    return {"fp32": H.HCCL_DATA_TYPE_FP32, "bf16": H.HCCL_DATA_TYPE_BFP16, "fp16": H.HCCL_DATA_TYPE_FP16}


def _scale_types(H):
    return {"none": H.HCCL_AMD_SCALE_NONE, "fp32": H.HCCL_AMD_SCALE_FP32, "e8m0": H.HCCL_AMD_SCALE_E8M0}


def _pointers(o, *names):
    return [o[n].data_ptr() if n in o else None for n in names]


def _quantise(x, scale):
    """32-bit rows of x[rows, width] in blocks of 128: 8-bit values and scales."""
    width = x.shape[-1]
    if width % 128:
        x = torch.nn.functional.pad(x, (0, _up(width) - width))
    x = x.reshape(x.shape[0], -1, 128)
    size = x.abs()
    top = torch.where(torch.isfinite(size), size, 0.0).amax(-1).clamp(min=_LEAST)
    if scale == "fp32":
        back, kept = 1.0 / top * _LARGEST, top * (1.0 / _LARGEST)
    else:
        half, power = torch.frexp(top)                       # top = half * 2^power, half in [1/2, 1)
        power = power - 9 + (half > 0.875).int()             # the least power of two that brings it to 448 or below
        kept = (power + 127).to(torch.uint8).view(_F8_SCALE)
        back = ((127 - power) << 23).to(torch.int32).view(torch.float32)
    return {"q": (x * back.unsqueeze(-1)).to(_F8).reshape(x.shape[0], -1), "scales": kept}


def _plain_norm(s):
    t = _TYPE[s.dtype]
    v = s.x.float() + s.r.float() if s.residual else s.x.float()
    gain = s.gain.float()
    y = v * torch.rsqrt((v * v).mean(1, keepdim=True) + _EPSILON) * gain
    out = {"sum": v.to(t)} if s.residual else {}
    if s.plain:
        out["y"] = y.to(t)
    if s.scale != "none":
        out |= _quantise(y, s.scale)
    if s.train:
        v, dy = (out["sum"] if s.residual else s.x).float(), s.y_grad.float()      # what was kept
        by = torch.rsqrt((v * v).mean(1, keepdim=True) + _EPSILON)
        v = v * by
        dn = dy * gain
        out["x_grad"] = (by * (dn - v * (dn * v).mean(1, keepdim=True)) + s.sum_grad.float()).to(t)
        out["gain_grad"] = (dy * v).sum(0, dtype=torch.float64).float()
    return out


def _own_norm(s):
    H, o = _package(), s.out
    t = _types(H)[s.dtype]
    total, y, q, scales, x_grad, gain_grad = _pointers(o, "sum", "y", "q", "scales", "x_grad", "gain_grad")
    H.norm_rows(s.x.data_ptr(), t, s.rows, s.width, s.stream, residual=s.r.data_ptr() if s.residual else None, gain=s.gain.data_ptr(), gain_dtype=t, epsilon=_EPSILON,
                sum=total, y=y, scale_type=_scale_types(H)[s.scale], q=q, scales=scales)
    if s.train:
        H.norm_rows_grad(s.y_grad.data_ptr(), total if s.residual else s.x.data_ptr(), t, s.rows, s.width, x_grad, s.stream, gain=s.gain.data_ptr(), gain_dtype=t,
                         epsilon=_EPSILON, sum_grad=s.sum_grad.data_ptr(), gain_grad=gain_grad, workspace=s.workspace.data_ptr(), workspace_bytes=s.workspace.numel())
    return o


def _row_of(expert, experts):
    """The row of every choice in expert order; -1 where there is none."""
    flat = torch.where(expert < 0, experts, expert).reshape(-1).long()
    order = torch.sort(flat, stable=True).indices
    row = torch.empty_like(flat)
    row[order] = torch.arange(flat.numel(), device=flat.device)
    return torch.where(flat < experts, row, -1).int().reshape(expert.shape)


def _plain_route(s):
    # in 64 bits: scores next to each other decide whole numbers
    T, E, G, k = s.tokens, s.experts, s.groups, s.topk
    x = s.logits.double()
    can = x > -math.inf
    if s.mask is not None:
        can = can & (s.mask[:, None] != 0)
    if s.score == "sigmoid":
        score = 1 / (1 + torch.exp(-x))
    else:
        e = torch.exp(x - x.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    key = torch.where(can, score + s.b.double() if s.bias else score, -math.inf)
    best = torch.sort(key.reshape(T, G, E // G), dim=2, descending=True).values[:, :, :s.group_top]
    any_left = best[:, :, :1] > -math.inf
    best = torch.where(any_left[:, :, 0], torch.where(best > -math.inf, best, 0.0).sum(2), -math.inf)
    rank = torch.sort(torch.sort(best, dim=1, descending=True, stable=True).indices, dim=1).indices      # equal groups: the lowest first
    key = torch.where((rank < s.kept)[:, :, None], key.reshape(T, G, E // G), -math.inf).reshape(T, E)
    value, expert = torch.sort(key, dim=1, descending=True, stable=True)                                  # equal experts: the lowest first
    value, expert = value[:, :k], expert[:, :k]
    taken = value > -math.inf
    p = torch.where(taken, torch.gather(score, 1, expert), 0.0)
    total = torch.where(taken[:, :1], p.sum(1, keepdim=True), 1.0) if s.renorm else 1.0
    w = 2.5 * p / total
    at = expert
    expert = torch.where(taken, expert, -1).int()
    n = torch.zeros(E + 1, dtype=torch.int64, device="cuda").scatter_add_(0, torch.where(taken, at, E).reshape(-1), torch.ones(1, dtype=torch.int64, device="cuda").expand(T * k))[:E]
    out = {"expert": expert, "weights": w.float(), "row_of": _row_of(expert, E), "counts": torch.cat([n, taken[:, :1].sum().reshape(1)]).int(),
           "offsets": torch.cat([n.new_zeros(1), n.cumsum(0)]).int()}
    if s.train:
        d = torch.where(taken, s.weight_grad.double(), 0.0)
        if s.renorm:
            d = w * (d - (w / 2.5 * d).sum(1, keepdim=True))
        else:
            d = w * d
        if s.score == "sigmoid":
            d = d * (1 - p)
        grad = torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_add_(1, at, d)
        if s.score == "softmax" and not s.renorm:
            grad = grad - torch.where(taken[:, :1], score, 0.0) * d.sum(1, keepdim=True)
        out["logit_grad"] = grad.to(s.logits.dtype)
        if s.bias:
            out["new_bias"] = s.b + _RATE * torch.sign(n.sum() - E * n).float()
    return out


def _own_route(s):
    H, o = _package(), s.out
    P = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    t, score = _types(H)[s.dtype], H.HCCL_AMD_SCORE_SIGMOID if s.score == "sigmoid" else H.HCCL_AMD_SCORE_SOFTMAX
    H.expert_route_scored(P(s.logits), t, s.tokens, s.experts, s.topk, score, P(o["expert"]), P(o["weights"]), P(o["row_of"]), P(o["counts"]), P(o["offsets"]),
                          P(s.workspace), s.workspace.numel(), s.stream, bias=P(s.b), groups=s.groups, groups_kept=s.kept, group_top=s.group_top,
                          renorm=s.renorm, weight_scale=2.5, mask=P(s.mask))
    if s.train:
        H.expert_route_scored_grad(P(s.logits), t, s.tokens, s.experts, s.topk, score, P(o["expert"]), P(s.weight_grad), P(o["logit_grad"]), s.stream,
                                   renorm=s.renorm, weight_scale=2.5)
        if s.bias:
            H.expert_bias(P(o["counts"]), s.experts, _RATE, P(s.b), P(o["new_bias"]), s.stream)
    return o


def _plain_gate(s):
    n, t = s.n, _TYPE[s.dtype]
    g, u = s.h[:n, :s.width].float(), s.h[:n, s.width:].float()
    gate = 1 / (1 + torch.exp(-g))
    a = g * gate * u
    rest = lambda v, like: torch.cat([v, like[n:]]) if n < s.rows else v  # noqa: E731
    if s.scale == "none":
        out = {"a": rest(a.to(t), s.out["a"])}
    else:
        out = {k: rest(v.view(torch.uint8), s.out[k].view(torch.uint8)).view(v.dtype) for k, v in _quantise(a, s.scale).items()}
    if s.train:
        d = s.a_grad[:n].float()
        h_grad = torch.cat([d * u * gate * (1 + g * (1 - gate)), d * g * gate], 1)
        out["h_grad"], out["a_again"] = rest(h_grad.to(t), s.out["h_grad"]), rest(a.to(t), s.out["a_again"])
    return out


def _own_gate(s):
    H, o = _package(), s.out
    t = _types(H)[s.dtype]
    a, q, scales, h_grad, a_again = _pointers(o, "a", "q", "scales", "h_grad", "a_again")
    used = s.rows_used.data_ptr()
    H.expert_gate(s.h.data_ptr(), t, s.rows, s.width, a or q, s.stream, used=used, scale_type=_scale_types(H)[s.scale], scales=scales)
    if s.train:
        H.expert_gate_grad(s.a_grad.data_ptr(), s.h.data_ptr(), t, s.rows, s.width, h_grad, s.stream, used=used, out=a_again)
    return o


def _plain_clip(s):
    squares = torch.stack([part.double().square().sum() for name, flat in s.flat.items() for part in flat.split(s.counts[name])]).sum().reshape(1)
    norm = torch.sqrt(squares)
    by = torch.where(norm > 1.0, 1.0 / norm, 1.0).float()
    clipped = {"clipped_" + name: torch.cat([(part.float() * by).to(flat.dtype) for part in flat.split(s.counts[name])]) for name, flat in s.flat.items()}
    return clipped | {"squares": squares, "norm": norm.float()}


def _own_clip(s):
    H, o = _package(), s.out
    squares, norm = _pointers(o, "squares", "norm")
    H.grad_squares(s.table.data_ptr(), s.n, squares, s.workspace.data_ptr(), s.workspace.numel(), s.stream)
    H.grad_clip(s.table.data_ptr(), s.n, squares, 1.0, norm, s.stream)
    return o


# ---- what it costs, and what it is --------------------------------------------------------------------------------------------


def work(case):
    c = _State(case)
    u = _SIZE[c.dtype]
    eight = lambda W, scale: {"none": 0, "fp32": _up(W) + _up(W) // 32, "e8m0": _up(W) + _up(W) // 128}[scale]  # noqa: E731
    if c.op == "norm":
        n = c.rows * c.width
        b = n * u * (1 + 2 * c.residual + c.plain) + c.rows * eight(c.width, c.scale) + c.width * u
        if c.train:       # y_grad, what was kept and its gradient in, x_grad and gain_grad out
            b += 4 * n * u + c.width * (u + 4)
        return {"bytes": b, "flops": n * (6 + (10 if c.train else 0))}
    if c.op == "route":
        T, E, k = c.tokens, c.experts, c.topk
        b = T * E * u + 12 * T * k + 8 * E + (4 * E if c.bias else 0)
        if c.train:       # only a softmax over all experts needs the logits of those that were not chosen
            b += T * E * u + 8 * T * k + (T * E if c.score == "softmax" and not c.renorm else T * k) * u + (12 * E if c.bias else 0)
        return {"bytes": b, "flops": T * E * (6 + (2 if c.train else 0))}
    if c.op == "gate":
        n = max(1, int(c.rows * c.used))
        b = n * (2 * c.width * u + (c.width * u if c.scale == "none" else eight(c.width, c.scale)))
        if c.train:
            b += n * c.width * u * 6
        return {"bytes": b, "flops": n * c.width * (6 + (14 if c.train else 0))}
    W, F, L, v = c.width, c.hidden, c.layers, _SIZE[c.vectors]
    matrices, vectors = L * (4 * W * W + 3 * W * F), L * (2 * W + F)
    return {"bytes": 3 * (matrices * u + vectors * v), "flops": 3 * (matrices + vectors)}


def exact(case, seed):
    """In 64 bits from the definitions.  Whole numbers have no such value; where the definition rounds what is read again, it is rounded."""
    s = prepare(case, seed)
    return globals()["_exact_" + s.op](s)


def _exact_rows8(y, scale):
    top = torch.nn.functional.pad(y, (0, _up(y.shape[1]) - y.shape[1])).unflatten(1, (-1, 128))
    kept = top.abs().amax(2, keepdim=True).clamp(min=_LEAST)
    kept = kept / _LARGEST if scale == "fp32" else torch.exp2(torch.ceil(torch.log2(kept / _LARGEST)))
    return {"q": (top / kept).float().to(_F8).double().flatten(1), "scales": kept[:, :, 0]}


def _exact_norm(s):
    total = s.x.double()
    if s.residual:
        total = total + s.r.double()
    gain = s.gain.double()
    length = total.square().sum(1).div(s.width).add(_EPSILON).sqrt()
    y = total / length[:, None] * gain
    out = {"sum": total} if s.residual else {}
    if s.plain:
        out["y"] = y
    if s.scale != "none":
        out |= _exact_rows8(y, s.scale)
    if s.train:
        v = total.to(_TYPE[s.dtype]).double()
        del y, total
        length = v.square().sum(1).div(s.width).add(_EPSILON).sqrt()[:, None]
        # d(v / length) = d v / length - v <v, d v> / (width length^3)
        d = s.y_grad.double()
        along = (d * gain * v).sum(1, keepdim=True) / (s.width * length ** 3)
        out["x_grad"] = d * gain / length - v * along + s.sum_grad.double()
        out["gain_grad"] = torch.mv((d * v).T, 1 / length[:, 0])
    return out


def _exact_route(s):
    T, E, G, k = s.tokens, s.experts, s.groups, s.topk
    x = s.logits.double()
    score = torch.sigmoid(x) if s.score == "sigmoid" else torch.softmax(x, 1)
    left = score if s.b is None else score + s.b.double()
    live = torch.ones(T, 1, dtype=torch.bool, device="cuda") if s.mask is None else (s.mask != 0)[:, None]
    first = lambda at_best: (at_best.to(torch.int16) * torch.arange(at_best.shape[1], 0, -1, device="cuda", dtype=torch.int16)).argmax(1)  # noqa: E731
    every = torch.arange(T, device="cuda")
    if G > 1:
        # groups one by one, the lowest of equal ones first
        of = torch.topk(left.view(T, G, -1), min(s.group_top, E // G), dim=2).values.sum(2)
        keep = torch.zeros(T, G, dtype=torch.bool, device="cuda")
        for _ in range(s.kept):
            j = first(of == of.max(1, keepdim=True).values)
            keep[every, j] = True
            of[every, j] = -math.inf
        left = left.masked_fill(~keep.repeat_interleave(E // G, 1), -math.inf)
    else:
        left = left.clone()
    chosen = torch.zeros(T, E, dtype=torch.bool, device="cuda")
    picks = []
    for _ in range(k):
        j = first(left == left.max(1, keepdim=True).values)
        picks.append(j)
        chosen[every, j] = True
        left[every, j] = -math.inf
    pick = torch.stack(picks, 1)
    p = torch.gather(score, 1, pick) * live
    inside = p.sum(1, keepdim=True) if s.renorm else torch.ones(T, 1, dtype=torch.float64, device="cuda")
    inside = torch.where(live, inside, 1.0)
    out = {"expert": None, "weights": 2.5 * p / inside, "row_of": None, "counts": None, "offsets": None}
    if s.train:
        up = s.weight_grad.double() * 2.5 * live                       # gradient of the scores of the chosen
        up = (up - (up * p / inside).sum(1, keepdim=True)) / inside if s.renorm else up
        all_up = torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_(1, pick, up)
        if s.score == "sigmoid":
            out["logit_grad"] = all_up * score * (1 - score)
        else:
            out["logit_grad"] = score * (all_up - (score * all_up).sum(1, keepdim=True))
        if s.bias:
            n = (chosen & live).sum(0).double()
            out["new_bias"] = s.b.double() + _RATE * torch.sign(n.mean() - n)
    return out


def _exact_gate(s):
    n = s.n
    g, u = s.h[:n].double().chunk(2, 1)
    a = torch.nn.functional.silu(g) * u
    whole = lambda v: torch.nn.functional.pad(v, (0, 0, 0, s.rows - n))  # noqa: E731
    out = {"a": whole(a)} if s.scale == "none" else {k: whole(v) for k, v in _exact_rows8(a, s.scale).items()}
    if s.scale == "e8m0" and n < s.rows:
        out["scales"][n:] = 2.0 ** -127                                # what a byte of zero stands for
    if s.train:
        d, sig = s.a_grad[:n].double(), torch.sigmoid(g)
        out["h_grad"] = whole(torch.cat([d * u * (sig + g * sig * torch.sigmoid(-g)), d * g * sig], 1))
        out["a_again"] = whole(a)
    return out


def _exact_clip(s):
    total = torch.zeros(1, dtype=torch.float64, device="cuda")
    for flat in s.flat.values():
        for part in flat.split(1 << 27):
            v = part.double()
            total += torch.dot(v, v)
    norm = total.sqrt()
    return {"clipped_" + name: flat.double() / norm.clamp(min=1.0) for name, flat in s.flat.items()} | {"squares": total, "norm": norm}
