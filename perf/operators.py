"""Timed operators: what an expert-parallel layer does around its all-to-all-v.

A router chooses experts for tokens and counts them (`route`), rows are laid out in expert order, plain or in 8-bit floating
point with a scale per 128 values (`pack`), the experts multiply them by their weights (`product`), and the results come back
to their tokens (`combine`).  Cases with `train` run the gradients too.

Shapes: x[tokens, width], logits[tokens, experts], row_of[tokens, topk] (the row in expert order, -1: none).  8-bit rows are
padded with zeros to a multiple of 128.
"""
import math
import os
import sys

import torch

own = False

_TYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_F8 = torch.float8_e4m3fn
_LEAST = 2.0 ** -96     # the smallest block maximum a scale is made from
_LARGEST = 448.0        # the largest value of the 8-bit type


def _up(n):
    return (n + 127) // 128 * 128


# ---- cases --------------------------------------------------------------------------------------------------------------


def _route(name, tokens, experts, topk, dtype, renorm, masked, train):
    """`masked`: the share of tokens that are padding."""
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "topk": topk, "dtype": dtype, "renorm": renorm,
            "masked": masked, "train": train}


def _pack(name, tokens, width, experts, topk, dtype, scale):
    """`scale`: "none" copies; "fp32" and "e8m0" are the scales' types of 8-bit rows."""
    return {"name": name, "op": "pack", "tokens": tokens, "width": width, "experts": experts, "topk": topk, "dtype": dtype, "scale": scale}


def _combine(name, tokens, width, experts, topk, dtype, train):
    return {"name": name, "op": "combine", "tokens": tokens, "width": width, "experts": experts, "topk": topk, "dtype": dtype, "train": train}


def _product(name, rows, experts, cols, depth, dtype, scale, train):
    """`train`: both gradients, of the rows and of the weights, from 16-bit rows."""
    return {"name": name, "op": "product", "rows": rows, "experts": experts, "cols": cols, "depth": depth, "dtype": dtype, "scale": scale, "train": train}


def listed():
    return [
        # one token of one decoding step
        _route("route_token", 1, 64, 6, "bf16", True, 0.0, False),
        # a training step's ragged batch, an odd number of experts, padded sequences
        _route("route_ragged_train", 5003, 60, 4, "fp32", False, 0.1, True),
        # a large batch over many experts
        _route("route_large_train", 65536, 256, 8, "bf16", True, 0.0, True),
        # 64 decoding tokens of width 8192 (the all-reduce suite's decoding step) on their way to the experts
        _pack("pack_decode", 64, 8192, 64, 8, "bf16", "fp32"),
        # a prompt batch on its way
        _pack("pack_prompt", 16384, 4096, 64, 8, "bf16", "e8m0"),
        # the decoding tokens on their way back
        _combine("combine_decode", 64, 8192, 64, 8, "bf16", False),
        # a training step whose width is no multiple of anything
        _combine("combine_odd_train", 8191, 2001, 60, 4, "fp16", True),
        # a large training batch
        _combine("combine_large_train", 16384, 4096, 64, 8, "bf16", True),
        # one token at its eight experts of 64: their weights are read, little else
        _product("product_token", 8, 64, 4096, 2048, "bf16", "fp32", False),
        # a dense layer over a large batch
        _product("product_dense", 8192, 1, 4096, 8192, "bf16", "e8m0", False),
        # a prompt batch over 64 experts, as unevenly as routers leave it
        _product("product_experts", 32768, 64, 4096, 2048, "bf16", "fp32", False),
        # both gradients of the experts' layer
        _product("product_experts_train", 16411, 16, 2048, 4096, "bf16", "fp32", True),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n if rng.random() < 0.5 else max(1, n // 64) * 64))


def draw(rng):
    op = rng.choice(["route", "pack", "combine", "product", "product"])
    if op == "route":
        experts = rng.choice([8, 16, 60, 64, 127, 128, 256])
        c = _route("", _log(rng, 1, 65536), experts, rng.randint(1, 8), rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.5,
                   rng.choice([0.0, 0.0, 0.1, 0.5]), rng.random() < 0.6)
    elif op in ("pack", "combine"):
        experts = rng.choice([8, 60, 64, 128])
        topk = rng.randint(1, 8)
        width = _log(rng, 64, 8192)
        tokens = _log(rng, 1, max(1, min(65536, (16384 * 4096 * 8) // (width * topk))))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32":
            tokens = max(1, tokens // 2)
        if op == "pack":
            c = _pack("", tokens, width, experts, topk, dtype, rng.choice(["none", "fp32", "fp32", "e8m0"]))
        else:
            c = _combine("", tokens, width, experts, topk, dtype, rng.random() < 0.5)
    else:
        experts = rng.choice([1, 1, 2, 8, 16, 60, 64])
        cols = _log(rng, 64, 8192)
        depth = _log(rng, 64, min(8192, (64 * 4096 * 2048) // (experts * cols)))
        train = rng.random() < 0.35
        most = 2.5e11 / (2.0 * cols * depth * (2 if train else 1))
        c = _product("", _log(rng, 1, max(1, min(65536, int(most)))), experts, cols, depth, rng.choice(["bf16", "bf16", "fp16"]),
                     rng.choice(["fp32", "fp32", "e8m0"]), train)
    del c["name"]
    return c


# ---- what a program has in hand --------------------------------------------------------------------------------------------


def _package():
    root = os.getcwd()
    if root not in sys.path:
        sys.path.insert(0, root)
    from __graft_entry__ import load_package
    return load_package()


def _quantise(x, scale):
    """Rows of x[..., width] in blocks of 128: (8-bit values [..., padded width], scales [..., blocks])."""
    x = x.float()
    width = x.shape[-1]
    if width % 128:
        x = torch.nn.functional.pad(x, (0, _up(width) - width))
    x = x.reshape(*x.shape[:-1], -1, 128)
    size = x.abs()
    top = torch.where(torch.isfinite(size), size, 0.0).amax(-1).clamp(min=_LEAST)
    if scale == "fp32":
        back, kept = _LARGEST / top, top / _LARGEST
    else:
        half, power = torch.frexp(top)                       # top = half * 2^power, half in [1/2, 1)
        power = power - 9 + (half > 0.875).int()             # the least power of two that brings it to 448 or below
        kept = (power + 127).to(torch.uint8)
        back = ((127 - power) << 23).to(torch.int32).view(torch.float32)
    q = (x * back.unsqueeze(-1)).to(_F8)
    return q.reshape(*q.shape[:-2], -1), kept


def _scale_values(scales, real=torch.float32):
    """Scales as numbers: 8-bit ones are powers of two."""
    return torch.exp2(scales.to(real) - 127) if scales.dtype == torch.uint8 else scales.to(real)


def _values(q, scales, real=torch.float32):
    """What 8-bit rows stand for, of the padded width."""
    v = q.to(torch.float32).to(real).reshape(*q.shape[:-1], -1, 128)
    return (v * _scale_values(scales, real).unsqueeze(-1)).reshape(q.shape)


def _rand(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _choices(tokens, experts, topk, g):
    """Distinct experts for every token, some experts liked more than others; some tokens are padding."""
    topk = min(topk, experts)
    liking = _rand((tokens, experts), g) + 0.7 * _rand((experts,), g)
    expert = liking.topk(topk, dim=1).indices.int()
    expert[torch.randperm(tokens, generator=g, device="cuda")[:tokens // 32]] = -1
    return expert


def _row_of(expert, experts):
    """The row of every choice in expert order; -1 where there is none."""
    flat = torch.where(expert < 0, experts, expert).reshape(-1).long()
    order = torch.sort(flat, stable=True).indices
    row = torch.empty_like(flat)
    row[order] = torch.arange(flat.numel(), device=flat.device)
    return torch.where(flat < experts, row, -1).int().reshape(expert.shape)


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


def _prepare_route(s, g):
    T, E, k = s.tokens, s.experts, s.topk
    t = _TYPE[s.dtype]
    s["logits"] = (1.5 * _rand((T, E), g) + 0.5 * _rand((E,), g)).to(t)
    s["mask"] = (torch.rand(T, generator=g, device="cuda") >= s.masked).to(torch.uint8) if s.masked else None
    s["weight_grad"] = _rand((T, k), g)
    s["loss_grad"] = 1.0 + torch.rand(1, generator=g, device="cuda")
    s["out"] = {"expert": torch.empty(T, k, dtype=torch.int32, device="cuda"), "weights": torch.empty(T, k, device="cuda"),
                "row_of": torch.empty(T, k, dtype=torch.int32, device="cuda"),
                "counts": torch.empty(E + 1, dtype=torch.int32, device="cuda"),
                "offsets": torch.empty(E + 1, dtype=torch.int32, device="cuda"), "loss": torch.empty(1, device="cuda")}
    if s.train:
        s.out["logit_grad"] = torch.empty(T, E, dtype=t, device="cuda")
    s["workspace"] = torch.empty((T // 8 + 1024) * (E + 8) * 8, dtype=torch.uint8, device="cuda")
    return s


def _prepare_pack(s, g):
    s["x"] = (_rand((s.tokens, s.width), g) * torch.exp(0.5 * _rand((s.tokens, 1), g))).to(_TYPE[s.dtype])
    s["row_of"] = _row_of(_choices(s.tokens, s.experts, s.topk, g), s.experts)
    s["topk"] = s.row_of.shape[1]
    s["rows"] = R = int((s.row_of >= 0).sum())
    W = _up(s.width)
    if s.scale == "none":
        s["out"] = {"rows": torch.empty(R, s.width, dtype=_TYPE[s.dtype], device="cuda")}
    else:
        s["out"] = {"rows": torch.empty(R, W, dtype=torch.uint8, device="cuda").view(_F8),
                    "scales": torch.empty(R, W // 128, dtype=torch.float32 if s.scale == "fp32" else torch.uint8, device="cuda")}
    return s


def _prepare_combine(s, g):
    t = _TYPE[s.dtype]
    s["row_of"] = _row_of(_choices(s.tokens, s.experts, s.topk, g), s.experts)
    s["topk"] = s.row_of.shape[1]
    s["rows"] = R = int((s.row_of >= 0).sum())
    s["x"] = _rand((R, s.width), g).to(t)
    w = torch.rand(s.row_of.shape, generator=g, device="cuda") + 0.05
    s["weights"] = torch.where(s.row_of < 0, 0.0, w / w.sum(1, keepdim=True)).contiguous()
    s["out"] = {"y": torch.empty(s.tokens, s.width, dtype=t, device="cuda")}
    if s.train:
        s["y_grad"] = _rand((s.tokens, s.width), g).to(t)
        s.out["x_grad"] = torch.empty(R, s.width, dtype=t, device="cuda")
        s.out["weight_grad"] = torch.empty(s.row_of.shape, device="cuda")
        # the gradient of the rows that went to the experts, and where it adds up: the tokens
        s["sent_grad"] = _rand((R, s.width), g).to(t)
        s.out["token_grad"] = torch.empty(s.tokens, s.width, dtype=t, device="cuda")
    return s


def _prepare_product(s, g):
    R, E, N, K = s.rows, s.experts, s.cols, s.depth
    t = _TYPE[s.dtype]
    # how many rows each expert has: some are liked several times as much as others, and of few rows most have none
    taken = torch.multinomial(torch.exp(0.5 * _rand((E,), g)), R, replacement=True, generator=g)
    counts = torch.bincount(taken, minlength=E)
    s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    host = counts.tolist()                                   # a program knows them: its all-to-all-v takes them
    hit = [e for e in range(E) if host[e]]
    s["hit"] = torch.tensor(hit, device="cuda")
    # the plain form multiplies expert by expert, all padded to the longest
    s["longest"] = longest = max(host)
    at = torch.arange(longest, device="cuda")
    s["place"] = torch.where(at < counts[s.hit][:, None], s.offsets[:-1].long()[s.hit][:, None] + at, R)
    weights = torch.randn((E, N, K), generator=g, device="cuda", dtype=torch.bfloat16 if E * N * K > (1 << 26) else torch.float32) * K ** -0.5
    blocks = torch.nn.functional.pad(weights, (0, _up(K) - K, 0, _up(N) - N)).reshape(E, _up(N) // 128, 128, _up(K) // 128, 128)
    blocks = blocks.permute(0, 1, 3, 2, 4).reshape(E, _up(N) // 128, _up(K) // 128, 128 * 128)
    top = blocks.abs().amax(-1).float().clamp(min=_LEAST)
    if s.scale == "fp32":
        scales = top / _LARGEST
    else:
        half, power = torch.frexp(top)
        scales = (power - 9 + (half > 0.875).int() + 127).to(torch.uint8)
    q = (blocks.float() / _scale_values(scales).unsqueeze(-1)).to(_F8)
    del blocks, weights
    q = q.reshape(E, _up(N) // 128, _up(K) // 128, 128, 128).permute(0, 1, 3, 2, 4).reshape(E, _up(N), _up(K))
    if not s.train:
        s["w"], s["w_scales"] = q[:, :N].contiguous(), scales
        s["x"], s["x_scales"] = _quantise(_rand((R, K), g), s.scale)
        s["out"] = {"y": torch.empty(R, N, dtype=t, device="cuda")}
        return s
    s["wt"], s["wt_scales"] = q.transpose(1, 2)[:, :K].contiguous(), scales.transpose(1, 2).contiguous()
    s["x"] = _rand((R, K), g).to(t)
    s["y_grad"] = (_rand((R, N), g) * 0.01).to(t)
    kept = torch.float32 if s.scale == "fp32" else torch.uint8
    s["yq"] = torch.empty(R, _up(N), dtype=torch.uint8, device="cuda")
    s["yq_scales"] = torch.empty(R, _up(N) // 128, dtype=kept, device="cuda")
    long = (R // 128 + E) * 128                              # every expert's rows padded to a multiple of 128
    for name, n in (("yt", N), ("xt", K)):
        s[name] = torch.empty(n, long, dtype=torch.uint8, device="cuda")
        s[name + "_scales"] = torch.empty(long // 128, n, dtype=kept, device="cuda")
    s["long"] = long
    s["out"] = {"x_grad": torch.empty(R, K, dtype=t, device="cuda"), "w_grad": torch.empty(E, N, K, device="cuda")}
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------


def run(state):
    return globals()[("_own_" if own else "_plain_") + state.op](state)


def _plain_route(s, real=torch.float32):
    T, E, k = s.tokens, s.experts, s.topk
    x = s.logits.to(real)
    key = torch.where(torch.isnan(x), -math.inf, x)
    if s.mask is not None:
        key = torch.where(s.mask[:, None] != 0, key, -math.inf)
    value, expert = torch.sort(key, dim=1, descending=True, stable=True)      # equal logits: the lowest expert first
    value, expert = value[:, :k], expert[:, :k]
    taken = value > -math.inf
    routed = taken[:, :1]
    e = torch.where(routed, torch.exp(x - torch.where(routed, value[:, :1], 0.0)), 0.0)
    p = e / torch.where(routed, e.sum(1, keepdim=True), 1.0)
    w = torch.where(taken, torch.gather(p, 1, expert), 0.0)
    if s.renorm:
        ew = torch.where(taken, torch.gather(e, 1, expert), 0.0)
        w = ew / torch.where(routed, ew.sum(1, keepdim=True), 1.0)
    expert = torch.where(taken, expert, -1).int()
    n = torch.zeros(E + 1, dtype=torch.int64, device="cuda").scatter_add_(0, torch.where(taken, expert, E).reshape(-1).long(), torch.ones(1, dtype=torch.int64, device="cuda").expand(T * k))[:E]
    rows, total = routed.sum(), n.sum()
    load = E * n.to(real) / (total.clamp(min=1) * rows.clamp(min=1)).to(real)
    loss = 0.01 * (load * p.sum(0)).sum().reshape(1)
    out = {"expert": expert, "weights": w, "row_of": _row_of(expert, E), "counts": torch.cat([n, rows.reshape(1)]).int(),
           "offsets": torch.cat([n.new_zeros(1), n.cumsum(0)]).int(), "loss": loss}
    if s.train:
        g = (0.01 * s.loss_grad.to(real) * load).expand(T, E)
        dw = torch.where(taken, s.weight_grad.to(real), 0.0)
        at = torch.where(taken, expert, 0).long()
        if not s.renorm:
            g = g.scatter_add(1, at, dw)
        d = p * (g - (p * g).sum(1, keepdim=True))
        if s.renorm:
            d = d.scatter_add(1, at, w * (dw - (w * dw).sum(1, keepdim=True)))
        out["logit_grad"] = d.to(s.logits.dtype) if real == torch.float32 else d
    return out


def _own_route(s):
    H, o = _package(), s.out
    P = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    t = {"fp32": H.HCCL_DATA_TYPE_FP32, "bf16": H.HCCL_DATA_TYPE_BFP16, "fp16": H.HCCL_DATA_TYPE_FP16}[s.dtype]
    H.expert_route(P(s.logits), t, s.tokens, s.experts, s.topk, P(o["expert"]), P(o["weights"]), P(o["row_of"]), P(o["counts"]), P(o["offsets"]),
                   P(o["loss"]), P(s.workspace), s.workspace.numel(), s.stream, renorm=s.renorm, mask=P(s.mask), loss_scale=0.01)
    if s.train:
        H.expert_route_grad(P(s.logits), t, s.tokens, s.experts, s.topk, P(o["expert"]), P(o["counts"]), P(s.weight_grad), P(s.loss_grad),
                            P(o["logit_grad"]), s.stream, renorm=s.renorm, mask=P(s.mask), loss_scale=0.01)
    return o


def _plain_pack(s):
    taken = s.row_of >= 0
    token = torch.arange(s.tokens, device="cuda")[:, None].expand(taken.shape)[taken]
    to = s.row_of[taken].long()
    source = torch.empty_like(token)
    source[to] = token
    if s.scale == "none":
        return {"rows": s.x[source]}
    q, kept = _quantise(s.x, s.scale)
    return {"rows": q.view(torch.uint8)[source].view(_F8), "scales": kept[source]}


def _types(H):
    return {"fp32": H.HCCL_DATA_TYPE_FP32, "bf16": H.HCCL_DATA_TYPE_BFP16, "fp16": H.HCCL_DATA_TYPE_FP16}


def _scale_types(H):
    return {"fp32": H.HCCL_AMD_SCALE_FP32, "e8m0": H.HCCL_AMD_SCALE_E8M0}


def _own_pack(s):
    H, o = _package(), s.out
    t = _types(H)[s.dtype]
    if s.scale == "none":
        H.expert_pack(s.x.data_ptr(), t, s.tokens, s.width, s.topk, s.row_of.data_ptr(), o["rows"].data_ptr(), s.rows, s.stream)
    else:
        H.expert_pack(s.x.data_ptr(), t, s.tokens, s.width, s.topk, s.row_of.data_ptr(), o["rows"].data_ptr(), s.rows, s.stream,
                      scales=o["scales"].data_ptr(), scale_type=_scale_types(H)[s.scale])
    return o


def _plain_combine(s, real=torch.float32):
    def rounded(v):
        return v.to(_TYPE[s.dtype]) if real == torch.float32 else v

    taken = s.row_of >= 0
    at = s.row_of.clamp(min=0).long()
    w = torch.where(taken, s.weights, 0.0).to(real)
    none = not s.rows                                        # no row at all: nothing to index
    x = s.x.new_zeros(*at.shape, s.width).to(real) if none else s.x[at].to(real)
    out = {"y": rounded((x * w[..., None]).sum(1))}
    if s.train:
        d = s.y_grad.to(real)
        out["weight_grad"] = torch.where(taken, (x * d[:, None]).sum(-1), 0.0)
        grad = torch.empty(s.rows, s.width, dtype=real, device="cuda")
        grad[at[taken]] = (w[..., None] * d[:, None])[taken]
        out["x_grad"] = rounded(grad)
        sent = s.x.new_zeros(*at.shape, s.width).to(real) if none else s.sent_grad[at].to(real)
        out["token_grad"] = rounded(torch.where(taken[..., None], sent, 0.0).sum(1))
    return out


def _own_combine(s):
    H, o = _package(), s.out
    t = _types(H)[s.dtype]
    H.expert_combine(s.x.data_ptr(), t, s.rows, s.width, s.tokens, s.topk, s.row_of.data_ptr(), s.weights.data_ptr(), o["y"].data_ptr(), s.stream)
    if s.train:
        H.expert_combine_grad(s.y_grad.data_ptr(), s.x.data_ptr(), t, s.rows, s.width, s.tokens, s.topk, s.row_of.data_ptr(), s.weights.data_ptr(),
                              o["x_grad"].data_ptr(), o["weight_grad"].data_ptr(), s.stream)
        # the rows' gradient of the way to the experts: every token adds up its rows
        H.expert_combine(s.sent_grad.data_ptr(), t, s.rows, s.width, s.tokens, s.topk, s.row_of.data_ptr(), None, o["token_grad"].data_ptr(), s.stream)
    return o


def _by_expert(v, s):
    """Rows of v as [experts that have any, longest, ...], zeros behind an expert's last one."""
    return torch.cat([v, v.new_zeros(1, *v.shape[1:])])[s.place]


def _from_experts(v, s):
    out = torch.empty(s.rows + 1, v.shape[-1], dtype=v.dtype, device=v.device)
    out[s.place.reshape(-1)] = v.reshape(-1, v.shape[-1])
    return out[:s.rows]


def _weight_values(q, scales, real=torch.float32):
    """Weights [experts, n, padded k] with one scale for 128 x 128."""
    n = q.shape[1]
    return _values(q, scales.repeat_interleave(128, 1)[:, :n], real)


def _plain_product(s, real=torch.float32):
    def rounded(v):
        return v.to(_TYPE[s.dtype]) if real == torch.float32 else v

    if not s.train:
        w = _weight_values(s.w.view(torch.uint8)[s.hit].view(_F8), s.w_scales[s.hit], real)
        x = _by_expert(_values(s.x, s.x_scales, real), s)
        return {"y": rounded(_from_experts(torch.matmul(x, w.transpose(1, 2).contiguous()), s))}
    # gradient of the rows: 8-bit gradients by the transposed weights
    wt = _weight_values(s.wt.view(torch.uint8)[s.hit].view(_F8), s.wt_scales[s.hit], real)
    d = _by_expert(_values(*_quantise(s.y_grad, s.scale), real), s)
    x_grad = _from_experts(torch.matmul(d, wt.transpose(1, 2).contiguous()), s)
    del wt, d
    # gradient of the weights: both sides 8-bit in blocks of 128 of an expert's rows
    at, bt = (_values(*_quantise(_by_expert(v, s).transpose(1, 2), s.scale), real) for v in (s.y_grad, s.x))
    w_grad = torch.zeros(s.experts, s.cols, s.depth, dtype=real, device="cuda")
    w_grad[s.hit] = torch.matmul(at, bt.transpose(1, 2).contiguous())
    return {"x_grad": rounded(x_grad), "w_grad": w_grad}


def _own_product(s):
    H, o = _package(), s.out
    t, st = _types(H)[s.dtype], _scale_types(H)[s.scale]
    P = lambda name: s[name].data_ptr()  # noqa: E731
    R, E, N, K = s.rows, s.experts, s.cols, s.depth
    if not s.train:
        H.block_matmul(P("x"), P("x_scales"), R, P("w"), P("w_scales"), E, N, K, st, o["y"].data_ptr(), t, s.stream, groups=E, offsets=P("offsets"))
        return o
    H.expert_pack(P("y_grad"), t, R, N, 1, None, P("yq"), R, s.stream, scales=P("yq_scales"), scale_type=st)
    H.block_matmul(P("yq"), P("yq_scales"), R, P("wt"), P("wt_scales"), E, K, N, st, o["x_grad"].data_ptr(), t, s.stream, groups=E, offsets=P("offsets"))
    H.block_quant_columns(P("y_grad"), t, R, N, E, P("offsets"), st, P("yt"), s.long, P("yt_scales"), s.stream)
    H.block_quant_columns(P("x"), t, R, K, E, P("offsets"), st, P("xt"), s.long, P("xt_scales"), s.stream)
    H.block_matmul_grad_weight(P("yt"), P("yt_scales"), P("xt"), P("xt_scales"), s.long, R, N, K, st, E, P("offsets"), E, o["w_grad"].data_ptr(),
                               H.HCCL_DATA_TYPE_FP32, s.stream)
    return o


# ---- what it costs, and what it is --------------------------------------------------------------------------------------------


def work(case):
    c = _State(case)
    if c.op == "route":
        T, E, k, u = c.tokens, c.experts, c.topk, _SIZE[c.dtype]
        b = T * E * u + 12 * T * k + 8 * E + 12
        f = 5 * T * E
        return {"bytes": b + (2 * T * E * u + 8 * T * k if c.train else 0), "flops": f * (2 if c.train else 1)}
    if c.op in ("pack", "combine"):
        T, W, u = c.tokens, c.width, _SIZE[c.dtype]
        rows = T * min(c.topk, c.experts)
        if c.op == "pack":
            blocks = _up(W) // 128
            out = {"none": W * u, "fp32": _up(W) + 4 * blocks, "e8m0": _up(W) + blocks}[c.scale]
            return {"bytes": T * W * u + rows * (out + 4), "flops": 3 * T * W if c.scale != "none" else 0}
        b = (rows * W + T * W) * u + 8 * rows
        f = 2 * rows * W
        if c.train:     # y_grad and x in, x_grad and weight_grad out; sent_grad in, token_grad out
            b += (T * W + 2 * rows * W) * u + 12 * rows + (rows * W + T * W) * u + 4 * rows
            f += 4 * rows * W
        return {"bytes": b, "flops": f}
    R, E, N, K, u = c.rows, c.experts, c.cols, c.depth, _SIZE[c.dtype]
    hit = E * (1 - (1 - 1 / E) ** R)        # how many experts R rows reach
    if not c.train:
        return {"bytes": R * K + hit * N * K + R * N * u, "flops": 2 * R * N * K}
    return {"bytes": R * (N + K) * u + hit * N * K + R * K * u + 4 * E * N * K, "flops": 4 * R * N * K}


def exact(case, seed):
    """In 64 bits from the definitions.  Choices, counts and rows are whole numbers; rounded 8-bit values are kept where the definition rounds."""
    s = prepare(case, seed)
    return globals()["_exact_" + s.op](s)


def _exact_route(s):
    T, E, k = s.tokens, s.experts, s.topk
    x = s.logits.double()
    live = torch.ones(T, dtype=torch.bool, device="cuda") if s.mask is None else s.mask != 0
    # the j-th choice is the largest logit not chosen yet; of equal ones argmax of the mirrored row names the lowest expert
    left = x.clone()
    chosen = torch.zeros(T, E, dtype=torch.bool, device="cuda")
    picks = []
    for _ in range(k):
        best = left.max(1, keepdim=True).values
        first = ((left == best).to(torch.int8) * torch.arange(E, 0, -1, device="cuda")).argmax(1)
        picks.append(first)
        left[torch.arange(T, device="cuda"), first] = -math.inf
        chosen[torch.arange(T, device="cuda"), first] = True
    pick = torch.stack(picks, 1)
    p = torch.exp(x - torch.logsumexp(x, 1, keepdim=True)) * live[:, None]
    chosen &= live[:, None]
    w = torch.gather(p, 1, pick)
    inside = w.sum(1, keepdim=True)
    if s.renorm:
        w = torch.where(live[:, None], w / inside, 0.0)
    n, rows = chosen.sum(0).double(), max(1, int(live.sum()))
    total = max(1.0, float(n.sum()))
    out = {"expert": None, "weights": w, "row_of": None, "counts": None, "offsets": None, "loss": (0.01 * E / total / rows * (n @ p.sum(0))).reshape(1)}
    if s.train:
        up = torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_(1, pick, s.weight_grad.double())
        if s.renorm:   # through the quotient p_j / (sum of the chosen p)
            share = torch.where(live[:, None], p / torch.where(inside > 0, inside, 1.0), 0.0)
            up = torch.where(chosen, up / torch.where(inside > 0, inside, 1.0) - (up * share * chosen).sum(1, keepdim=True) / torch.where(inside > 0, inside, 1.0), 0.0)
        up = up * live[:, None] + 0.01 * float(s.loss_grad) * E / total / rows * n
        out["logit_grad"] = p * up - p * (p * up).sum(1, keepdim=True)
    return out


def _exact_pack(s):
    if s.scale == "none":
        return None
    at = torch.full((s.rows,), -1, dtype=torch.long, device="cuda")
    for j in range(s.topk):
        taken = s.row_of[:, j] >= 0
        at[s.row_of[taken, j].long()] = torch.nonzero(taken)[:, 0]
    W = _up(s.width)
    rows, kept = torch.zeros(s.rows, W, device="cuda", dtype=torch.float64), []
    for b in range(W // 128):
        v = s.x[:, 128 * b:128 * b + 128].double()
        top = v.abs().amax(1).clamp(min=_LEAST)
        scale = top / _LARGEST if s.scale == "fp32" else torch.exp2(torch.ceil(torch.log2(top / _LARGEST)))
        q = (v / scale[:, None]).float().to(_F8).double()
        rows[:, 128 * b:128 * b + v.shape[1]] = q[at]
        kept.append(scale[at])
    return {"rows": rows, "scales": torch.stack(kept, 1) if s.scale == "fp32" else None}


def _exact_combine(s):
    T, W = s.tokens, s.width
    y = torch.zeros(T, W, dtype=torch.float64, device="cuda")
    out = {"y": y}
    if s.train:
        out |= {"x_grad": torch.zeros(s.rows, W, dtype=torch.float64, device="cuda"), "weight_grad": torch.zeros(T, s.topk, dtype=torch.float64, device="cuda"),
                "token_grad": torch.zeros_like(y)}
    for j in range(s.topk):
        t = torch.nonzero(s.row_of[:, j] >= 0)[:, 0]
        r = s.row_of[t, j].long()
        w = s.weights[t, j].double()[:, None]
        y[t] += w * s.x[r].double()
        if s.train:
            d = s.y_grad[t].double()
            out["x_grad"][r] = w * d
            out["weight_grad"][t, j] = (d * s.x[r].double()).sum(1)
            out["token_grad"][t] += s.sent_grad[r].double()
    return out


def _exact_product(s):
    offsets = s.offsets.tolist()
    N, K = s.cols, s.depth

    def expand(q, scales):
        """128 x 128 blocks: every value times its block's scale."""
        v, f = q.float().double(), _scale_values(scales, torch.float64)
        i = torch.arange(v.shape[0], device="cuda") // 128
        j = torch.arange(v.shape[1], device="cuda") // 128
        return v * f[i][:, j]

    def rounded(v):
        """8-bit values in blocks of 128 along a row, as numbers."""
        n = v.shape[1]
        v = torch.nn.functional.pad(v.double(), (0, _up(n) - n)).reshape(v.shape[0], -1, 128)
        top = v.abs().amax(2, keepdim=True).clamp(min=_LEAST)
        f = top / _LARGEST if s.scale == "fp32" else torch.exp2(torch.ceil(torch.log2(top / _LARGEST)))
        return ((v / f).float().to(_F8).double() * f).reshape(v.shape[0], -1)[:, :n]

    if not s.train:
        y = torch.zeros(s.rows, N, dtype=torch.float64, device="cuda")
        f = _scale_values(s.x_scales, torch.float64).repeat_interleave(128, 1)
        x = s.x.float().double() * f
        for e in range(s.experts):
            lo, hi = offsets[e], offsets[e + 1]
            if hi > lo:
                y[lo:hi] = x[lo:hi] @ expand(s.w[e], s.w_scales[e]).T
        return {"y": y}
    x_grad = torch.zeros(s.rows, K, dtype=torch.float64, device="cuda")
    w_grad = torch.zeros(s.experts, N, K, dtype=torch.float64, device="cuda")
    d = rounded(s.y_grad)
    for e in range(s.experts):
        lo, hi = offsets[e], offsets[e + 1]
        if hi > lo:
            x_grad[lo:hi] = d[lo:hi] @ expand(s.wt[e], s.wt_scales[e])[:, :N].T
            w_grad[e] = rounded(s.y_grad[lo:hi].T) @ rounded(s.x[lo:hi].T).T
    return {"x_grad": x_grad, "w_grad": w_grad}
