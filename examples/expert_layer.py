"""An expert-parallel layer over the ranks of one communicator: its forward pass, its gradients, one step of them.

    python examples/expert_layer.py [--ranks 8] [--experts 16] [--tokens 2048] [--width 1024] [--hidden 2048] [--topk 4]

Every rank holds tokens and experts / ranks of the experts.  The router chooses topk experts for every token; the tokens go
to them in 8 bits with a scale per 128 values (HcclAlltoAllV of the rows and of their scales), the experts multiply the
receive buffer as it lies -- source rank by source rank, each with all local experts -- and the results go back in 16 bits and are
weighted and summed.  All ranks are driven from one thread on one stream, as everywhere in this library.
"""
import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
from __graft_entry__ import load_package  # noqa: E402

H = load_package()
BF16 = torch.bfloat16


def _new(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="cuda")


class ExpertLayer:
    """y = sum over a token's experts of weight * W2 silu(W1 x), W1[hidden, width] and W2[width, hidden] of every expert."""

    def __init__(self, ranks, experts, width, hidden, topk, w_router, w1, w2, loss_scale=0.01):
        """w_router[experts, width]; w1[experts, hidden, width], w2[experts, width, hidden]: 16-bit masters."""
        assert experts % ranks == 0
        self.p, self.E, self.mine, self.W, self.F, self.k = ranks, experts, experts // ranks, width, hidden, topk
        self.w_router, self.loss_scale = w_router, loss_scale
        self.comms = H.comm_init_all(ranks)
        self.stream = torch.cuda.Stream()
        # which weights a group of the receive buffer uses: (source rank, local expert), expert varying fastest
        self.owner = torch.arange(self.mine, dtype=torch.int32, device="cuda").repeat(ranks)
        self.ranks = [dict(w1=w1[r * self.mine:(r + 1) * self.mine].contiguous(), w2=w2[r * self.mine:(r + 1) * self.mine].contiguous())
                      for r in range(ranks)]
        torch.cuda.synchronize()
        for s in self.ranks:
            for name, n, k in (("w1", hidden, width), ("w2", width, hidden)):
                kp, np_ = -(-k // 128) * 128, -(-n // 128) * 128
                s[name + "_q"], s[name + "_s"] = _new(self.mine, n, kp, dtype=torch.uint8), _new(self.mine, np_ // 128, kp // 128, dtype=torch.float32)
                s[name + "_qt"], s[name + "_st"] = _new(self.mine, k, np_, dtype=torch.uint8), _new(self.mine, kp // 128, np_ // 128, dtype=torch.float32)
                H.block_quant_weights(s[name].data_ptr(), H.HCCL_DATA_TYPE_BFP16, self.mine, n, k, H.HCCL_AMD_SCALE_FP32, s[name + "_q"].data_ptr(),
                                      s[name + "_s"].data_ptr(), s[name + "_qt"].data_ptr(), s[name + "_st"].data_ptr(), self.stream.cuda_stream)
        self.stream.synchronize()

    def close(self):
        torch.cuda.synchronize()
        H.comm_destroy(self.comms)

    # ---- the pieces, per rank ---------------------------------------------------------------------------------------------

    def _exchange(self, sends, rows, width, dtype):
        """All-to-all-v of rows of `width` elements; rows[i][j]: from rank i to rank j.  Returns the receive buffers."""
        p = self.p
        code = {torch.uint8: H.HCCL_DATA_TYPE_UINT8, torch.float32: H.HCCL_DATA_TYPE_FP32, BF16: H.HCCL_DATA_TYPE_BFP16}[dtype]
        before = lambda v: [sum(v[:i]) * width for i in range(p)]  # noqa: E731
        into = [[rows[i][j] for i in range(p)] for j in range(p)]
        recvs = [_new(max(1, sum(into[j])), width, dtype=dtype) for j in range(p)]
        H.all_to_all_v(self.comms, [s.data_ptr() for s in sends], [[n * width for n in row] for row in rows], [before(row) for row in rows],
                       [t.data_ptr() for t in recvs], [[n * width for n in row] for row in into], [before(row) for row in into], code,
                       self.stream.cuda_stream)
        return recvs

    def _quantise(self, x):
        q, s = _new(x.shape[0], -(-x.shape[1] // 128) * 128, dtype=torch.uint8), _new(x.shape[0], -(-x.shape[1] // 128), dtype=torch.float32)
        H.expert_pack(x.data_ptr(), H.HCCL_DATA_TYPE_BFP16, x.shape[0], x.shape[1], 1, None, q.data_ptr(), x.shape[0], self.stream.cuda_stream,
                      scales=s.data_ptr(), scale_type=H.HCCL_AMD_SCALE_FP32)
        return q, s

    def _multiply(self, s, q, scales, w, w_scales, n, k):
        y = _new(q.shape[0], n)
        H.block_matmul(q.data_ptr(), scales.data_ptr(), s["rows"], w.data_ptr(), w_scales.data_ptr(), self.mine, n, k, H.HCCL_AMD_SCALE_FP32,
                       y.data_ptr(), H.HCCL_DATA_TYPE_BFP16, self.stream.cuda_stream, groups=self.p * self.mine, offsets=s["groups"].data_ptr(),
                       expert_of_group=self.owner.data_ptr())
        return y

    def _weight_gradient(self, s, dy, x):
        """Sum over each local expert's rows of dy^T x."""
        groups, rows, S = self.p * self.mine, s["rows"], self.stream.cuda_stream
        columns = H.block_columns(rows, groups)
        q, sc = [], []
        for v in (dy, x):
            q.append(_new(v.shape[1], columns, dtype=torch.uint8))
            sc.append(_new(columns // 128, v.shape[1], dtype=torch.float32))
            H.block_quant_columns(v.data_ptr(), H.HCCL_DATA_TYPE_BFP16, rows, v.shape[1], groups, s["groups"].data_ptr(), H.HCCL_AMD_SCALE_FP32,
                                  q[-1].data_ptr(), columns, sc[-1].data_ptr(), S)
        grad = _new(self.mine, dy.shape[1], x.shape[1], dtype=torch.float32)
        H.block_matmul_grad_weight(q[0].data_ptr(), sc[0].data_ptr(), q[1].data_ptr(), sc[1].data_ptr(), columns, rows, dy.shape[1], x.shape[1],
                                   H.HCCL_AMD_SCALE_FP32, groups, s["groups"].data_ptr(), self.mine, grad.data_ptr(), H.HCCL_DATA_TYPE_FP32, S,
                                   expert_of_group=self.owner.data_ptr())
        return grad

    # ---- the layer ------------------------------------------------------------------------------------------------------------

    def forward(self, xs):
        """xs: the ranks' tokens [tokens, width].  Returns their outputs and balance losses; keeps what backward needs."""
        with torch.cuda.stream(self.stream):
            S, p, E, k = self.stream.cuda_stream, self.p, self.E, self.k
            for s, x in zip(self.ranks, xs):
                T = x.shape[0]
                s["x"], s["logits"] = x, (x @ self.w_router.t()).float()
                s["expert"], s["row_of"] = _new(T, k, dtype=torch.int32), _new(T, k, dtype=torch.int32)
                s["weights"], s["loss"] = _new(T, k, dtype=torch.float32), _new(1, dtype=torch.float32)
                s["counts"], s["offsets"] = _new(E + 1, dtype=torch.int32), _new(E + 1, dtype=torch.int32)
                need = H.expert_route_workspace(T, E)
                work = _new(max(16, need), dtype=torch.uint8)
                H.expert_route(s["logits"].data_ptr(), H.HCCL_DATA_TYPE_FP32, T, E, k, s["expert"].data_ptr(), s["weights"].data_ptr(),
                               s["row_of"].data_ptr(), s["counts"].data_ptr(), s["offsets"].data_ptr(), s["loss"].data_ptr(), work.data_ptr(), need, S,
                               renorm=True, loss_scale=self.loss_scale)
                wp = -(-self.W // 128) * 128
                s["q"], s["q_s"] = _new(T * k, wp, dtype=torch.uint8), _new(T * k, wp // 128, dtype=torch.float32)
                H.expert_pack(x.data_ptr(), H.HCCL_DATA_TYPE_BFP16, T, self.W, k, s["row_of"].data_ptr(), s["q"].data_ptr(), T * k, S,
                              scales=s["q_s"].data_ptr(), scale_type=H.HCCL_AMD_SCALE_FP32)
            # the all-to-all-v's tables are on the host: the counts come there, and with them the groups of every receive buffer
            counts = [s["counts"][:E].tolist() for s in self.ranks]
            self.rows = [[sum(c[j * self.mine:(j + 1) * self.mine]) for j in range(p)] for c in counts]
            for j, s in enumerate(self.ranks):
                sizes = [counts[i][j * self.mine + e] for i in range(p) for e in range(self.mine)]
                s["rows"] = sum(sizes)
                s["groups"] = torch.tensor([0] + sizes, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
            qs = self._exchange([s["q"] for s in self.ranks], self.rows, self.ranks[0]["q"].shape[1], torch.uint8)
            scales = self._exchange([s["q_s"] for s in self.ranks], self.rows, self.ranks[0]["q_s"].shape[1], torch.float32)
            for s, q, q_s in zip(self.ranks, qs, scales):
                s["xq"], s["xq_s"] = q, q_s
                s["h"] = self._multiply(s, q, q_s, s["w1_q"], s["w1_s"], self.F, self.W)
                s["a"] = torch.nn.functional.silu(s["h"])
                s["out"] = self._multiply(s, *self._quantise(s["a"]), s["w2_q"], s["w2_s"], self.W, self.F)
            back = self._exchange([s["out"] for s in self.ranks], [list(c) for c in zip(*self.rows)], self.W, BF16)
            ys = []
            for s, rows in zip(self.ranks, back):
                T = s["x"].shape[0]
                s["back"], y = rows, _new(T, self.W)
                H.expert_combine(rows.data_ptr(), H.HCCL_DATA_TYPE_BFP16, T * k, self.W, T, k, s["row_of"].data_ptr(), s["weights"].data_ptr(),
                                 y.data_ptr(), S)
                ys.append(y)
            return ys, [s["loss"] for s in self.ranks]

    def backward(self, dys, dloss=1.0):
        """Gradients of the tokens (the router's path through x included), the router's and the experts' weights."""
        with torch.cuda.stream(self.stream):
            S, E, k = self.stream.cuda_stream, self.E, self.k
            one = torch.full((1,), dloss, device="cuda")
            sent = []
            for s, dy in zip(self.ranks, dys):
                T = dy.shape[0]
                s["d_weights"] = _new(T, k, dtype=torch.float32)
                sent.append(_new(T * k, self.W))
                H.expert_combine_grad(dy.data_ptr(), s["back"].data_ptr(), H.HCCL_DATA_TYPE_BFP16, T * k, self.W, T, k, s["row_of"].data_ptr(),
                                      s["weights"].data_ptr(), sent[-1].data_ptr(), s["d_weights"].data_ptr(), S)
            d_out = self._exchange(sent, self.rows, self.W, BF16)
            d_rows = []
            for s, d in zip(self.ranks, d_out):
                s["d_w2"] = self._weight_gradient(s, d, s["a"])
                da = self._multiply(s, *self._quantise(d), s["w2_qt"], s["w2_st"], self.F, self.W)
                gate = torch.sigmoid(s["h"].float())
                dh = (da.float() * gate * (1 + s["h"].float() * (1 - gate))).to(BF16)
                x = (s["xq"].view(torch.float8_e4m3fn).float().reshape(*s["xq_s"].shape, 128) * s["xq_s"][..., None]).reshape(s["xq"].shape)
                s["d_w1"] = self._weight_gradient(s, dh, x[:, :self.W].to(BF16).contiguous())
                d_rows.append(self._multiply(s, *self._quantise(dh), s["w1_qt"], s["w1_st"], self.W, self.F))
            back = self._exchange(d_rows, [list(c) for c in zip(*self.rows)], self.W, BF16)
            dxs, d_router = [], 0
            for s, rows in zip(self.ranks, back):
                T = s["x"].shape[0]
                dx, d_logits = _new(T, self.W), _new(T, E, dtype=torch.float32)
                H.expert_combine(rows.data_ptr(), H.HCCL_DATA_TYPE_BFP16, T * k, self.W, T, k, s["row_of"].data_ptr(), None, dx.data_ptr(), S)
                H.expert_route_grad(s["logits"].data_ptr(), H.HCCL_DATA_TYPE_FP32, T, E, k, s["expert"].data_ptr(), s["counts"].data_ptr(),
                                    s["d_weights"].data_ptr(), one.data_ptr(), d_logits.data_ptr(), S, renorm=True, loss_scale=self.loss_scale)
                dxs.append((dx.float() + d_logits @ self.w_router.float()).to(BF16))
                d_router = d_router + d_logits.t() @ s["x"].float()
            return dxs, d_router, torch.cat([s["d_w1"] for s in self.ranks]), torch.cat([s["d_w2"] for s in self.ranks])


def make(ranks, experts, width, hidden, topk, tokens, seed=0):
    """A layer and the ranks' tokens, random."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    w_router = (draw(experts, width) * width ** -0.5).to(BF16)
    w1, w2 = (draw(experts, hidden, width) * width ** -0.5).to(BF16), (draw(experts, width, hidden) * hidden ** -0.5).to(BF16)
    xs = [draw(tokens, width).to(BF16) for _ in range(ranks)]
    return ExpertLayer(ranks, experts, width, hidden, topk, w_router, w1, w2), (w_router, w1, w2), xs


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("ranks", 8), ("experts", 16), ("tokens", 2048), ("width", 1024), ("hidden", 2048), ("topk", 4), ("steps", 5)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    layer, _, xs = make(a.ranks, a.experts, a.width, a.hidden, a.topk, a.tokens)
    dys = [torch.randn_like(x) for x in xs]
    torch.cuda.synchronize()
    for i in range(a.steps):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record(layer.stream)
        ys, losses = layer.forward(xs)
        grads = layer.backward(dys)
        end.record(layer.stream)
        layer.stream.synchronize()
        print("step %d: %.2f ms, balance loss %.5f, |y| %.3f, |dx| %.3f" % (i, begin.elapsed_time(end), float(losses[0]), float(ys[0].float().norm()),
                                                                        float(grads[0][0].float().norm())), flush=True)
    layer.close()


if __name__ == "__main__":
    main()
