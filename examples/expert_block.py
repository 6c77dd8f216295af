"""A block with gated experts over the ranks of one communicator: norm, scored router, experts, residual and norm; its gradients, held to a norm over all
ranks; one step of the bias that balances the experts.

    python examples/expert_block.py [--ranks 8] [--experts 32] [--tokens 2048] [--width 1024] [--hidden 1024] [--topk 4]

Every rank holds tokens and experts / ranks of the experts.  The tokens are normed once into 8-bit rows, which go to their experts as they are; the experts
multiply, gate into 8-bit rows and multiply again; what comes back is added to the tokens and normed for what follows.  All ranks are driven from one thread on
one stream.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from expert_layer import BF16, H, ExpertLayer, _new  # noqa: E402

BF, F32 = H.HCCL_DATA_TYPE_BFP16, H.HCCL_DATA_TYPE_FP32
EPSILON = 1e-6


def _up(n):
    return -(-n // 128) * 128


class ExpertBlock(ExpertLayer):
    """z = x + sum over a token's experts of weight * W2 gate(W1 norm(x)), y = norm(z).  W1[2 * hidden, width] and W2[width, hidden] of every expert."""

    def __init__(self, ranks, experts, width, hidden, topk, w_router, w1, w2, gain1, gain2, groups=4, kept=2, weight_scale=2.5):
        """w_router[experts, width]; w1[experts, 2 * hidden, width], w2[experts, width, hidden], gain1[width], gain2[width]: 16-bit masters."""
        assert experts % ranks == 0 and experts % groups == 0
        self.p, self.E, self.mine, self.W, self.F, self.k = ranks, experts, experts // ranks, width, hidden, topk
        self.w_router, self.gain1, self.gain2, self.scale = w_router, gain1, gain2, weight_scale
        self.groups, self.kept = groups, kept
        self.bias = torch.zeros(experts, device="cuda")
        self.comms = H.comm_init_all(ranks)
        self.stream = torch.cuda.Stream()
        self.owner = torch.arange(self.mine, dtype=torch.int32, device="cuda").repeat(ranks)
        self.ranks = [dict(w1=w1[r * self.mine:(r + 1) * self.mine].contiguous(), w2=w2[r * self.mine:(r + 1) * self.mine].contiguous())
                      for r in range(ranks)]
        torch.cuda.synchronize()
        for s in self.ranks:
            for name, n, k in (("w1", 2 * hidden, width), ("w2", width, hidden)):
                s[name + "_q"], s[name + "_s"] = _new(self.mine, n, _up(k), dtype=torch.uint8), _new(self.mine, _up(n) // 128, _up(k) // 128, dtype=torch.float32)
                s[name + "_qt"], s[name + "_st"] = _new(self.mine, k, _up(n), dtype=torch.uint8), _new(self.mine, _up(k) // 128, _up(n) // 128, dtype=torch.float32)
                H.block_quant_weights(s[name].data_ptr(), BF, self.mine, n, k, H.HCCL_AMD_SCALE_FP32, s[name + "_q"].data_ptr(), s[name + "_s"].data_ptr(),
                                      s[name + "_qt"].data_ptr(), s[name + "_st"].data_ptr(), self.stream.cuda_stream)
        self.stream.synchronize()

    def forward(self, xs):
        """xs: the ranks' tokens [tokens, width].  Returns y and z of every rank; keeps what backward needs."""
        with torch.cuda.stream(self.stream):
            S, p, E, k, W = self.stream.cuda_stream, self.p, self.E, self.k, self.W
            wp = _up(W)
            for s, x in zip(self.ranks, xs):
                T = x.shape[0]
                s["x"], s["normed"] = x, _new(T, W)
                q, q_s = _new(T, wp, dtype=torch.uint8), _new(T, wp // 128, dtype=torch.float32)
                H.norm_rows(x.data_ptr(), BF, T, W, S, gain=self.gain1.data_ptr(), gain_dtype=BF, epsilon=EPSILON, y=s["normed"].data_ptr(),
                            scale_type=H.HCCL_AMD_SCALE_FP32, q=q.data_ptr(), scales=q_s.data_ptr())
                s["logits"] = (s["normed"] @ self.w_router.t()).float()
                s["expert"], s["row_of"], s["weights"] = _new(T, k, dtype=torch.int32), _new(T, k, dtype=torch.int32), _new(T, k, dtype=torch.float32)
                s["counts"], s["offsets"] = _new(E + 1, dtype=torch.int32), _new(E + 1, dtype=torch.int32)
                need = H.expert_route_scored_workspace(T, E)
                work = _new(max(16, need), dtype=torch.uint8)
                H.expert_route_scored(s["logits"].data_ptr(), F32, T, E, k, H.HCCL_AMD_SCORE_SIGMOID, s["expert"].data_ptr(), s["weights"].data_ptr(),
                                      s["row_of"].data_ptr(), s["counts"].data_ptr(), s["offsets"].data_ptr(), work.data_ptr(), need, S,
                                      bias=self.bias.data_ptr(), groups=self.groups, groups_kept=self.kept, renorm=True, weight_scale=self.scale)
                # 8-bit rows and their scales into expert order: a copy moves bits, two values to a 16-bit word
                s["q"], s["q_s"] = _new(T * k, wp, dtype=torch.uint8), _new(T * k, wp // 128, dtype=torch.float32)
                H.expert_pack(q.data_ptr(), BF, T, wp // 2, k, s["row_of"].data_ptr(), s["q"].data_ptr(), T * k, S)
                H.expert_pack(q_s.data_ptr(), F32, T, wp // 128, k, s["row_of"].data_ptr(), s["q_s"].data_ptr(), T * k, S)
            counts = [s["counts"][:E].tolist() for s in self.ranks]
            self.rows = [[sum(c[j * self.mine:(j + 1) * self.mine]) for j in range(p)] for c in counts]
            for j, s in enumerate(self.ranks):
                sizes = [counts[i][j * self.mine + e] for i in range(p) for e in range(self.mine)]
                s["rows"] = sum(sizes)
                s["groups"] = torch.tensor([0] + sizes, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
            qs = self._exchange([s["q"] for s in self.ranks], self.rows, wp, torch.uint8)
            scales = self._exchange([s["q_s"] for s in self.ranks], self.rows, wp // 128, torch.float32)
            for s, q, q_s in zip(self.ranks, qs, scales):
                s["xq"], s["xq_s"] = q, q_s
                s["h"] = self._multiply(s, q, q_s, s["w1_q"], s["w1_s"], 2 * self.F, W)
                R = s["h"].shape[0]
                a, a_s = _new(R, _up(self.F), dtype=torch.uint8), _new(R, _up(self.F) // 128, dtype=torch.float32)
                # how many rows there are the groups' last offset says, on the device
                H.expert_gate(s["h"].data_ptr(), BF, R, self.F, a.data_ptr(), S, used=s["groups"][-1:].data_ptr(), scale_type=H.HCCL_AMD_SCALE_FP32,
                              scales=a_s.data_ptr())
                s["out"] = self._multiply(s, a, a_s, s["w2_q"], s["w2_s"], W, self.F)
            back = self._exchange([s["out"] for s in self.ranks], [list(c) for c in zip(*self.rows)], W, BF16)
            ys, zs = [], []
            for s, rows in zip(self.ranks, back):
                T = s["x"].shape[0]
                s["back"], m, s["z"], y = rows, _new(T, W), _new(T, W), _new(T, W)
                H.expert_combine(rows.data_ptr(), BF, T * k, W, T, k, s["row_of"].data_ptr(), s["weights"].data_ptr(), m.data_ptr(), S)
                H.norm_rows(m.data_ptr(), BF, T, W, S, residual=s["x"].data_ptr(), gain=self.gain2.data_ptr(), gain_dtype=BF, epsilon=EPSILON,
                            sum=s["z"].data_ptr(), y=y.data_ptr())
                ys.append(y)
                zs.append(s["z"])
            return ys, zs

    def _norm_grad(self, dy, total, gain, more):
        T, W = dy.shape
        dx, d_gain, need = _new(T, W), _new(W, dtype=torch.float32), H.norm_rows_grad_workspace(T, W)
        work = _new(max(16, need), dtype=torch.uint8)
        H.norm_rows_grad(dy.data_ptr(), total.data_ptr(), BF, T, W, dx.data_ptr(), self.stream.cuda_stream, gain=gain.data_ptr(), gain_dtype=BF, epsilon=EPSILON,
                         sum_grad=None if more is None else more.data_ptr(), gain_grad=d_gain.data_ptr(), workspace=work.data_ptr(), workspace_bytes=need)
        return dx, d_gain

    def backward(self, dys):
        """Every rank's gradients: of its tokens, its experts' weights, and its part of those that all ranks share (router and gains)."""
        with torch.cuda.stream(self.stream):
            S, E, k, W, F = self.stream.cuda_stream, self.E, self.k, self.W, self.F
            sent = []
            for s, dy in zip(self.ranks, dys):
                T = dy.shape[0]
                s["d_z"], s["d_gain2"] = self._norm_grad(dy, s["z"], self.gain2, None)
                s["d_weights"] = _new(T, k, dtype=torch.float32)
                sent.append(_new(T * k, W))
                H.expert_combine_grad(s["d_z"].data_ptr(), s["back"].data_ptr(), BF, T * k, W, T, k, s["row_of"].data_ptr(), s["weights"].data_ptr(),
                                      sent[-1].data_ptr(), s["d_weights"].data_ptr(), S)
            d_rows = []
            for s, d in zip(self.ranks, self._exchange(sent, self.rows, W, BF16)):
                R = s["h"].shape[0]
                da = self._multiply(s, *self._quantise(d), s["w2_qt"], s["w2_st"], F, W)
                dh, a = _new(R, 2 * F), _new(R, F)
                H.expert_gate_grad(da.data_ptr(), s["h"].data_ptr(), BF, R, F, dh.data_ptr(), S, used=s["groups"][-1:].data_ptr(), out=a.data_ptr())
                s["d_w2"] = self._weight_gradient(s, d, a)
                x = (s["xq"].view(torch.float8_e4m3fn).float().reshape(*s["xq_s"].shape, 128) * s["xq_s"][..., None]).reshape(s["xq"].shape)
                s["d_w1"] = self._weight_gradient(s, dh, x[:, :W].to(BF16).contiguous())
                d_rows.append(self._multiply(s, *self._quantise(dh), s["w1_qt"], s["w1_st"], W, 2 * F))
            for s, rows in zip(self.ranks, self._exchange(d_rows, [list(c) for c in zip(*self.rows)], W, BF16)):
                T = s["x"].shape[0]
                d, d_logits = _new(T, W), _new(T, E, dtype=torch.float32)
                H.expert_combine(rows.data_ptr(), BF, T * k, W, T, k, s["row_of"].data_ptr(), None, d.data_ptr(), S)
                H.expert_route_scored_grad(s["logits"].data_ptr(), F32, T, E, k, H.HCCL_AMD_SCORE_SIGMOID, s["expert"].data_ptr(), s["d_weights"].data_ptr(),
                                           d_logits.data_ptr(), S, renorm=True, weight_scale=self.scale)
                d = (d.float() + d_logits @ self.w_router.float()).to(BF16)
                s["d_router"] = d_logits.t() @ s["normed"].float()
                s["d_x"], s["d_gain1"] = self._norm_grad(d, s["x"], self.gain1, s["d_z"])
            return self.ranks

    def _sum(self, name, dtype):
        """The ranks' s[name] added up; every rank has the sum afterwards."""
        sums = [torch.empty_like(s[name]) for s in self.ranks]
        H.all_reduce(self.comms, [s[name].data_ptr() for s in self.ranks], [t.data_ptr() for t in sums], sums[0].numel(), dtype, H.HCCL_REDUCE_SUM,
                     self.stream.cuda_stream)
        for s, t in zip(self.ranks, sums):
            s[name] = t

    def clip(self, max_norm):
        """Adds up what the ranks share, holds all gradients to one norm over all ranks, in place; returns every rank's norm."""
        with torch.cuda.stream(self.stream):
            S = self.stream.cuda_stream
            for name in ("d_router", "d_gain1", "d_gain2"):
                self._sum(name, F32)
            for r, s in enumerate(self.ranks):
                # the shared ones count once: with rank 0
                own, shared = [s["d_w1"], s["d_w2"]], [s["d_router"], s["d_gain1"], s["d_gain2"]]
                s["tensors"] = H.grad_tensors([(t.data_ptr(), t.data_ptr(), t.numel(), F32) for t in own + shared])
                counted = len(own) + (len(shared) if r == 0 else 0)
                need = H.grad_squares_workspace(s["tensors"], counted)
                s["squares"], work = _new(1, dtype=torch.float64), _new(max(16, need), dtype=torch.uint8)
                H.grad_squares(s["tensors"], counted, s["squares"].data_ptr(), work.data_ptr(), need, S)
            self._sum("squares", H.HCCL_DATA_TYPE_FP64)
            for s in self.ranks:
                s["norm"] = _new(1, dtype=torch.float32)
                H.grad_clip(s["tensors"], len(s["tensors"]), s["squares"].data_ptr(), max_norm, s["norm"].data_ptr(), S)
            return [s["norm"] for s in self.ranks]

    def balance(self, rate):
        """A step of the bias, by the counts of all ranks."""
        with torch.cuda.stream(self.stream):
            self._sum("counts", H.HCCL_DATA_TYPE_INT32)
            H.expert_bias(self.ranks[0]["counts"].data_ptr(), self.E, rate, self.bias.data_ptr(), self.bias.data_ptr(), self.stream.cuda_stream)


def make(ranks, experts, width, hidden, topk, tokens, seed=0, groups=4, kept=2):
    """A block and the ranks' tokens, random."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    w_router = (draw(experts, width) * width ** -0.5).to(BF16)
    w1, w2 = (draw(experts, 2 * hidden, width) * width ** -0.5).to(BF16), (draw(experts, width, hidden) * hidden ** -0.5).to(BF16)
    gain1, gain2 = (1 + 0.1 * draw(width)).to(BF16), (1 + 0.1 * draw(width)).to(BF16)
    xs = [draw(tokens, width).to(BF16) for _ in range(ranks)]
    return ExpertBlock(ranks, experts, width, hidden, topk, w_router, w1, w2, gain1, gain2, groups, kept), (w_router, w1, w2, gain1, gain2), xs


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("ranks", 8), ("experts", 32), ("tokens", 2048), ("width", 1024), ("hidden", 1024), ("topk", 4), ("steps", 5)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    block, _, xs = make(a.ranks, a.experts, a.width, a.hidden, a.topk, a.tokens)
    dys = [torch.randn_like(x) for x in xs]
    torch.cuda.synchronize()
    for i in range(a.steps):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record(block.stream)
        block.forward(xs)
        block.backward(dys)
        norms = block.clip(1.0)
        block.balance(1e-3)
        end.record(block.stream)
        block.stream.synchronize()
        n = block.ranks[0]["counts"][:block.E].float()
        print("step %d: %.2f ms, gradients' norm %.3f, fullest expert %.2f of the mean" % (i, begin.elapsed_time(end), float(norms[0]), float(n.max() / n.mean())),
              flush=True)
    block.close()


if __name__ == "__main__":
    main()
