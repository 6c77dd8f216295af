"""The example's expert-parallel layer, operators and all-to-all-vs together, against the same layer in 64 bits without any rounding:
what 8 bits cost, and nothing more."""
import importlib.util
import os

import pytest
import torch

from hccl_loader import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("expert_layer", os.path.join(ROOT, "examples", "expert_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def reference(layer, weights, xs, dys):
    """Autograd in 64 bits on the CPU; the choices are the layer's (16-bit logits may tie)."""
    w_router, w1, w2 = (w.double().cpu().requires_grad_() for w in weights)
    outs, total, inputs = [], 0, []
    for s, x, dy in zip(layer.ranks, xs, dys):
        x = x.double().cpu().requires_grad_()
        inputs.append(x)
        logits = x @ w_router.t()
        p = torch.softmax(logits, 1)
        chosen = s["expert"].cpu().long()
        w = torch.gather(p, 1, chosen)
        w = w / w.sum(1, keepdim=True)
        y = torch.zeros_like(x)
        for e in range(layer.E):
            for j in range(layer.k):
                t = (chosen[:, j] == e).nonzero()[:, 0]
                if t.numel():
                    y = y.index_add(0, t, w[t, j:j + 1] * (torch.nn.functional.silu(x[t] @ w1[e].t()) @ w2[e].t()))
        n = torch.bincount(chosen.reshape(-1), minlength=layer.E).double()
        loss = layer.loss_scale * layer.E * (n / n.sum() * p.mean(0)).sum()
        outs.append((y.detach(), float(loss.detach())))
        total = total + (y * dy.double().cpu()).sum() + loss
    total.backward()
    return outs, [x.grad for x in inputs], w_router.grad, w1.grad, w2.grad


@pytest.mark.parametrize("ranks,experts,tokens,width,hidden,topk", [(2, 4, 70, 200, 136, 2), (4, 8, 300, 256, 384, 4), (8, 8, 33, 128, 129, 1)])
def test_layer_over_ranks(example, ranks, experts, tokens, width, hidden, topk):
    print("expert layer", ranks, experts, tokens, width, hidden, topk, flush=True)
    layer, weights, xs = example.make(ranks, experts, width, hidden, topk, tokens, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    dys = [torch.randn(x.shape, generator=g, device="cuda").bfloat16() for x in xs]
    torch.cuda.synchronize()
    try:
        ys, losses = layer.forward(xs)
        dxs, d_router, d_w1, d_w2 = layer.backward(dys)
        layer.stream.synchronize()
        first = [t.clone() for t in ys + dxs + [d_w1, d_w2]]
        layer.forward(xs)
        again = layer.backward(dys)
        layer.stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first[len(ys):], again[0] + [again[2], again[3]]))
        outs, rx, rr, r1, r2 = reference(layer, weights, xs, dys)
        # rounding to 8 bits moves a value by at most 2^-4 of itself, 2^-4 / sqrt(3) in the mean square: two rounded factors in a product,
        # two products one behind the other forwards (three and the activation backwards), all errors independent
        rounding = 2.0 ** -4 / 3 ** 0.5
        for got, want, factors in ((torch.cat(ys), torch.cat([o[0] for o in outs]), 4), (torch.cat(dxs), torch.cat(rx), 8), (d_w1, r1, 8), (d_w2, r2, 6),
                                   (d_router, rr, 8)):
            off = (got.double().cpu() - want).norm() / want.norm()
            assert off < rounding * factors ** 0.5, (float(off), factors)
        for loss, (_, want) in zip(losses, outs):
            # 16-bit logits: a probability moves by 2^-8 of the logit's size (4 at most) and back
            assert abs(float(loss) - want) < 2.0 ** -6 * want
    finally:
        layer.close()
