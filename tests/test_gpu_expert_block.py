"""The example's block of gated experts -- norm, scored router, products, gate, residual and norm, their gradients, clipping over the ranks, the bias --
against the same block in 64 bits without any rounding: what 8 bits cost, and nothing more."""
import importlib.util
import os

import pytest
import torch

import layer_reference as ref
from hccl_loader import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("expert_block", os.path.join(ROOT, "examples", "expert_block.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def norm(x, gain):
    return x * gain / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)


def reference(block, weights, xs, dys):
    """Autograd in 64 bits on the CPU; the choices are the block's (16-bit values may tie)."""
    w_router, w1, w2, gain1, gain2 = (w.double().cpu().requires_grad_() for w in weights)
    outs, total, inputs = [], 0, []
    for s, x, dy in zip(block.ranks, xs, dys):
        x = x.double().cpu().requires_grad_()
        inputs.append(x)
        n = norm(x, gain1)
        chosen = s["expert"].cpu().long()
        w = torch.gather(torch.sigmoid(n @ w_router.t()), 1, chosen)
        w = block.scale * w / w.sum(1, keepdim=True)
        m = torch.zeros_like(x)
        for e in range(block.E):
            for j in range(block.k):
                t = (chosen[:, j] == e).nonzero()[:, 0]
                if t.numel():
                    g, u = (n[t] @ w1[e].t()).chunk(2, 1)
                    m = m.index_add(0, t, w[t, j:j + 1] * ((torch.nn.functional.silu(g) * u) @ w2[e].t()))
        y = norm(x + m, gain2)
        outs.append(y.detach())
        total = total + (y * dy.double().cpu()).sum()
    total.backward()
    return outs, [x.grad for x in inputs], [t.grad for t in (w_router, w1, w2, gain1, gain2)]


@pytest.mark.parametrize("ranks,experts,tokens,width,hidden,topk,groups,kept", [(2, 4, 70, 200, 136, 2, 2, 1), (4, 8, 300, 256, 384, 4, 4, 2),
                                                                               (8, 16, 33, 128, 129, 1, 1, 1)])
def test_block_over_ranks(example, ranks, experts, tokens, width, hidden, topk, groups, kept):
    print("expert block", ranks, experts, tokens, width, hidden, topk, groups, kept, flush=True)
    block, weights, xs = example.make(ranks, experts, width, hidden, topk, tokens, seed=3, groups=groups, kept=kept)
    g = torch.Generator(device="cuda").manual_seed(4)
    dys = [torch.randn(x.shape, generator=g, device="cuda").bfloat16() for x in xs]
    torch.cuda.synchronize()
    try:
        ys, _ = block.forward(xs)
        block.backward(dys)
        block.stream.synchronize()
        names = ("d_x", "d_w1", "d_w2", "d_router", "d_gain1", "d_gain2")
        first = [[s[n].clone() for n in names] for s in block.ranks]
        block.forward(xs)
        block.backward(dys)
        block.stream.synchronize()
        assert all(torch.equal(a, s[n]) for f, s in zip(first, block.ranks) for a, n in zip(f, names))
        outs, rx, (rr, r1, r2, rg1, rg2) = reference(block, weights, xs, dys)
        # rounding to 8 bits moves a value by at most 2^-4 of itself, 2^-4 / sqrt(3) in the mean square: two rounded factors in a product, two products one
        # behind the other forwards with a gate of two rounded factors between them, three and the gate's backwards, all errors independent
        rounding = 2.0 ** -4 / 3 ** 0.5
        shared = [sum(s[n].double().cpu() for s in block.ranks) for n in ("d_router", "d_gain1", "d_gain2")]
        for got, want, factors in ((torch.cat(ys), torch.cat(outs), 6), (torch.cat([s["d_x"] for s in block.ranks]), torch.cat(rx), 12),
                                   (torch.cat([s["d_w1"] for s in block.ranks]), r1, 12), (torch.cat([s["d_w2"] for s in block.ranks]), r2, 10),
                                   (shared[0], rr, 12), (shared[1], rg1, 12), (shared[2], rg2, 6)):
            if topk == 1 and want is rr:
                # one choice's weight over itself is constant: no gradient, and what 64 bits leave of it is their own rounding
                assert not got.any() and want.norm() < 1e-12 * r1.norm()
                continue
            off = (got.double().cpu() - want).norm() / want.norm()
            assert off < rounding * factors ** 0.5, (float(off), factors)
        # one norm over all ranks, what they share counted once; everything is held to it
        before = [[s[n].double().cpu() for n in ("d_w1", "d_w2")] for s in block.ranks]
        want = (sum((t ** 2).sum() for b in before for t in b) + sum((t ** 2).sum() for t in shared)) ** 0.5
        counts = sum(s["counts"].cpu() for s in block.ranks)
        norms = block.clip(1.0)
        block.balance(0.01)
        block.stream.synchronize()
        for s, n, b in zip(block.ranks, norms, before):
            # (the shared ones are added up in 32 bits, up to eight of them)
            assert abs(float(n) - float(want)) <= 16 * 2.0 ** -24 * float(want)
            for name, t in list(zip(("d_w1", "d_w2"), b)) + list(zip(("d_router", "d_gain1", "d_gain2"), shared)):
                by = 1 / max(1.0, float(want))
                assert (s[name].double().cpu() - by * t).norm() <= 32 * 2.0 ** -24 * by * t.norm()
            assert torch.equal(s["counts"].cpu(), counts.int())
        assert torch.equal(block.bias.cpu(), torch.from_numpy(ref.bias_step(counts[:experts].numpy(), 0.01, torch.zeros(experts).numpy())))
    finally:
        block.close()
