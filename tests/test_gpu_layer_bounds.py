"""Norm, scored router and gate on the GPU where their definitions and their precision are easily missed: bounds here count each rounding once, so that a
power whose argument is rounded, or a sum over many rows in 32 bits, is outside of them.

One rounding is half a unit in the last place, U = 2^-24 of the value in 32 bits; the hardware's power and reciprocal are within a unit, 2 U."""
import numpy as np
import pytest
import torch

import layer_reference as ref
from experts_reference import U
from hccl_loader import load
from test_gpu_experts import Out, dt
from test_gpu_layer import TYPE, draw, f64, grad_norm, near, put, ready, run_route

pytestmark = pytest.mark.gpu
H = load()


@pytest.fixture(scope="module")
def stream():
    yield torch.cuda.Stream()
    # (blocks of this size that torch keeps would lie between buffers that tests of small collectives expect near each other)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


# ---- scored router ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups,kept,experts", [(1, 1, 64), (8, 3, 64), (8, 3, 256), (5, 2, 40), (1, 1, 300)])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 25, 2.0 ** 32, -2.0 ** 40, 1e17, -3e38])
def test_route_large_biases(stream, kind, groups, kept, experts, size):
    """Next to a large bias 64 bits hold little of a score, or nothing: what ties there goes to the lowest group and expert, whatever 32 bits could tell apart."""
    x = draw(experts, 150, experts)
    equal = np.full(experts, size, np.float32)
    step = equal.copy()
    step[::3] = np.nextafter(np.float32(size), np.float32(np.inf))
    mixed = np.where(np.arange(experts) % 2 == 0, equal, np.float32(0.25))
    for bias in (equal, step, mixed):
        for top in (1, 2):
            got, _ = run_route(stream, x, kind, bias, groups, kept, top, 6, True, 1.0, None)
            r = ref.route_many(f64(x), kind, bias.astype(np.float64), groups, kept, top, 6, True, 1.0)
            for k in ("expert", "row_of"):
                assert np.array_equal(got[k], r[k]), (k, int((got[k] != r[k]).any(1).sum()))


def few_left(seed, tokens, experts, dtype):
    """Eight logits of each token between -80 and 0, -inf at its other experts."""
    rng = np.random.default_rng(seed)
    at = np.argsort(rng.random((tokens, experts)), axis=1)[:, :8]
    x = np.full((tokens, experts), -np.inf, np.float32)
    np.put_along_axis(x, at, rng.uniform(-80, 0, (tokens, 8)).astype(np.float32), 1)
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("tokens,experts", [(300, 8), (4200, 64), (300, 100), (4200, 128), (4200, 256), (300, 256), (300, 600)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_weights_of_small_scores(stream, tokens, experts, dtype, kind, renorm):
    """Weights and gradients are as exact for scores of 1e-30 as for those next to 1.

    A power is within 3 U: its argument loses nothing, the hardware's power 2 U, the product of the two one more.  With e = exp(-|x|), 1 / (1 + e) is within 3.5 U (half
    of e's, sum, quotient) and e / (1 + e) within 6 (e's, sum, quotient, product).
      weights    sigmoid 6;  renormalised: a share is a power times 1 / (1 + e), 7.5, four sums on top for eight of them, the quotient: 20
                 softmax: the power's 3, the sum's 3 + 13 (eight to each of four sums of a lane, then 2 and 3 levels; 16 to 64 lanes 4 + 2 + 6), the quotient: 20
                 renormalised: 3 for the share, 7 for the sum, 1: 11;  all of them one more for the scale
      gradients, of their magnitudes
                 sigmoid: 6 + 3.5, two products, the scale: 12.5
                 softmax: power 3, inverse of the sum 3 + 16 + 6 + 1, product: 30; times a sum over the chosen, 32 and 6, and product: 69, sum 70, scale 71
                 renormalised, with w's 20 (sigmoid) or 11: the mean w's and 5, the difference and two products 3, 1 - s 7, scale: 56 and 31"""
    x = few_left(experts + tokens, tokens, experts, TYPE[dtype])
    dw = np.random.default_rng(1).standard_normal((tokens, 8)).astype(np.float32)
    got, grad = run_route(stream, x, kind, None, 1, 1, 1, 8, renorm, 1.5, None, dw)
    r = ref.route_many(f64(x), kind, None, 1, 1, 1, 8, renorm, 1.5)
    assert np.array_equal(got["expert"], r["expert"])
    weights = {("sigmoid", False): 7, ("sigmoid", True): 21, ("softmax", False): 21, ("softmax", True): 12}[kind, renorm]
    assert near(got["weights"], r["weights"], weights * U * r["weights"] + 2.0 ** -126)
    some = slice(0, 300)
    want, size = ref.route_grad(f64(x)[some], {k: r[k][some] for k in ("expert", "weights", "scores")}, kind, 8, renorm, 1.5, dw[some])
    rel = {("sigmoid", False): 12.5, ("sigmoid", True): 56, ("softmax", False): 71, ("softmax", True): 31}[kind, renorm]
    assert near(grad[some], want, rel * U * size + 2.0 ** -120, x.dtype)


@pytest.mark.parametrize("tokens,experts", [(40, 24), (4200, 24), (40, 200), (40, 300)])
@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_grad_of_tokens_that_are_not_finite(stream, tokens, experts, kind, renorm):
    """NaN and +inf, chosen and not: what their tokens' gradients are, and that the other tokens' are as ever."""
    inf, nan = float("inf"), float("nan")
    x, bias = draw(4, tokens, experts), np.zeros(experts, np.float32)
    bias[7] = -np.inf                                      # never chosen
    x[3, 5], x[5, 5], x[9, 7], x[11, 5], x[11, 6] = nan, inf, inf, inf, inf
    dw = np.random.default_rng(1).standard_normal((tokens, 4)).astype(np.float32)
    got, grad = run_route(stream, x, kind, bias, 1, 1, 1, 4, renorm, 1.5, None, dw)
    y = f64(x)
    r = ref.route(y, kind, bias, 1, 1, 1, 4, renorm, 1.5, None)
    assert np.array_equal(got["expert"], r["expert"]) and (r["expert"] >= 0).all()
    assert np.array_equal(np.isnan(got["weights"]), np.isnan(r["weights"]))
    if kind == "softmax":
        assert np.isnan(r["weights"]).all(1).nonzero()[0].tolist() == [3, 5, 9, 11]
    if kind == "softmax" and renorm:
        chosen = np.take_along_axis(y, r["expert"].astype(np.int64), 1)
        with np.errstate(invalid="ignore"):
            w = np.exp(chosen - chosen.max(1, keepdims=True))
        r["weights"] = 1.5 * w / w.sum(1, keepdims=True)   # without the others
    want, size = ref.route_grad(y, r, kind, 4, renorm, 1.5, dw)
    if kind == "softmax" and not renorm:
        want[[3, 5, 9, 11]] = np.nan
    nans = {("softmax", False): 4 * experts, ("softmax", True): 8}.get((kind, renorm), 0)
    assert np.isnan(want).sum() == nans and np.array_equal(np.isnan(grad), np.isnan(want))
    # (the bound of the test above, for the largest of its forms)
    assert near(grad, want, 71 * U * np.nan_to_num(size) + 2.0 ** -120)


# ---- gate ---------------------------------------------------------------------------------------------------------------------

def run_gate(stream, g, u, da):
    """a, a once more, dh, all in 32 bits."""
    rows, width = g.shape
    ins, das = put(torch.cat([g, u], 1)), put(da)
    a, again, dh = Out(rows, width, torch.float32), Out(rows, width, torch.float32), Out(rows, 2 * width, torch.float32)
    ready()
    H.expert_gate(ins.ptr, dt(g.dtype), rows, width, a.ptr, stream.cuda_stream)
    H.expert_gate_grad(das.ptr, ins.ptr, dt(g.dtype), rows, width, dh.ptr, stream.cuda_stream, out=again.ptr)
    stream.synchronize()
    return a.numpy(), again.numpy(), dh.numpy()[:, :width], dh.numpy()[:, width:]


@pytest.mark.parametrize("low,high", [(-1, 1), (-10, 0), (0, 8), (8, 17), (17, 60), (-40, -10), (-87, -40), (-110, -87)])
@pytest.mark.parametrize("width", [512, 501])
def test_gate_is_as_exact_everywhere(stream, low, high, width):
    """With E = exp(-g), t = 1 / (1 + E): the power 2 U, its factor 1, the sum 1, the reciprocal 2, t 6 in all.  a and du have two products more.  1 - t is E t where g > 0 (3 for E,
    a product, 6 for t, a product: 11), else 7; 1 + g (1 - t) multiplies that by g (one more), and the sum, t's 6 and three products are 10."""
    g = torch.rand(200, width, generator=torch.Generator().manual_seed(low + 200)) * (high - low) + low
    u, da = draw(1, 200, width), draw(2, 200, width)
    a, again, dg, du = run_gate(stream, g, u, da)
    g, u, da = f64(g), f64(u), f64(da)
    want_g, want_u, size_g, size_u = ref.gate_grad(da, g, u)
    least = 2.0 ** -125 * (1 + np.abs(g)) * (1 + np.abs(u)) * (1 + np.abs(da))      # what a sigmoid below 2^-126 that is 0 makes
    assert near(a, ref.gate(g, u), 8 * U * np.abs(ref.gate(g, u)) + least) and np.array_equal(a, again)
    assert near(du, want_u, 8 * U * size_u + least)
    part = np.abs(g) * ref.sigmoid(-g)
    assert near(dg, want_g, (10 + 12 * part / (1 + part)) * U * size_g + least)


def test_gate_far_and_not_finite(stream):
    """Gates beyond the power's range, infinities and NaN: results and both gradients are the formula's, as it comes out in 64 bits and is rounded to 32."""
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([[0.0, -0.0, 90.0, -90.0, 200.0, -200.0, 3e38, -3e38, inf, -inf, nan, 1e-30, -1e-30, 1e5, -1e5, 1.0, 1.0, 1.0, 0.0, 0.0]])
    u = torch.full_like(g, 2.0)
    u[0, 15:] = torch.tensor([inf, -inf, nan, inf, nan])
    a, again, dg, du = run_gate(stream, g, u, torch.ones_like(g))
    with np.errstate(all="ignore"):
        want = ref.gate(f64(g), f64(u))
        want_g, want_u, _, _ = ref.gate_grad(np.ones(g.shape), f64(g), f64(u))
        # in 64 bits t is not 0 at -200, and its product with 3e38 no infinity
        for got, w in ((a, want), (again, want), (dg, want_g), (du, want_u)):
            w = w.astype(np.float32).astype(np.float64)
            assert np.array_equal(np.isnan(got), np.isnan(w)) and np.array_equal(np.isposinf(got), np.isposinf(w)) and np.array_equal(np.isneginf(got), np.isneginf(w))
            fine = np.isfinite(w)
            assert near(got[fine], w[fine], 22 * U * np.abs(w[fine]) + 2.0 ** -117)


# ---- norm ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,width", [(20000, 64), (40000, 512), (20000, 1000), (10000, 2001), (8000, 4096), (6000, 8192), (3000, 16384), (1200, 32767)])
@pytest.mark.parametrize("start", [False, True])
def test_gain_gradient_of_many_rows(stream, rows, width, start):
    """Terms of one sign, where every sum's rounding shows.  A term has the roundings of the row's factor and of two products, a workgroup's sum one, the result one: 5 U, and
    beyond 8192 columns one for each row of a workgroup, of which there are 256.  As a whole the terms' roundings, thousands that are independent, leave little, and the workgroups'
    as much: the result's own, 3^-1/2 U on average, has to be most of it."""
    s, dy = draw(1, rows, width).abs(), draw(2, rows, width).abs()
    before = draw(3, width).abs() if start else None
    _, dgain = grad_norm(stream, dy, s, None, 1e-6, None, want_dx=False, start=before)
    want = f64(before) if start else np.zeros(width)
    for at in range(0, rows, 1000):
        v = s[at:at + 1000].cuda().double()
        n = v * (v.square().mean(1, keepdim=True) + float(np.float32(1e-6))).rsqrt()
        want += (dy[at:at + 1000].cuda().double() * n).sum(0).cpu().numpy()
    off = np.abs(dgain.numpy()[0] - want) / want
    assert off.max() <= (5 + (-(-rows // 256) if width > 8192 else 0)) * U
    assert (off ** 2).mean() ** 0.5 <= U
