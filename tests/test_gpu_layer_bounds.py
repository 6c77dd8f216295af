"""Norm, scored router and gate on the GPU where their definitions and their precision are easily missed: bounds here count each rounding once, so that a
power whose argument is rounded, or a sum over many rows in 32 bits, is outside of them.

One rounding is half a unit in the last place, U = 2^-24 of the value in 32 bits; the hardware's power and reciprocal are within a unit, 2 U."""
import numpy as np
import pytest
import torch

import layer_reference as ref
from experts_reference import U
from hccl_loader import load
from test_gpu_layer import TYPE, draw, f64, near, run_route

pytestmark = pytest.mark.gpu
H = load()


@pytest.fixture(scope="module")
def stream():
    return torch.cuda.Stream()


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
