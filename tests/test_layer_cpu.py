"""Norm, scored router, gate and gradient clipping without a GPU: what they refuse and need, the 64-bit reference's gradients against differences."""
import ctypes

import numpy as np
import pytest

import layer_reference as ref
from hccl_loader import load

H = load()
P, N = 1 << 12, 1          # an address that is aligned and never followed, a stream likewise: what is refused is not launched
OK, PARA, PTR, NOT_SUPPORT = 0, 1, 2, 5
FP32, FP16, BF16, INT8, FP64 = 4, 3, 11, 0, 10


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(x=None)), (PTR, dict(q=None)), (PTR, dict(scales=None)), (NOT_SUPPORT, dict(type=INT8)), (NOT_SUPPORT, dict(type=FP64)),
    (NOT_SUPPORT, dict(gain_type=FP16)), (NOT_SUPPORT, dict(kind=3)), (PARA, dict(width=32769, q_stride=0)), (PARA, dict(rows=1 << 31)), (PARA, dict(epsilon=-1.0)),
    (PARA, dict(epsilon=float("nan"))), (PARA, dict(x_stride=299)), (PARA, dict(r_stride=299)), (PARA, dict(sum_stride=299)), (PARA, dict(y_stride=299)),
    (PARA, dict(q_stride=383)), (PARA, dict(q_stride=392)), (PARA, dict(q=P + 8)), (PARA, dict(scales=P + 2)), (PARA, dict(scale_stride=2)),
    (PARA, dict(x=P + 1)), (PARA, dict(residual=P + 1)), (PARA, dict(sum=P + 1)), (PARA, dict(y=P + 1)), (PARA, dict(gain=P + 1)),
    (PARA, dict(kind=0)), (PARA, dict(sum=P, sum_stride=400)), (PARA, dict(sum=P * 2, sum_stride=400)),
    (OK, dict(rows=0, x=None)), (OK, dict(width=0, x=None)), (OK, dict(sum=None, y=None, kind=0, q=None, scales=None, x=None)),
])
def test_norm_refuses(want, kw):
    a = dict(x=P, type=BF16, rows=10, width=300, x_stride=0, residual=P * 2, r_stride=0, gain=P, gain_type=FP32, epsilon=1e-6, sum=P * 3, sum_stride=0, y=P * 4,
             y_stride=0, kind=1, q=P, q_stride=0, scales=P, scale_stride=0, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdNormRows(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(dy=None)), (PTR, dict(sum=None)), (PTR, dict(workspace=None)), (NOT_SUPPORT, dict(type=INT8)),
    (NOT_SUPPORT, dict(gain_type=FP16)), (PARA, dict(width=32769)), (PARA, dict(epsilon=-1.0)), (PARA, dict(dy_stride=299)), (PARA, dict(sum_stride=299)),
    (PARA, dict(dsum_stride=299)), (PARA, dict(dx_stride=299)), (PARA, dict(dx=P + 1)), (PARA, dict(dgain=P + 2)), (PARA, dict(bytes=300 * 4 * 3 - 1)),
    (PARA, dict(workspace=P + 8)), (PARA, dict(dx=P, dx_stride=400)), (PARA, dict(dx=P * 3, dx_stride=400)),
    (OK, dict(width=0, dy=None)), (OK, dict(dx=None, dgain=None, dy=None)), (OK, dict(rows=0, dgain=None, dy=None)),
])
def test_norm_grad_refuses(want, kw):
    a = dict(dy=P, dy_stride=0, sum=P * 2, type=BF16, rows=10, width=300, sum_stride=0, gain=P, gain_type=BF16, epsilon=1e-6, dsum=P * 3, dsum_stride=0, dx=P * 4,
             dx_stride=0, dgain=P, accumulate=0, workspace=P, bytes=1 << 30, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdNormRowsGrad(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(h=None)), (PTR, dict(out=None)), (PTR, dict(scales=None)), (NOT_SUPPORT, dict(type=INT8)), (NOT_SUPPORT, dict(kind=3)),
    (PARA, dict(rows=1 << 31)), (PARA, dict(width=1 << 30)), (PARA, dict(h_stride=599)), (PARA, dict(out_stride=383)), (PARA, dict(out_stride=392)),
    (PARA, dict(out=P + 8)), (PARA, dict(scales=P + 2)), (PARA, dict(scale_stride=2)), (PARA, dict(h=P + 1)), (PARA, dict(used=P + 2)),
    (PARA, dict(kind=0, out_stride=299)), (PARA, dict(kind=0, out=P + 1)), (OK, dict(rows=0, h=None)), (OK, dict(width=0, h=None)),
])
def test_gate_refuses(want, kw):
    a = dict(h=P, type=BF16, rows=10, width=300, h_stride=0, used=P, kind=1, out=P, out_stride=0, scales=P, scale_stride=0, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdExpertGate(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(da=None)), (PTR, dict(h=None)), (NOT_SUPPORT, dict(type=INT8)), (PARA, dict(da_stride=299)), (PARA, dict(h_stride=599)),
    (PARA, dict(dh_stride=599)), (PARA, dict(a_stride=299)), (PARA, dict(dh=P + 1)), (PARA, dict(a=P + 1)), (PARA, dict(used=P + 1)),
    (PARA, dict(dh=P * 2, dh_stride=700)), (PARA, dict(a=P, a_stride=400)), (OK, dict(rows=0, h=None)), (OK, dict(dh=None, a=None, h=None)),
])
def test_gate_grad_refuses(want, kw):
    a = dict(da=P, da_stride=0, h=P * 2, type=BF16, rows=10, width=300, h_stride=0, used=None, dh=P * 3, dh_stride=0, a=P * 4, a_stride=0, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdExpertGateGrad(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(logits=None)), (PTR, dict(expert=None)), (PTR, dict(weights=None)), (PTR, dict(row=None)), (PTR, dict(counts=None)),
    (PTR, dict(offsets=None)), (PTR, dict(workspace=None)), (NOT_SUPPORT, dict(type=INT8)), (NOT_SUPPORT, dict(score=2)), (PARA, dict(experts=0)),
    (PARA, dict(experts=1025, groups=1, kept=1)), (PARA, dict(groups=0)), (PARA, dict(groups=7)), (PARA, dict(groups=128, experts=128)), (PARA, dict(kept=0)),
    (PARA, dict(kept=9)), (PARA, dict(top=0)), (PARA, dict(top=3)), (PARA, dict(topk=0)), (PARA, dict(topk=17)), (PARA, dict(kept=1, topk=9)),
    (PARA, dict(stride=63)), (PARA, dict(bytes=100)), (PARA, dict(workspace=P + 4)), (PARA, dict(logits=P + 1)), (PARA, dict(bias=P + 1)), (PARA, dict(expert=P + 2)),
    (PARA, dict(tokens=(1 << 25) + 1)),
])
def test_route_refuses(want, kw):
    a = dict(logits=P, type=BF16, tokens=100, experts=64, stride=0, score=1, bias=P, groups=8, kept=4, top=2, topk=8, renorm=0, scale=1.0, mask=None, expert=P,
             weights=P, row=P, counts=P, offsets=P, workspace=P, bytes=1 << 30, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdExpertRouteScored(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(logits=None)), (PTR, dict(expert=None)), (PTR, dict(dw=None)), (PTR, dict(out=None)), (NOT_SUPPORT, dict(type=FP64)),
    (NOT_SUPPORT, dict(score=7)), (PARA, dict(topk=17)), (PARA, dict(topk=65)), (PARA, dict(stride=8)), (PARA, dict(out_stride=8)), (PARA, dict(out=P + 1)),
    (PARA, dict(dw=P + 1)), (OK, dict(tokens=0, logits=None)),
])
def test_route_grad_refuses(want, kw):
    a = dict(logits=P, type=BF16, tokens=100, experts=64, stride=0, score=1, topk=8, renorm=0, scale=1.0, expert=P, dw=P, out=P, out_stride=0, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdExpertRouteScoredGrad(*a.values()) == want


@pytest.mark.parametrize("want,args", [
    (PTR, (P, 64, 0.1, P, P, None)), (PTR, (None, 64, 0.1, P, P, N)), (PTR, (P, 64, 0.1, None, P, N)), (PTR, (P, 64, 0.1, P, None, N)),
    (PARA, (P, 0, 0.1, P, P, N)), (PARA, (P, 1025, 0.1, P, P, N)), (PARA, (P + 1, 64, 0.1, P, P, N)), (PARA, (P, 64, 0.1, P + 1, P, N)),
])
def test_bias_refuses(want, args):
    assert H.lib().HcclAmdExpertBias(*args) == want


def tensors(*of):
    return H.grad_tensors([(P, P * 2, 100, BF16)] + list(of))


@pytest.mark.parametrize("want,of", [
    (NOT_SUPPORT, (P, P, 100, INT8)), (NOT_SUPPORT, (P, P, 0, FP64)), (PARA, (P + 1, P, 100, BF16)), (PARA, (P + 2, P, 100, FP32)), (PARA, (P, P, 1 << 38, BF16)),
    (PTR, (None, P, 100, BF16)),
])
def test_squares_and_clip_refuse_tensors(want, of):
    t = tensors(of)
    at = ctypes.addressof(t)
    assert H.lib().HcclAmdGradSquares(at, 2, 0, P, P, 1 << 20, N) == want
    assert H.lib().HcclAmdGradClip(at, 2, P, 1.0, P, N) == want
    assert H.lib().HcclAmdGradSquaresWorkspace(at, 2, ctypes.byref(ctypes.c_uint64())) == want


def test_squares_and_clip_refuse():
    t = tensors()
    at, L = ctypes.addressof(t), H.lib()
    for want, args in ((PTR, (at, 1, 0, P, P, 1 << 20, None)), (PTR, (at, 1, 0, None, P, 1 << 20, N)), (PTR, (None, 1, 0, P, P, 1 << 20, N)),
                       (PTR, (at, 1, 0, P, None, 1 << 20, N)), (PARA, (at, 1, 0, P + 4, P, 1 << 20, N)), (PARA, (at, 1, 0, P, P + 8, 1 << 20, N)),
                       (PARA, (at, 1, 0, P, P, 7, N))):
        assert L.HcclAmdGradSquares(*args) == want
    for want, args in ((PTR, (at, 1, P, 1.0, P, None)), (PTR, (at, 1, None, 1.0, P, N)), (PTR, (None, 1, P, 1.0, P, N)), (PARA, (at, 1, P + 4, 1.0, P, N)),
                       (PARA, (at, 1, P, 1.0, P + 2, N)), (PARA, (at, 1, P, -1.0, P, N)), (PARA, (at, 1, P, float("nan"), P, N)), (OK, (None, 0, P, 1.0, None, N))):
        assert L.HcclAmdGradClip(*args) == want
    for out in (None, P + 1):
        bad = H.grad_tensors([(P, out, 100, BF16)])
        assert L.HcclAmdGradClip(ctypes.addressof(bad), 1, P, 1.0, P, N) == (PTR if out is None else PARA)
    t[0].reserved = 1
    assert L.HcclAmdGradSquares(at, 1, 0, P, P, 1 << 20, N) == PARA


def test_workspaces():
    L, need = H.lib(), ctypes.c_uint64(77)
    assert L.HcclAmdNormRowsGradWorkspace(0, 300, ctypes.byref(need)) == OK and need.value == 0
    for rows, width in ((1, 1), (10, 300), (1 << 20, 32768)):
        assert H.norm_rows_grad_workspace(rows, width) >= 4 * width
        assert H.norm_rows_grad_workspace(rows, width) <= 4 * 2048 * width
    assert L.HcclAmdNormRowsGradWorkspace(1, 1, None) == PTR and L.HcclAmdNormRowsGradWorkspace(1, 32769, ctypes.byref(need)) == PARA
    assert L.HcclAmdExpertRouteScoredWorkspace(1, 64, None) == PTR
    for tokens, experts in ((1, 0), (1, 1025), ((1 << 25) + 1, 8)):
        assert L.HcclAmdExpertRouteScoredWorkspace(tokens, experts, ctypes.byref(need)) == PARA
    for tokens in (0, 1, 65, 1000, 65536, 1 << 25):
        for experts in (1, 60, 256, 1024):
            assert H.expert_route_scored_workspace(tokens, experts) < 1 << 24
    assert L.HcclAmdGradSquaresWorkspace(None, 0, ctypes.byref(need)) == OK and need.value == 0
    assert L.HcclAmdGradSquaresWorkspace(None, 1, ctypes.byref(need)) == PTR and L.HcclAmdGradSquaresWorkspace(None, 0, None) == PTR
    many = H.grad_tensors([(P, None, 1, FP32)] * 1000)
    assert 8000 <= H.grad_squares_workspace(many, 1000) < 1 << 20


@pytest.mark.parametrize("stride", [2 ** 64 - 1024, 2 ** 63, 2 ** 40 + 16])
def test_strides_that_no_memory_has(stride):
    calls = [("HcclAmdNormRows", (P, BF16, 10, 300, 0, P, 0, P, FP32, 1e-6, P * 3, 0, P, 0, 1, P, 0, P, 0, N), (4, 6, 11, 13, 16, 18)),
             ("HcclAmdNormRowsGrad", (P, 0, P, BF16, 10, 300, 0, P, FP32, 1e-6, P, 0, P * 5, 0, None, 0, None, 0, N), (1, 6, 11, 13)),
             ("HcclAmdExpertGate", (P, BF16, 10, 300, 0, None, 1, P, 0, P, 0, N), (4, 8, 10)),
             ("HcclAmdExpertGate", (P, BF16, 10, 300, 0, None, 0, P, 0, None, 0, N), (4, 8)),
             ("HcclAmdExpertGateGrad", (P, 0, P, BF16, 10, 300, 0, None, P * 3, 0, P * 4, 0, N), (1, 6, 9, 11)),
             ("HcclAmdExpertRouteScored", (P, BF16, 100, 64, 0, 1, None, 1, 1, 1, 8, 0, 1.0, None, P, P, P, P, P, P, 1 << 30, N), (4,)),
             ("HcclAmdExpertRouteScoredGrad", (P, BF16, 100, 64, 0, 1, 8, 0, 1.0, P, P, P, 0, N), (4, 12))]
    for fn, args, at in calls:
        for i in at:
            assert args[i] == 0
            assert getattr(H.lib(), fn)(*args[:i], stride, *args[i + 1:]) == PARA, (fn, i)


def test_native_calls_and_ctypes_refuse_alike():
    calls = [(9, (P, BF16, 10, 300, 0, None, 0, None, FP32, -1.0, P, 0, P, 0, 0, None, 0, None, 0, N)), (10, (P, 0, P, BF16, 10, 300, 0, None, FP32, -1.0, None, 0, P, 0, None, 0, None, 0, N)),
             (11, (P, INT8, 10, 300, 0, None, 0, P, 0, None, 0, N)), (12, (P, 0, P, INT8, 10, 300, 0, None, P, 0, None, 0, N)),
             (13, (P, BF16, 100, 64, 0, 2, None, 1, 1, 1, 8, 0, 1.0, None, P, P, P, P, P, P, 1 << 30, N)), (14, (P, BF16, 100, 64, 0, 2, 8, 0, 1.0, P, P, P, 0, N)),
             (15, (P, 0, 0.5, P, P, N)), (16, (None, 1, 0, P, P, 100, N)), (17, (None, 1, P, 1.0, P, N))]
    assert len(H._EXPERT_CALLS) == 18
    for kind, args in calls:
        code = getattr(H.lib(), H._EXPERT_CALLS[kind])(*args)
        assert code in (PARA, PTR, NOT_SUPPORT)
        assert H._expert(kind, *args) in ((code,) if H._expert is not H._through_ctypes else (-1,))
        with pytest.raises(H.HcclError) as e:
            H._expert_call(kind, *args)
        assert e.value.code == code


# ---- the reference's gradients against differences ----------------------------------------------------------------------------------

def slopes(f, x, h):
    out = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        step = np.zeros_like(x)
        step[i] = h
        out[i] = (f(x + step) - f(x - step)) / (2 * h)
    return out


@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (2, 16)])
def test_reference_norm_gradient(rows, width):
    rng = np.random.default_rng(rows + width)
    x, r, dy, dsum = (rng.standard_normal((rows, width)) for _ in range(4))
    gain, eps = rng.uniform(0.5, 1.5, width), 0.01

    def value(x, gain):
        s, y = ref.norm(x, r, gain, eps)
        return (y * dy).sum() + (s * dsum).sum()

    dx, dgain, _, _ = ref.norm_grad(dy, x + r, gain, eps, dsum)
    # (eps holds third derivatives below 1e4 times the gradients; cancellation costs 2^-53 / h)
    assert np.abs(slopes(lambda v: value(v, gain), x, 1e-5) - dx).max() < 1e-5
    assert np.abs(slopes(lambda v: value(x, v), gain, 1e-5) - dgain).max() < 1e-8


def test_reference_gate_gradient():
    rng = np.random.default_rng(3)
    g, u, da = (2 * rng.standard_normal((5, 9)) for _ in range(3))
    dg, du, _, _ = ref.gate_grad(da, g, u)
    assert np.abs(slopes(lambda v: (ref.gate(v, u) * da).sum(), g, 1e-5) - dg).max() < 1e-7
    assert np.abs(slopes(lambda v: (ref.gate(g, v) * da).sum(), u, 1e-5) - du).max() < 1e-7


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("tokens,experts,groups,kept,topk", [(1, 1, 1, 1, 1), (5, 12, 3, 2, 3), (7, 9, 1, 1, 9), (4, 16, 8, 3, 4)])
def test_reference_route_gradient(kind, renorm, tokens, experts, groups, kept, topk):
    rng = np.random.default_rng(tokens * 100 + experts)
    # logits far enough apart that no step changes a choice
    x = np.stack([rng.permutation(experts) * 0.3 - 1 for _ in range(tokens)]) + rng.uniform(0, 0.1, (tokens, experts))
    bias = rng.permutation(experts) * 0.01
    mask = np.ones(tokens, np.uint8)
    if tokens > 4:
        mask[2] = 0
        x[2, 0] = np.nan
    dw = rng.standard_normal((tokens, topk))
    base = ref.route(x, kind, bias, groups, kept, 2, topk, renorm, 2.5, mask)
    got, _ = ref.route_grad(x, base, kind, topk, renorm, 2.5, dw)

    def value(v):
        r = ref.route(v, kind, bias, groups, kept, 2, topk, renorm, 2.5, mask)
        assert np.array_equal(r["expert"], base["expert"])
        return (r["weights"] * dw).sum()

    assert np.abs(slopes(value, x, 1e-5) - got).max() < 1e-7 * (1 + np.abs(dw).sum())


def test_reference_bias():
    counts = np.array([5, 0, 3, 4, 3], np.int32)      # mean 3
    assert np.array_equal(ref.bias_step(counts, 0.5, np.zeros(5, np.float32)), np.float32([-0.5, 0.5, 0, -0.5, 0]))


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups,kept,top,topk", [(1, 1, 1, 5), (4, 2, 2, 3), (6, 3, 1, 4)])
def test_reference_of_many_tokens_is_the_reference(kind, groups, kept, top, topk):
    rng = np.random.default_rng(groups)
    x = rng.integers(-4, 4, (60, 12)) * 0.5                   # ties everywhere
    bias = rng.integers(-1, 2, 12) * 0.25
    for renorm in (False, True):
        a = ref.route(x, kind, bias, groups, kept, top, topk, renorm, 1.5, None)
        b = ref.route_many(x, kind, bias, groups, kept, top, topk, renorm, 1.5)
        for k in ("expert", "row_of", "counts", "offsets"):
            assert np.array_equal(a[k], b[k]), k
        assert np.allclose(a["weights"], b["weights"], rtol=1e-13)
