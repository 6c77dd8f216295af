"""The experts' operators without a GPU: what they refuse, what they need, the 64-bit reference's gradients against differences."""
import ctypes
import importlib.util
import os
import re

import numpy as np
import pytest

import experts_reference as ref
from hccl_loader import ROOT, load

H = load()
P, N = 1 << 12, 1          # an address that is aligned and never followed, a stream likewise: what is refused is not launched
OK, PARA, PTR, NOT_SUPPORT = 0, 1, 2, 5
FP32, FP16, BF16, INT8, FP64 = 4, 3, 11, 0, 10


def test_header_is_bound():
    with open(os.path.join(ROOT, "include", "hccl", "hccl_amd_experts.h")) as f:
        declared = set(re.findall(r"^extern HcclResult (\w+)\(", f.read(), re.M))
    assert declared == set(H.EXPERT_EXPORTS)
    for name in declared:
        assert getattr(H.lib(), name).argtypes is not None


def route(**kw):
    a = dict(logits=P, type=BF16, tokens=100, experts=64, stride=0, topk=8, renorm=0, mask=None, scale=1.0, expert=P, weights=P, row=P, counts=P,
             offsets=P, loss=P, workspace=P, bytes=1 << 30, stream=N)
    a.update(kw)
    return H.lib().HcclAmdExpertRoute(*a.values())


def test_workspace():
    need = ctypes.c_uint64(77)
    L = H.lib()
    assert L.HcclAmdExpertRouteWorkspace(64, 256, ctypes.byref(need)) == OK and need.value == 0
    last = 0
    for tokens in (65, 1000, 16383, 65536, 1 << 25):
        for experts in (1, 60, 256, 1024):
            assert L.HcclAmdExpertRouteWorkspace(tokens, experts, ctypes.byref(need)) == OK
            assert need.value >= experts * 4 and need.value < 1 << 36
    assert L.HcclAmdExpertRouteWorkspace(1, 64, None) == PTR
    for tokens, experts in ((1, 0), (1, 1025), ((1 << 25) + 1, 8)):
        assert L.HcclAmdExpertRouteWorkspace(tokens, experts, ctypes.byref(need)) == PARA


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(logits=None)), (PTR, dict(expert=None)), (PTR, dict(weights=None)), (PTR, dict(row=None)),
    (PTR, dict(counts=None)), (PTR, dict(offsets=None)), (PTR, dict(loss=None)), (PTR, dict(workspace=None)),
    (NOT_SUPPORT, dict(type=INT8)), (NOT_SUPPORT, dict(type=FP64)), (NOT_SUPPORT, dict(type=14)),
    (PARA, dict(experts=0)), (PARA, dict(experts=1025)), (PARA, dict(topk=0)), (PARA, dict(topk=17)), (PARA, dict(experts=4, topk=5)),
    (PARA, dict(stride=63)), (PARA, dict(bytes=100)), (PARA, dict(workspace=P + 4)), (PARA, dict(logits=P + 1)), (PARA, dict(expert=P + 2)),
    (PARA, dict(tokens=(1 << 25) + 1)),
])
def test_route_refuses(want, kw):
    assert route(**kw) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(logits=None)), (PTR, dict(expert=None)), (PTR, dict(counts=None)), (PTR, dict(out=None)),
    (NOT_SUPPORT, dict(type=FP64)), (PARA, dict(topk=17)), (PARA, dict(stride=8)), (PARA, dict(out_stride=8)), (PARA, dict(out=P + 1)),
    (PARA, dict(dw=P + 1)), (OK, dict(tokens=0, logits=None, expert=None, counts=None, out=None)),
])
def test_route_grad_refuses(want, kw):
    a = dict(logits=P, type=BF16, tokens=100, experts=64, stride=0, topk=8, renorm=0, mask=None, scale=1.0, expert=P, counts=P, dw=P, dloss=P, out=P,
             out_stride=0, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdExpertRouteGrad(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(x=None)), (PTR, dict(out=None)), (PTR, dict(scales=None)),
    (NOT_SUPPORT, dict(type=INT8)), (NOT_SUPPORT, dict(kind=3)),
    (PARA, dict(topk=0)), (PARA, dict(topk=17)), (PARA, dict(row=None)), (PARA, dict(x_stride=299)), (PARA, dict(out_stride=383)),
    (PARA, dict(out_stride=392)), (PARA, dict(out=P + 8)), (PARA, dict(scale_stride=2)), (PARA, dict(scales=P + 2)), (PARA, dict(x=P + 1)),
    (PARA, dict(kind=0, out_stride=299)), (PARA, dict(kind=0, out=P + 1)),
    (OK, dict(tokens=0, x=None)), (OK, dict(rows=0, out=None)), (OK, dict(width=0, x=None)),
])
def test_pack_refuses(want, kw):
    a = dict(x=P, type=BF16, tokens=10, width=300, x_stride=0, topk=2, row=P, kind=1, out=P, rows=20, out_stride=0, scales=P, scale_stride=0, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdExpertPack(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(x=None)), (PTR, dict(y=None)), (NOT_SUPPORT, dict(type=14)), (PARA, dict(topk=17)), (PARA, dict(row=None)),
    (PARA, dict(x_stride=9)), (PARA, dict(y_stride=9)), (PARA, dict(y=P + 1)), (PARA, dict(weights=P + 2)), (OK, dict(tokens=0, y=None)),
    (OK, dict(width=0, x=None, y=None)),
])
def test_combine_refuses(want, kw):
    a = dict(x=P, type=BF16, rows=20, width=300, x_stride=0, tokens=10, topk=2, row=P, weights=P, y=P, y_stride=0, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdExpertCombine(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(dy=None)), (PTR, dict(x=None)), (NOT_SUPPORT, dict(type=INT8)), (PARA, dict(topk=0)), (PARA, dict(row=None)),
    (PARA, dict(dy_stride=9)), (PARA, dict(x_stride=9)), (PARA, dict(dx_stride=9)), (PARA, dict(dx=P + 1)), (PARA, dict(dw=P + 2)),
    (OK, dict(tokens=0)), (OK, dict(dx=None, dw=None)),
])
def test_combine_grad_refuses(want, kw):
    a = dict(dy=P, dy_stride=0, x=P, type=FP16, rows=20, width=300, x_stride=0, tokens=10, topk=2, row=P, weights=P, dx=P, dx_stride=0, dw=P, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdExpertCombineGrad(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(w=None)), (PTR, dict(scales=None)), (PTR, dict(scales_t=None)), (NOT_SUPPORT, dict(type=INT8)),
    (NOT_SUPPORT, dict(kind=0)), (PARA, dict(stride=99)), (PARA, dict(q=P + 8)), (PARA, dict(q_t=P + 8)), (PARA, dict(experts=4097)),
    (OK, dict(q=None, q_t=None)), (OK, dict(experts=0)), (OK, dict(n=0)), (OK, dict(k=0)),
])
def test_quant_weights_refuses(want, kw):
    a = dict(w=P, type=BF16, experts=2, n=300, k=100, stride=0, kind=1, q=P, scales=P, q_t=P, scales_t=P, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdBlockQuantWeights(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(x=None)), (PTR, dict(q=None)), (PTR, dict(scales=None)), (NOT_SUPPORT, dict(type=INT8)),
    (NOT_SUPPORT, dict(kind=0)), (PARA, dict(groups=0)), (PARA, dict(groups=4097)), (PARA, dict(offsets=None)), (PARA, dict(columns=1000)),
    (PARA, dict(columns=1024 - 128)), (PARA, dict(stride=9)), (PARA, dict(q=P + 8)), (PARA, dict(rows=(1 << 28) + 1, columns=1 << 30)),
    (OK, dict(rows=0, x=None)), (OK, dict(width=0, x=None)),
])
def test_quant_columns_refuses(want, kw):
    a = dict(x=P, type=BF16, rows=600, width=100, stride=0, groups=4, offsets=P, kind=1, q=P, columns=1024, scales=P, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdBlockQuantColumns(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(a=None)), (PTR, dict(sa=None)), (PTR, dict(w=None)), (PTR, dict(sw=None)), (PTR, dict(y=None)),
    (NOT_SUPPORT, dict(type=INT8)), (NOT_SUPPORT, dict(kind=0)), (NOT_SUPPORT, dict(kind=7)),
    (PARA, dict(groups=0)), (PARA, dict(experts=0)), (PARA, dict(groups=4097, owner=P)), (PARA, dict(offsets=None)), (PARA, dict(groups=5)),
    (PARA, dict(stride=299)), (PARA, dict(stride=392)), (PARA, dict(a=P + 8)), (PARA, dict(w=P + 8)), (PARA, dict(s_stride=2)), (PARA, dict(sa=P + 1)),
    (PARA, dict(y_stride=99)), (PARA, dict(y=P + 1)), (PARA, dict(offsets=P + 1)), (PARA, dict(rows=(1 << 28) + 1)),
    (PARA, dict(stride=1 << 23)), (PARA, dict(k=1 << 23)),
    (OK, dict(rows=0, a=None)), (OK, dict(n=0, w=None)),
])
def test_matmul_refuses(want, kw):
    a = dict(a=P, stride=0, sa=P, s_stride=0, rows=50, groups=4, offsets=P, owner=None, w=P, sw=P, experts=4, n=100, k=300, kind=1, y=P, type=BF16,
             y_stride=0, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdBlockMatmul(*a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (PTR, dict(stream=None)), (PTR, dict(dy=None)), (PTR, dict(sdy=None)), (PTR, dict(x=None)), (PTR, dict(sx=None)), (PTR, dict(dw=None)),
    (NOT_SUPPORT, dict(type=INT8)), (NOT_SUPPORT, dict(kind=0)), (PARA, dict(groups=0)), (PARA, dict(experts=4097)), (PARA, dict(offsets=None)),
    (PARA, dict(columns=384)), (PARA, dict(columns=513)), (PARA, dict(columns=1 << 23)), (PARA, dict(dy=P + 8)), (PARA, dict(dw=P + 1)), (OK, dict(n=0)), (OK, dict(k=0)),
])
def test_grad_weight_refuses(want, kw):
    a = dict(dy=P, sdy=P, x=P, sx=P, columns=512, rows=50, n=100, k=300, kind=1, groups=4, offsets=P, owner=None, experts=4, dw=P, type=BF16, add=0, stream=N)
    a.update(kw)
    assert H.lib().HcclAmdBlockMatmulGradWeight(*a.values()) == want


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("tokens,experts,topk", [(1, 1, 1), (5, 4, 2), (7, 9, 9), (11, 16, 3)])
def test_reference_route_gradient_against_differences(tokens, experts, topk, renorm):
    rng = np.random.default_rng(tokens * 100 + experts)
    # logits far enough apart that no step changes a choice
    x = np.stack([rng.permutation(experts) * 0.3 for _ in range(tokens)]) + rng.uniform(0, 0.1, (tokens, experts))
    mask = np.ones(tokens, np.uint8)
    if tokens > 4:
        mask[2] = 0
        x[2, 0] = np.nan
    dw, dl = rng.standard_normal((tokens, topk)), 1.7
    base = ref.route(x, topk, renorm, mask, 0.3)
    got, _ = ref.route_grad(base, topk, renorm, 0.3, dw, dl)

    def value(x):
        r = ref.route(x, topk, renorm, mask, 0.3)
        assert np.array_equal(r["expert"], base["expert"])
        return (r["weights"] * dw).sum() + dl * r["loss"]

    h = 1e-5
    for t in range(tokens):
        for e in range(experts):
            step = np.zeros_like(x)
            step[t, e] = h
            slope = (value(x + step) - value(x - step)) / (2 * h)
            # (third derivatives of a softmax stay below 1 times the gradients given; cancellation costs 2^-53 / h)
            assert abs(slope - got[t, e]) < 1e-8 * (1 + np.abs(dw).sum())


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_reference_of_many_tokens_is_the_reference(renorm, masked):
    rng = np.random.default_rng(21)
    x = rng.integers(-4, 4, (60, 9)) * 0.5                   # ties everywhere, zeros of both signs
    x[x == 0] *= rng.choice([-1.0, 1.0], (x == 0).sum())
    mask = (rng.random(60) > 0.3).astype(np.uint8) if masked else None
    dw, dl = rng.standard_normal((60, 4)), -0.7
    want = ref.route(x, 4, renorm, mask, 0.3)
    grad, size = ref.route_grad(want, 4, renorm, 0.3, dw, dl)
    got, got_grad, got_size = ref.route_finite(x, 4, renorm, mask, 0.3, dw, dl)
    for k in ("expert", "row_of", "counts", "offsets"):
        assert np.array_equal(got[k], want[k]), k
    for a, b in ((got["weights"], want["weights"]), (got["loss"], want["loss"]), (got_grad, grad), (got_size, size)):
        assert np.allclose(a, b, rtol=1e-13, atol=1e-15)


def test_reference_scales():
    """The least power of two that brings a maximum to 448 or below, at the powers' edges; floats next to them."""
    tops = []
    for p in (-96, -30, -1, 0, 8, 9, 100, 127):
        for m in (1.0, 1.75, np.nextafter(np.float32(1.75), np.float32(2)), np.nextafter(np.float32(1.75), np.float32(1)), 1.9999999):
            tops.append(np.float32(m) * np.float32(2.0 ** p))
    tops = np.array(tops, np.float32)
    stored, times, value = ref.block_scale(tops, ref.E8M0)
    assert (tops.astype(np.float64) <= 448 * value).all() and (tops.astype(np.float64) > 224 * value).all()
    assert np.array_equal(times.astype(np.float64) * value, np.ones(len(tops)))
    assert ref.block_scale(np.float32([0]), ref.E8M0)[0][0] == 127 - 96 - 8


@pytest.mark.parametrize("stride", [2 ** 64 - 1024, 2 ** 63, 2 ** 40 + 16])
def test_strides_that_no_memory_has(stride):
    """What a negative number becomes on its way to an unsigned one, and anything else beyond 2^40, is refused and not followed."""
    calls = [("HcclAmdExpertRoute", (P, BF16, 100, 64, 0, 8, 0, None, 1.0, P, P, P, P, P, P, P, 1 << 30, N), (4,)),
             ("HcclAmdExpertRouteGrad", (P, BF16, 100, 64, 0, 8, 0, None, 1.0, P, P, P, P, P, 0, N), (4, 14)),
             ("HcclAmdExpertPack", (P, BF16, 10, 300, 0, 2, P, 1, P, 20, 0, P, 0, N), (4, 10, 12)),
             ("HcclAmdExpertPack", (P, BF16, 10, 300, 0, 2, P, 0, P, 20, 0, None, 0, N), (4, 10)),
             ("HcclAmdExpertCombine", (P, BF16, 20, 300, 0, 10, 2, P, P, P, 0, N), (4, 10)),
             ("HcclAmdExpertCombineGrad", (P, 0, P, FP16, 20, 300, 0, 10, 2, P, P, P, 0, P, N), (1, 6, 12)),
             ("HcclAmdBlockQuantWeights", (P, BF16, 2, 300, 100, 0, 1, P, P, P, P, N), (5,)),
             ("HcclAmdBlockQuantColumns", (P, BF16, 600, 100, 0, 4, P, 1, P, 1024, P, N), (4,)),
             ("HcclAmdBlockMatmul", (P, 0, P, 0, 50, 4, P, None, P, P, 4, 100, 300, 1, P, BF16, 0, N), (1, 3, 16))]
    for fn, args, at in calls:
        for i in at:
            assert args[i] == 0
            assert getattr(H.lib(), fn)(*args[:i], stride, *args[i + 1:]) == PARA, (fn, i)


def test_grad_weight_refuses_groups_without_weights():
    """Group g uses weights g: more groups than weights are refused, as the product refuses them."""
    for fn, args in (("HcclAmdBlockMatmulGradWeight", (P, P, P, P, 1024, 50, 100, 300, 1, 5, P, None, 4, P, BF16, 0, N)),
                     ("HcclAmdBlockMatmul", (P, 0, P, 0, 50, 5, P, None, P, P, 4, 100, 300, 1, P, BF16, 0, N))):
        assert getattr(H.lib(), fn)(*args) == PARA


@pytest.mark.parametrize("rows,groups,n", [(1 << 28, 1, 257), ((1 << 28) - 1, 4096, 200), (1 << 16, 4096, 128 * 1100)])
def test_matmul_refuses_more_tiles_than_a_launch_holds(rows, groups, n):
    assert (rows // 128 + min(rows, groups)) * -(-n // 128) > 1 << 22
    assert H.lib().HcclAmdBlockMatmul(P, 0, P, 0, rows, groups, P, None if groups == 1 else P, P, P, 4, n, 128, 1, P, BF16, 0, N) == PARA


def test_native_calls_and_ctypes_refuse_alike():
    """The mirror's two ways to a call give the same answers; what the native one does not recognise it leaves alone."""
    L = H.lib()
    pack = (P, BF16, 10, 300, 0, 2, P, 1, P, 20, 0, P, 0, N)
    for at, value in ((13, None), (0, None), (1, INT8), (5, 0), (6, None), (10, 392), (11, P + 2)):
        args = pack[:at] + (value,) + pack[at + 1:]
        code = L.HcclAmdExpertPack(*args)
        assert code in (PARA, PTR, NOT_SUPPORT)
        assert H._expert(2, *args) in ((code,) if H._expert is not H._through_ctypes else (-1,))
        with pytest.raises(H.HcclError) as e:
            H._expert_call(2, *args)
        assert e.value.code == code
    if H._expert is not H._through_ctypes:
        refused = (P, BF16, 0, 64, 0, 8, 0, None, 0.01, None, None, None, None, None, None, None, 0, N)
        assert H._expert(0, *refused) == PTR
        for args in (refused[:-1], refused + (1,), refused[:8] + (1,) + refused[9:], ("1",) + refused[1:], refused[:2] + (1.0,) + refused[3:]):
            assert H._expert(0, *args) == -1
        assert H._expert(9) == -1 and H._expert() == -1 and H._expert("0") == -1
        assert H._expert(0, ctypes.c_void_p(P), *refused[1:]) == PTR


def test_native_module_is_built_again_when_a_prototype_changes(monkeypatch, tmp_path):
    """It calls the library by the prototypes in the public headers: newer than the module, any of them has it compiled again."""
    spec = importlib.util.spec_from_file_location("hccl_build_under_test", os.path.join(ROOT, "cann-hccl_amd", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    module, ran = tmp_path / "module.so", []
    module.write_bytes(b"")
    monkeypatch.setattr(build, "RANKS", str(module))
    monkeypatch.setattr(build, "_run", ran.append)
    times = {}
    monkeypatch.setattr(build.os.path, "getmtime", lambda p: times.get(os.path.basename(p), 1.0))
    times["module.so"] = 2.0
    build.build_ranks()
    assert not ran
    for newer in ("pyranks.cc", "hccl_amd_experts.h", "hccl.h", "hccl_types.h"):
        times[newer] = 3.0
        build.build_ranks()
        assert len(ran) == 1 and ran.pop()[0] == "g++", newer
        del times[newer]
