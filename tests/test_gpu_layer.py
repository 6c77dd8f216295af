"""Norm, scored router, gate and gradient clipping on the GPU against 64-bit references: sizes from one row up, odd and ragged ones, strides and
alignments, masks that leave nothing, NaN and infinities, the bytes around every output untouched, replays of captured graphs, calls in place, on two
streams at once and far into memory.  Choices, counts, rows, biases and 8-bit values are compared exactly where their inputs are exact; sums within bounds
that count roundings (experts_reference.close adds half a unit of the output's type)."""
import numpy as np
import pytest
import torch

import experts_reference as eight
import layer_reference as ref
from experts_reference import U, close, up128
from hccl_loader import load
from test_gpu_experts import Out, dt

pytestmark = pytest.mark.gpu
H = load()
TYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
KIND = {"none": 0, "fp32": 1, "e8m0": 2}


@pytest.fixture(scope="module")
def stream():
    return torch.cuda.Stream()


def ready():
    torch.cuda.synchronize()


def f64(t):
    return t.detach().cpu().double().numpy()


def near(got, want, bound, dtype=torch.float32):
    """close(), equal infinities being equal."""
    same = np.isinf(want) & (got == want)
    return close(np.where(same, 0, got), np.where(same, 0, want), np.where(same, 0, bound), dtype)


def draw(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def put(values, stride=0, shift=0):
    return Out(values.shape[0], values.shape[1], values.dtype, stride, shift).fill(values.cuda())


def check_eight(codes, scales, kind, want, off):
    """8-bit rows of values that are `off` (relative) from want [rows, width] in 32 bits."""
    rows, width = want.shape
    W = up128(width)
    want = np.pad(want, ((0, 0), (0, W - width))).reshape(rows, W // 128, 128)
    fine = np.isfinite(want)
    top = np.maximum(np.where(fine, np.abs(want), 0).max(2), 2.0 ** -96)
    value = np.exp2(scales.astype(np.float64) - 127) if kind == 2 else scales.astype(np.float64)
    if kind == 1:
        assert (np.abs(value - top / 448) <= (off + 4 * U) * top / 448).all()
    else:
        assert (top * (1 - off) <= 448 * value).all() and (top * (1 + off) >= 224 * value).all()
    got = eight.from_fp8(codes).reshape(rows, W // 128, 128)
    assert np.array_equal(np.isnan(got), ~fine)
    # half a step of three bits of mantissa, or of the smallest step, 2^-9
    room = (2.0 ** -4 + 2 * off) * np.abs(want) + (2.0 ** -10 + off * 448) * value[..., None]
    assert (np.abs(got * value[..., None] - want)[fine] <= room[fine]).all()


# ---- norm ---------------------------------------------------------------------------------------------------------------------

def run_norm(stream, x, r, gain, eps, kind=0, want_sum=True, want_y=True, strides=(0, 0, 0, 0, 0, 0), shift=0):
    rows, width = x.shape
    xs, rs = put(x, strides[0], shift), None if r is None else put(r, strides[1], shift)
    total, y = (Out(rows, width, x.dtype, strides[2], shift) if want_sum else None), (Out(rows, width, x.dtype, strides[3], shift) if want_y else None)
    q = Out(rows, up128(width), torch.uint8, strides[4]) if kind else None
    scales = Out(rows, up128(width) // 128, torch.float32 if kind == 1 else torch.uint8, strides[5]) if kind else None
    g = None if gain is None else gain.cuda()
    p = lambda o: None if o is None else o.ptr  # noqa: E731
    ready()
    H.norm_rows(xs.ptr, dt(x.dtype), rows, width, stream.cuda_stream, residual=p(rs), gain=None if g is None else g.data_ptr(),
                gain_dtype=dt(x.dtype if g is None else g.dtype), epsilon=eps, sum=p(total), y=p(y), scale_type=kind, q=p(q), scales=p(scales), x_stride=strides[0],
                residual_stride=strides[1], sum_stride=strides[2], y_stride=strides[3], q_stride=strides[4], scale_stride=strides[5])
    stream.synchronize()
    return total, y, q, scales


def check_norm(x, r, gain, eps, kind, out):
    total, y, q, scales = out
    s, want = ref.norm(f64(x), None if r is None else f64(r), None if gain is None else f64(gain), np.float64(np.float32(eps)))
    if total is not None:
        assert near(total.numpy(), s, U * np.abs(s), x.dtype)
    # the sum is off by U of itself, and with it the root; the root, two products: half a unit each
    off = 6 * U
    if y is not None:
        assert near(y.numpy(), want, off * np.abs(want), x.dtype)
    if kind:
        check_eight(q.get().cpu().numpy(), scales.get().cpu().numpy(), kind, want, off)


NORMS = [
    # rows, width, type, gain's type, residual, 8 bits
    (1, 1, "fp32", "fp32", True, "none"), (1, 8192, "bf16", "bf16", True, "fp32"), (3, 128, "fp16", "fp32", True, "e8m0"), (5, 127, "bf16", "fp32", False, "fp32"),
    (7, 129, "fp32", None, True, "e8m0"), (130, 512, "bf16", "bf16", True, "none"), (129, 513, "fp16", "fp16", True, "fp32"), (65, 1000, "bf16", "bf16", False, "e8m0"),
    (33, 1024, "fp32", "fp32", True, "fp32"), (17, 1025, "bf16", "fp32", True, "none"), (300, 2001, "fp16", "fp16", True, "fp32"), (9, 2048, "bf16", "bf16", True, "fp32"),
    (5, 4096, "fp16", None, True, "e8m0"), (4, 4097, "fp32", "fp32", True, "fp32"), (6, 8191, "bf16", "bf16", True, "none"), (2, 8200, "bf16", "fp32", True, "fp32"),
    (3, 16384, "fp32", "fp32", False, "e8m0"), (2, 16385, "bf16", "bf16", True, "fp32"), (2, 32768, "fp32", "fp32", True, "fp32"), (2, 32767, "fp16", "fp16", True, "none"),
]


@pytest.mark.parametrize("rows,width,dtype,gain,residual,kind", NORMS)
def test_norm(stream, rows, width, dtype, gain, residual, kind):
    print("norm", rows, width, dtype, gain, residual, kind, flush=True)
    t = TYPE[dtype]
    x, r = draw(1, rows, width, dtype=t), draw(2, rows, width, dtype=t, scale=3.0) if residual else None
    g = None if gain is None else (1 + draw(3, width, scale=0.2)).to(TYPE[gain])
    out = run_norm(stream, x, r, g, 1e-6, KIND[kind])
    check_norm(x, r, g, 1e-6, KIND[kind], out)
    if dtype == "fp32" and kind != "none":
        # y is there in 32 bits: its 8-bit rows are known to the last bit
        codes, stored, _ = eight.quant_rows(out[1].get().cpu().numpy(), KIND[kind])
        assert eight.same_codes(out[2].get().cpu().numpy(), codes) and np.array_equal(out[3].get().cpu().numpy(), stored)


@pytest.mark.parametrize("shift,strides", [(0, (304, 312, 320, 328, 400, 5)), (1, (301, 303, 305, 307, 384, 3)), (3, (0, 0, 0, 0, 0, 0))])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_norm_strides(stream, dtype, shift, strides):
    x, r, g = draw(1, 37, 300, dtype=TYPE[dtype]), draw(2, 37, 300, dtype=TYPE[dtype]), draw(3, 300)
    check_norm(x, r, g, 1e-5, 1, run_norm(stream, x, r, g, 1e-5, 1, strides=strides, shift=shift))


def test_norm_each_output_alone(stream):
    x, r = draw(1, 9, 640, dtype=torch.bfloat16), draw(2, 9, 640, dtype=torch.bfloat16)
    for want_sum, want_y, kind in ((True, False, 0), (False, True, 0), (False, False, 1), (False, False, 2), (True, False, 2)):
        check_norm(x, r, None, 0.0, kind, run_norm(stream, x, r, None, 0.0, kind, want_sum, want_y))


def test_norm_far_values(stream):
    """Squares beyond the range of 32 bits on both sides, zeros, infinities and NaN in their own rows alone."""
    x = draw(1, 8, 300)
    x[0] *= 1e25
    x[1] *= 1e-25
    x[2] = 0
    x[3, 7] = float("inf")
    x[4, 9] = float("nan")
    x[5] = 0
    x[5, 299] = 1e-30
    out = run_norm(stream, x, None, None, 0.0, 1)
    s, want = ref.norm(f64(x), None, None, 0.0)
    assert np.isnan(want[2]).all() and np.isnan(want[3, 7]) and np.isnan(want[4]).all()
    check_norm(x, None, None, 0.0, 1, out)
    zero = run_norm(stream, torch.zeros(3, 300), None, None, 1e-6, 2)
    assert not zero[1].numpy().any() and not zero[2].numpy().any() and (zero[3].numpy() == 127 - 96 - 8).all()


def grad_norm(stream, dy, s, gain, eps, dsum, want_dx=True, want_gain=True, start=None, stride=0, shift=0):
    rows, width = s.shape
    dys, ss = put(dy, stride, shift), put(s, stride, shift)
    ds = None if dsum is None else put(dsum, stride, shift)
    dx, dgain = Out(rows, width, s.dtype, stride, shift) if want_dx else None, Out(1, width, torch.float32) if want_gain else None
    if start is not None:
        dgain.fill(start[None].cuda())
    need = H.norm_rows_grad_workspace(rows, width)
    work = torch.full((need + 64,), 0xC3, dtype=torch.uint8, device="cuda")
    g = None if gain is None else gain.cuda()
    ready()
    H.norm_rows_grad(dys.ptr, ss.ptr, dt(s.dtype), rows, width, dx.ptr if want_dx else None, stream.cuda_stream, gain=None if g is None else g.data_ptr(),
                     gain_dtype=dt(s.dtype if g is None else g.dtype), epsilon=eps, sum_grad=None if ds is None else ds.ptr, gain_grad=dgain.ptr if want_gain else None,
                     accumulate=start is not None, workspace=work.data_ptr(), workspace_bytes=need, y_grad_stride=stride, sum_stride=stride, sum_grad_stride=stride,
                     x_grad_stride=stride)
    stream.synchronize()
    assert bool((work[need:] == 0xC3).all())
    return dx, dgain


def check_norm_grad(dy, s, gain, eps, dsum, start, dx, dgain):
    want, want_gain, size, gain_size = ref.norm_grad(f64(dy), f64(s), None if gain is None else f64(gain), np.float64(np.float32(eps)), None if dsum is None else f64(dsum))
    if dx is not None:
        assert near(dx.numpy(), want, 10 * U * size, s.dtype)
    if dgain is not None:
        start = 0 if start is None else f64(start)
        rows = s.shape[0]
        assert near(dgain.numpy()[0], want_gain + start, (rows + 6) * U * gain_size + U * np.abs(start))
        # as a whole: rounding errors of sums in 32 bits are independent, a sum kept in fewer bits is far outside
        if rows > 8:
            assert np.linalg.norm(dgain.numpy()[0] - want_gain - start) <= 8 * rows ** 0.5 * U * np.linalg.norm(gain_size)


@pytest.mark.parametrize("rows,width,dtype,gain,residual,kind", NORMS + [(5003, 2001, "fp16", "fp16", False, "none"), (2100, 256, "bf16", "fp32", True, "none"),
                                                                        (0, 100, "bf16", "bf16", True, "none"), (1025, 4096, "bf16", "bf16", True, "none")])
def test_norm_grad(stream, rows, width, dtype, gain, residual, kind):
    print("norm grad", rows, width, dtype, gain, residual, flush=True)
    t = TYPE[dtype]
    dy, s, dsum = draw(1, rows, width, dtype=t), draw(2, rows, width, dtype=t, scale=2.0), draw(3, rows, width, dtype=t) if residual else None
    g = None if gain is None else (1 + draw(4, width, scale=0.2)).to(TYPE[gain])
    start = draw(5, width) if rows % 2 else None
    dx, dgain = grad_norm(stream, dy, s, g, 1e-6, dsum, start=start)
    check_norm_grad(dy, s, g, 1e-6, dsum, start, dx, dgain)
    again = grad_norm(stream, dy, s, g, 1e-6, dsum, start=start)
    assert torch.equal(again[0].get(), dx.get()) and torch.equal(again[1].get(), dgain.get())


def test_norm_grad_parts(stream):
    dy, s, g = draw(1, 50, 300, dtype=torch.bfloat16), draw(2, 50, 300, dtype=torch.bfloat16), draw(3, 300)
    for want_dx, want_gain, stride, shift in ((True, False, 0, 0), (False, True, 0, 0), (True, True, 304, 0), (True, True, 301, 1)):
        dx, dgain = grad_norm(stream, dy, s, g, 1e-6, None, want_dx, want_gain, stride=stride, shift=shift)
        check_norm_grad(dy, s, g, 1e-6, None, None, dx, dgain)


def test_norm_in_place(stream):
    """The sum in the residual's or x's place, the gradient in that of either gradient it is made from."""
    t = torch.bfloat16
    x, r, dy = (draw(i, 70, 1000, dtype=t).cuda() for i in range(3))
    outs = []
    for place in ("none", "residual", "x"):
        a, b, s, y = x.clone(), r.clone(), torch.empty_like(x), torch.empty_like(x)
        to = {"none": s, "residual": b, "x": a}[place]
        ready()
        H.norm_rows(a.data_ptr(), dt(t), 70, 1000, stream.cuda_stream, residual=b.data_ptr(), sum=to.data_ptr(), y=y.data_ptr())
        stream.synchronize()
        outs.append((to.clone(), y))
    assert all(torch.equal(outs[0][i], o[i]) for o in outs[1:] for i in range(2))
    outs = []
    for place in ("none", "y_grad", "sum_grad"):
        d, e, dx = dy.clone(), r.clone(), torch.empty_like(x)
        to = {"none": dx, "y_grad": d, "sum_grad": e}[place]
        ready()
        H.norm_rows_grad(d.data_ptr(), x.data_ptr(), dt(t), 70, 1000, to.data_ptr(), stream.cuda_stream, sum_grad=e.data_ptr())
        stream.synchronize()
        outs.append(to.clone())
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- gate ---------------------------------------------------------------------------------------------------------------------

def rel_gate(g):
    # the power's argument is rounded (2 U of itself), power, sum, reciprocal and three products: a unit or half one each
    return (3 * np.abs(g) + 10) * U


GATES = [(1, 1, "fp32", "none"), (1, 128, "bf16", "fp32"), (3, 127, "fp16", "e8m0"), (5, 129, "bf16", "fp32"), (8, 512, "fp32", "fp32"), (65, 513, "bf16", "none"),
         (300, 1000, "fp16", "fp32"), (33, 2048, "bf16", "e8m0"), (17, 4095, "bf16", "fp32"), (2, 20001, "fp32", "e8m0")]


@pytest.mark.parametrize("rows,width,dtype,kind", GATES)
@pytest.mark.parametrize("used", [None, 0.6])
def test_gate(stream, rows, width, dtype, kind, used):
    print("gate", rows, width, dtype, kind, used, flush=True)
    t, k = TYPE[dtype], KIND[kind]
    h = draw(7, rows, 2 * width, dtype=t, scale=3.0)
    n = rows if used is None else int(rows * used)
    on = None if used is None else torch.tensor([n], dtype=torch.int32, device="cuda")
    ins = put(h)
    out = Out(rows, up128(width) if k else width, torch.uint8 if k else t)
    scales = Out(rows, up128(width) // 128, torch.float32 if k == 1 else torch.uint8) if k else None
    ready()
    H.expert_gate(ins.ptr, dt(t), rows, width, out.ptr, stream.cuda_stream, used=None if on is None else on.data_ptr(), scale_type=k, scales=scales.ptr if k else None)
    stream.synchronize()
    g, u = f64(h)[:n, :width], f64(h)[:n, width:]
    want = ref.gate(g, u)
    got = out.get().cpu()
    assert bool((got[n:].contiguous().view(torch.uint8) == 0xA5).all())
    if not k:
        assert near(got[:n].double().numpy(), want, rel_gate(g) * np.abs(want), t)
    else:
        assert bool((scales.get().cpu()[n:].contiguous().view(torch.uint8) == 0xA5).all())
        off = float(rel_gate(np.abs(g).max() if g.size else 0.0))
        check_eight(got[:n].numpy(), scales.get().cpu().numpy()[:n], k, want, off)


@pytest.mark.parametrize("rows,width,dtype,kind", GATES)
@pytest.mark.parametrize("used", [None, 0.6])
def test_gate_grad(stream, rows, width, dtype, kind, used):
    print("gate grad", rows, width, dtype, used, flush=True)
    t = TYPE[dtype]
    h, da = draw(7, rows, 2 * width, dtype=t, scale=3.0), draw(8, rows, width, dtype=t)
    n = rows if used is None else int(rows * used)
    on = None if used is None else torch.tensor([n], dtype=torch.int32, device="cuda")
    for stride, shift, want_h, want_a in ((0, 0, True, True), (2 * width + 5, 1, True, True), (0, 0, False, True), (0, 0, True, False)):
        ins, das = put(h, stride, shift), put(da, stride, shift)
        dh, a = Out(rows, 2 * width, t, stride, shift), Out(rows, width, t, stride, shift)
        ready()
        H.expert_gate_grad(das.ptr if want_h else None, ins.ptr, dt(t), rows, width, dh.ptr if want_h else None, stream.cuda_stream,
                           used=None if on is None else on.data_ptr(), out=a.ptr if want_a else None, out_grad_stride=stride, h_stride=stride,
                           h_grad_stride=stride, out_stride=stride)
        stream.synchronize()
        g, u, d = f64(h)[:n, :width], f64(h)[:n, width:], f64(da)[:n]
        dg, du, dg_size, du_size = ref.gate_grad(d, g, u)
        got, got_a = dh.get().cpu(), a.get().cpu()
        first = n if want_h else 0
        assert bool((got[first:].contiguous().view(torch.uint8) == 0xA5).all())
        first = n if want_a else 0
        assert bool((got_a[first:].contiguous().view(torch.uint8) == 0xA5).all())
        if want_h:
            rel = rel_gate(g) + 6 * U
            assert near(got[:n, :width].double().numpy(), dg, rel * dg_size, t) and near(got[:n, width:].double().numpy(), du, rel * du_size, t)
        if want_a:
            want = ref.gate(g, u)
            assert near(got_a[:n].double().numpy(), want, rel_gate(g) * np.abs(want), t)


@pytest.mark.parametrize("count,n", [(-5, 0), (0, 0), (7, 7), (1000, 9)])
def test_gate_used(stream, count, n):
    """A count on the device that is not within the rows is brought there; nothing behind it is written."""
    h, da = draw(1, 9, 600, dtype=torch.bfloat16), draw(2, 9, 300, dtype=torch.bfloat16)
    on = torch.tensor([count], dtype=torch.int32, device="cuda")
    ins, das, out, dh = put(h), put(da), Out(9, 300, torch.bfloat16), Out(9, 600, torch.bfloat16)
    ready()
    H.expert_gate(ins.ptr, dt(h.dtype), 9, 300, out.ptr, stream.cuda_stream, used=on.data_ptr())
    H.expert_gate_grad(das.ptr, ins.ptr, dt(h.dtype), 9, 300, dh.ptr, stream.cuda_stream, used=on.data_ptr())
    stream.synchronize()
    for o in (out, dh):
        v = o.get().cpu()
        assert bool((v[n:].contiguous().view(torch.uint8) == 0xA5).all())
        assert bool(torch.isfinite(v[:n].float()).all()) and not bool((v[:n].contiguous().view(torch.uint8) == 0xA5).all(1).any())


def test_gate_far_values(stream):
    """Gates so far out that the power overflows or vanishes, zeros, infinities, NaN: what the formula says, in their own values alone."""
    g = torch.tensor([[0.0, -0.0, 90.0, -90.0, 200.0, -200.0, 3e38, -3e38, float("inf"), float("nan"), 1e-30, -1e-30]])
    h = torch.cat([g, torch.full_like(g, 2.0)], 1)
    da = torch.ones_like(g)
    ins, das, out, dh = put(h), put(da), Out(1, 12, torch.float32), Out(1, 24, torch.float32)
    ready()
    H.expert_gate(ins.ptr, dt(h.dtype), 1, 12, out.ptr, stream.cuda_stream)
    H.expert_gate_grad(das.ptr, ins.ptr, dt(h.dtype), 1, 12, dh.ptr, stream.cuda_stream)
    stream.synchronize()
    with np.errstate(all="ignore"):
        want = ref.gate(f64(g), np.full((1, 12), 2.0))
        _, du, _, _ = ref.gate_grad(np.ones((1, 12)), f64(g), np.full((1, 12), 2.0))
        bound = np.where(np.isfinite(want), rel_gate(np.minimum(np.abs(f64(g)), 110)) * np.abs(want), 0) + 2.0 ** -118
    assert np.array_equal(np.isposinf(out.numpy()), np.isposinf(want)) or (out.numpy()[0, 6] == np.inf)     # 2 * 3e38 is beyond 32 bits
    fine = [0, 1, 2, 3, 4, 5, 7, 10, 11]
    assert near(out.numpy()[0, fine], want[0, fine], bound[0, fine]) and np.isnan(out.numpy()[0, 9])
    assert near(dh.numpy()[0, 12:][fine], du[0, fine], bound[0, fine])
    assert np.isfinite(dh.numpy()[0, :9][[0, 1, 2, 3, 4, 5, 10 - 4]]).all()


@pytest.mark.parametrize("kind", [1, 2])
def test_gate_not_finite_in_8_bits(stream, kind):
    """Infinities and NaN become the type's NaN in their own place and leave their block's scale alone."""
    g, u = draw(1, 40, 300), draw(2, 40, 300)
    u[3, 5], u[3, 290], g[7, 130], u[9], g[11] = float("inf"), float("nan"), float("nan"), float("-inf"), float("inf")
    h = torch.cat([g, u], 1)
    ins, q = put(h), Out(40, 384, torch.uint8)
    scales = Out(40, 3, torch.float32 if kind == 1 else torch.uint8)
    ready()
    H.expert_gate(ins.ptr, dt(h.dtype), 40, 300, q.ptr, stream.cuda_stream, scale_type=kind, scales=scales.ptr)
    stream.synchronize()
    with np.errstate(all="ignore"):
        want = ref.gate(f64(g), f64(u))
    assert (~np.isfinite(want)).sum() >= 600
    check_eight(q.get().cpu().numpy(), scales.get().cpu().numpy(), kind, want, float(rel_gate(5.0)))


def test_gate_in_place(stream):
    h, da = draw(1, 40, 1300, dtype=torch.float16).cuda(), draw(2, 40, 650, dtype=torch.float16).cuda()
    dh, a = torch.empty_like(h), torch.empty_like(da)
    h2, da2 = h.clone(), da.clone()
    ready()
    H.expert_gate_grad(da.data_ptr(), h.data_ptr(), dt(h.dtype), 40, 650, dh.data_ptr(), stream.cuda_stream, out=a.data_ptr())
    H.expert_gate_grad(da2.data_ptr(), h2.data_ptr(), dt(h.dtype), 40, 650, h2.data_ptr(), stream.cuda_stream, out=da2.data_ptr())
    stream.synchronize()
    assert torch.equal(dh, h2) and torch.equal(a, da2)


# ---- scored router --------------------------------------------------------------------------------------------------------------

def run_route(stream, x, kind, bias, groups, kept, top, topk, renorm, scale, mask, dw=None, stride=0, shift=0):
    T, E = x.shape
    score = H.HCCL_AMD_SCORE_SIGMOID if kind == "sigmoid" else H.HCCL_AMD_SCORE_SOFTMAX
    ins = put(x, stride, shift)
    o = {"expert": Out(T, topk, torch.int32), "weights": Out(T, topk, torch.float32), "row_of": Out(T, topk, torch.int32), "counts": Out(1, E + 1, torch.int32),
         "offsets": Out(1, E + 1, torch.int32)}
    need = H.expert_route_scored_workspace(T, E)
    work = torch.full((need + 64,), 0xC3, dtype=torch.uint8, device="cuda")
    b = None if bias is None else torch.from_numpy(bias).cuda()
    m = None if mask is None else torch.from_numpy(mask).cuda()
    grad, g = Out(T, E, x.dtype, stride, shift), None if dw is None else torch.from_numpy(dw.astype(np.float32)).cuda()
    ready()
    H.expert_route_scored(ins.ptr, dt(x.dtype), T, E, topk, score, o["expert"].ptr, o["weights"].ptr, o["row_of"].ptr, o["counts"].ptr, o["offsets"].ptr,
                          work.data_ptr() if need else None, need, stream.cuda_stream, bias=None if b is None else b.data_ptr(), groups=groups, groups_kept=kept,
                          group_top=top, renorm=renorm, weight_scale=scale, mask=None if m is None else m.data_ptr(), stride=stride)
    if dw is not None:
        H.expert_route_scored_grad(ins.ptr, dt(x.dtype), T, E, topk, score, o["expert"].ptr, g.data_ptr(), grad.ptr, stream.cuda_stream, renorm=renorm,
                                   weight_scale=scale, stride=stride, grad_stride=stride)
    stream.synchronize()
    assert bool((work[need:] == 0xC3).all())
    return {k: v.numpy() for k, v in o.items()}, grad.numpy() if dw is not None else None


def check_route(x, kind, bias, groups, kept, top, topk, renorm, scale, mask, dw, got, grad):
    dtype, x = x.dtype, f64(x)
    T, E = x.shape
    r = ref.route(x, kind, None if bias is None else bias.astype(np.float64), groups, kept, top, topk, renorm, scale, mask)
    for k in ("expert", "row_of"):
        assert np.array_equal(got[k], r[k]), k
    assert np.array_equal(got["counts"][0], r["counts"]) and np.array_equal(got["offsets"][0], r["offsets"])
    fine = np.where(np.isfinite(x), np.abs(x), 0)
    far = np.minimum(2 * fine.max(1, keepdims=True), 200.0) if E else np.zeros((T, 1))
    # arguments of powers are off by 2 U of themselves (differences of logits, and logarithms of scores as large); sums over the experts by E + 1
    rel = (3 * far + E + 24) * U
    assert near(got["weights"], r["weights"], rel * np.abs(np.nan_to_num(r["weights"])) + 1e-37)
    if dw is not None:
        want, size = ref.route_grad(x, r, kind, topk, renorm, scale, dw)
        assert near(grad, want, 3 * rel * np.nan_to_num(size) + 1e-37, dtype)


ROUTES = [
    # tokens, experts, groups, kept, top, topk, type
    (1, 1, 1, 1, 1, 1, "fp32"), (1, 256, 8, 4, 2, 8, "bf16"), (5, 8, 2, 1, 1, 2, "fp16"), (16, 64, 8, 3, 2, 6, "bf16"), (17, 60, 4, 2, 2, 6, "fp32"),
    (33, 126, 9, 4, 1, 5, "fp16"), (70, 160, 8, 3, 2, 16, "fp32"), (100, 129, 3, 2, 2, 7, "bf16"), (200, 255, 5, 5, 2, 3, "fp32"), (9, 257, 1, 1, 1, 8, "bf16"),
    (13, 1024, 64, 7, 2, 16, "fp32"), (6, 1000, 10, 1, 2, 10, "fp16"), (300, 256, 1, 1, 2, 8, "fp32"), (64, 128, 64, 5, 2, 4, "bf16"), (40, 12, 12, 5, 2, 5, "fp32"),
    (21, 1024, 2, 1, 2, 8, "fp32"), (7, 1020, 4, 2, 2, 16, "bf16"), (4, 1024, 1, 1, 1, 16, "bf16"),
]


@pytest.mark.parametrize("tokens,experts,groups,kept,top,topk,dtype", ROUTES)
@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route(stream, tokens, experts, groups, kept, top, topk, dtype, kind, renorm):
    print("route", tokens, experts, groups, kept, top, topk, dtype, kind, renorm, flush=True)
    x = draw(tokens + experts, tokens, experts, dtype=TYPE[dtype], scale=2.0)
    rng = np.random.default_rng(experts)
    bias = (rng.standard_normal(experts) * 0.1).astype(np.float32) if tokens % 2 else None
    mask = (rng.random(tokens) > 0.2).astype(np.uint8) if tokens % 3 == 0 else None
    dw = rng.standard_normal((tokens, topk)).astype(np.float32)
    got, grad = run_route(stream, x, kind, bias, groups, kept, top, topk, renorm, 2.5, mask, dw)
    check_route(x, kind, bias, groups, kept, top, topk, renorm, 2.5, mask, dw, got, grad)


@pytest.mark.parametrize("tokens", [0, 16, 17, 512, 513, 1500])
def test_route_many_tokens(stream, tokens):
    x = draw(tokens, tokens, 32, dtype=torch.bfloat16, scale=1.5)
    bias = np.round(np.random.default_rng(1).standard_normal(32) * 20).astype(np.float32) * np.float32(1e-3)
    dw = np.random.default_rng(2).standard_normal((tokens, 3)).astype(np.float32)
    got, grad = run_route(stream, x, "sigmoid", bias, 4, 2, 2, 3, True, 1.0, None, dw)
    check_route(x, "sigmoid", bias, 4, 2, 2, 3, True, 1.0, None, dw, got, grad)


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups,kept,experts", [(1, 1, 64), (8, 3, 64), (8, 3, 256), (5, 2, 40)])
def test_route_ties(stream, kind, groups, kept, experts):
    """Few distinct logits and biases: ties between experts, groups and at every border, to the lowest."""
    rng = np.random.default_rng(groups + experts)
    x = torch.from_numpy(rng.integers(-2, 3, (120, experts)) * 0.5).to(torch.bfloat16)
    x[:10] = 1.0
    for bias in (None, np.zeros(experts, np.float32), (rng.integers(-1, 2, experts) * 0.25).astype(np.float32)):
        got, _ = run_route(stream, x, kind, bias, groups, kept, 2, 6, True, 1.0, None)
        check_route(x, kind, bias, groups, kept, 2, 6, True, 1.0, None, None, got, None)


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
def test_route_next_to_each_other(stream, kind):
    """Scores that differ by less than 32 bits hold: the choice is that of 64 bits."""
    rng = np.random.default_rng(5)
    x = torch.from_numpy((1.0 + rng.integers(0, 3, (200, 64)) * 2.0 ** -23).astype(np.float32))
    x[100:] += torch.from_numpy(rng.integers(0, 2, (100, 64)) * 20.0).float()      # and where a sigmoid is 1 to 32 bits
    bias = np.float32(0.5) + (rng.integers(0, 4, 64) * 2.0 ** -25).astype(np.float32)
    for groups, kept in ((1, 1), (8, 3)):
        got, _ = run_route(stream, x, kind, bias, groups, kept, 2, 8, True, 1.0, None)
        check_route(x, kind, bias, groups, kept, 2, 8, True, 1.0, None, None, got, None)


@pytest.mark.parametrize("tokens,experts,groups,kept,top,topk,dtype", [
    (4097, 30, 5, 2, 2, 4, "fp32"), (5000, 64, 8, 3, 2, 6, "bf16"), (4500, 100, 1, 1, 1, 8, "fp16"), (6001, 128, 4, 2, 1, 8, "bf16"), (4999, 200, 10, 4, 2, 7, "fp32"),
    (5001, 256, 8, 4, 2, 8, "bf16"), (4200, 256, 1, 1, 1, 3, "fp32"), (4100, 256, 8, 4, 2, 12, "bf16"), (70001, 16, 4, 2, 2, 2, "bf16"), (5003, 320, 5, 2, 2, 8, "fp16"),
])
@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("data", ["spread", "close"])
def test_route_large(stream, tokens, experts, groups, kept, top, topk, dtype, kind, data):
    """Every layout for many tokens, several tiles to a workgroup; and scores so close to each other that many choices take 64 bits."""
    print("route large", tokens, experts, groups, kept, top, topk, dtype, kind, data, flush=True)
    x = draw(experts, tokens, experts, dtype=TYPE[dtype], scale=1.5)
    if data == "close":
        # logits of a few values, biases a few steps of 2^-24 apart: next to each other, not equal
        x = torch.round(x.float() * 2).clamp(-2, 2).mul(0.5).to(x.dtype)
        if dtype == "fp32":
            x += draw(9, tokens, experts).sign() * 2.0 ** -21
    rng = np.random.default_rng(topk)
    step = 2.0 ** -24 if data == "close" else 1e-3
    bias = (0.25 + rng.integers(-20, 20, experts) * step).astype(np.float32)
    got, _ = run_route(stream, x, kind, bias, groups, kept, top, topk, True, 1.0, None)
    r = ref.route_many(f64(x), kind, bias.astype(np.float64), groups, kept, top, topk, True, 1.0)
    for k in ("expert", "row_of"):
        assert np.array_equal(got[k], r[k]), (k, int((got[k] != r[k]).any(1).sum()))
    assert np.array_equal(got["counts"][0], r["counts"]) and np.array_equal(got["offsets"][0], r["offsets"])
    assert near(got["weights"], r["weights"], (3 * 2 * np.abs(f64(x)).max() + experts + 24) * U * r["weights"])


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
def test_route_nothing_left(stream, kind):
    """Masked tokens that hold anything, rows of -inf or NaN, groups without an expert, experts that the bias switches off, infinite logits."""
    inf, nan = float("inf"), float("nan")
    x = draw(3, 12, 24)
    x[0] = nan
    x[1] = -inf
    x[2] = nan
    x[3, :6] = -inf
    x[4, 6:] = -inf
    x[5, 1:] = -inf
    x[6, 3] = nan
    x[7, 5] = inf
    x[8] = -300.0
    x[9] = torch.linspace(-1000, -900, 24)
    mask = np.ones(12, np.uint8)
    mask[0] = mask[11] = 0
    x[11] = inf
    off = np.zeros(24, np.float32)
    off[[0, 7]] = -np.inf
    off[8] = np.nan
    dw = np.random.default_rng(1).standard_normal((12, 5)).astype(np.float32)
    for bias in (None, off):
        for renorm in (True, False):
            got, grad = run_route(stream, x, kind, bias, 4, 2, 2, 5, renorm, 1.5, mask, dw)
            finite = [t for t in range(12) if t not in (6, 7)]
            check_route(x, kind, bias, 4, 2, 2, 5, renorm, 1.5, mask, None, got, None)
            r = ref.route(f64(x), kind, bias, 4, 2, 2, 5, renorm, 1.5, mask)
            want, size = ref.route_grad(f64(x), r, kind, 5, renorm, 1.5, dw)
            assert near(grad[finite], want[finite], 2000 * U * size[finite] + 1e-37)
            assert not grad[[0, 1, 2, 11]].any()


@pytest.mark.parametrize("topk", [6, 12])
def test_route_weights_are_a_tokens_own(stream, topk):
    """Scores near the end of 32 bits in one token change no bit of its neighbours' weights."""
    x = draw(8, 64, 32, scale=2.0)
    got, _ = run_route(stream, x, "sigmoid", None, 1, 1, 1, topk, True, 1.0, None)
    x[5::8] = -100 + x[5::8]
    apart, _ = run_route(stream, x, "sigmoid", None, 1, 1, 1, topk, True, 1.0, None)
    others = np.arange(64) % 8 != 5
    assert np.array_equal(got["weights"][others], apart["weights"][others]) and np.array_equal(got["expert"][others], apart["expert"][others])
    check_route(x, "sigmoid", None, 1, 1, 1, topk, True, 1.0, None, None, apart, None)


def test_route_strides_and_shared_words(stream):
    for dtype, stride, shift in (("bf16", 72, 0), ("bf16", 67, 1), ("fp32", 65, 1), ("fp16", 64, 8)):
        x = draw(9, 50, 64, dtype=TYPE[dtype])
        dw = np.random.default_rng(2).standard_normal((50, 4)).astype(np.float32)
        for kind in ("sigmoid", "softmax"):
            got, grad = run_route(stream, x, kind, None, 4, 2, 1, 4, False, 1.0, None, dw, stride, shift)
            check_route(x, kind, None, 4, 2, 1, 4, False, 1.0, None, dw, got, grad)


def test_route_grad_many_tokens(stream):
    """Gradients of more tokens than workgroups take at once, experts in every layout."""
    for experts, topk, dtype in ((64, 4, torch.bfloat16), (200, 8, torch.float32), (500, 3, torch.float16)):
        x = draw(experts, 9000, experts, dtype=dtype)
        dw = np.random.default_rng(2).standard_normal((9000, topk)).astype(np.float32)
        for kind in ("sigmoid", "softmax"):
            for renorm in (True, False):
                got, grad = run_route(stream, x, kind, None, 1, 1, 1, topk, renorm, 1.5, None, dw)
                r = ref.route_many(f64(x), kind, None, 1, 1, 1, topk, renorm, 1.5)
                assert np.array_equal(got["expert"], r["expert"])
                some = np.concatenate([np.arange(50), np.arange(8000, 8050), np.arange(8950, 9000)])
                r = {k: v[some] for k, v in r.items() if k in ("expert", "weights", "scores")}
                want, size = ref.route_grad(f64(x)[some], r, kind, topk, renorm, 1.5, dw[some])
                rel = (3 * 2 * np.abs(f64(x)).max() + experts + 24) * U
                assert near(grad[some], want, 3 * rel * size + 1e-37, dtype), (experts, kind, renorm)


def test_route_grad_skips_bad_experts(stream):
    """Expert numbers that point outside are skipped."""
    x = draw(1, 3, 16).cuda()
    expert = torch.tensor([[0, 99], [-7, 3], [2**31 - 1, -2**31]], dtype=torch.int32, device="cuda")
    dw, out = torch.ones(3, 2, device="cuda"), Out(3, 16, torch.float32)
    ready()
    H.expert_route_scored_grad(x.data_ptr(), dt(x.dtype), 3, 16, 2, H.HCCL_AMD_SCORE_SIGMOID, expert.data_ptr(), dw.data_ptr(), out.ptr, stream.cuda_stream)
    stream.synchronize()
    got = out.numpy()
    s = ref.sigmoid(f64(x))
    want = np.zeros((3, 16))
    want[0, 0], want[1, 3] = (s * (1 - s))[0, 0], (s * (1 - s))[1, 3]
    assert near(got, want, 40 * U * np.abs(want))


def test_bias(stream):
    rng = np.random.default_rng(1)
    for experts in (1, 5, 256, 1000, 1024):
        counts = rng.integers(0, 2**31 - 1 if experts > 256 else 9, experts).astype(np.int32)
        counts[: experts // 3] = int(counts.astype(np.int64).mean())
        bias = rng.standard_normal(experts).astype(np.float32)
        c, b, new = torch.from_numpy(counts).cuda(), torch.from_numpy(bias).cuda(), Out(1, experts, torch.float32)
        ready()
        H.expert_bias(c.data_ptr(), experts, 0.01, b.data_ptr(), new.ptr, stream.cuda_stream)
        H.expert_bias(c.data_ptr(), experts, 0.01, b.data_ptr(), b.data_ptr(), stream.cuda_stream)
        stream.synchronize()
        want = ref.bias_step(counts, 0.01, bias)
        assert np.array_equal(new.get().cpu().numpy()[0], want) and np.array_equal(b.cpu().numpy(), want)


# ---- gradient clipping ------------------------------------------------------------------------------------------------------------

def clip_all(stream, tensors, max_norm, in_place=False, accumulate=None, shift=0, out_shift=None):
    """Norm, squares and the tensors afterwards."""
    outs, ins = [], []
    for v in tensors:
        ins.append(Out(1, max(1, v.numel()), v.dtype, 0, shift))
        if v.numel():
            ins[-1].fill(v.cuda()[None])
        outs.append(ins[-1] if in_place else Out(1, max(1, v.numel()), v.dtype, 0, shift if out_shift is None else out_shift))
    table = H.grad_tensors([(i.ptr, o.ptr, v.numel(), dt(v.dtype)) for i, o, v in zip(ins, outs, tensors)])
    n = len(tensors)
    need = H.grad_squares_workspace(table, n)
    work = torch.full((need + 64,), 0xC3, dtype=torch.uint8, device="cuda")
    squares, norm = Out(1, 1, torch.float64), Out(1, 1, torch.float32)
    if accumulate is not None:
        squares.fill(torch.tensor([[accumulate]], dtype=torch.float64, device="cuda"))
    ready()
    H.grad_squares(table, n, squares.ptr, work.data_ptr(), need, stream.cuda_stream, accumulate=accumulate is not None)
    H.grad_clip(table, n, squares.ptr, max_norm, norm.ptr, stream.cuda_stream)
    stream.synchronize()
    assert bool((work[need:] == 0xC3).all())
    return norm.numpy()[0, 0], squares.numpy()[0, 0], [o.get().cpu()[0, :v.numel()] for o, v in zip(outs, tensors)]


def check_clip(tensors, max_norm, got, accumulate=0.0):
    norm, squares, outs = got
    want = sum(float((v.double() ** 2).sum()) for v in tensors) + accumulate
    # (products and sums in 64 bits, all of one sign)
    assert abs(squares - want) <= sum(v.numel() for v in tensors) * 2.0 ** -52 * want
    if want ** 0.5 < 2.0 ** 128 * (1 - U):
        assert abs(norm - want ** 0.5) <= 2 * U * want ** 0.5
    else:
        assert np.isposinf(norm)     # the norm is left in 32 bits, which end there; the tensors are clipped by what it is in 64
    by = max_norm / want ** 0.5 if want ** 0.5 > max_norm else 1.0
    for v, o in zip(tensors, outs):
        if by == 1.0:
            assert torch.equal(o, v)
        else:
            assert near(o.double().numpy(), by * f64(v), 3 * U * by * np.abs(f64(v)), v.dtype)


LISTS = {
    "one": [(1, "fp32")], "short": [(1, "bf16"), (7, "fp16"), (8, "fp32"), (0, "bf16"), (9, "bf16")], "chunks": [(16384, "fp32"), (16383, "bf16"), (16385, "fp16"), (40000, "bf16")],
    "many": [(37 * i % 501, ("fp32", "bf16", "fp16")[i % 3]) for i in range(500)], "exactly a launch": [(100, "bf16")] * 120, "one more": [(100, "bf16")] * 121,
    "large": [(5_000_001, "bf16"), (3_000_000, "fp32"), (11, "fp16")], "none": [], "empty": [(0, "fp32")] * 3,
}


@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("max_norm", [0.5, 1e9, 0.0])
@pytest.mark.parametrize("shift,out_shift", [(0, 0), (1, 1), (3, 0), (0, 5)])
def test_clip(stream, name, max_norm, shift, out_shift):
    print("clip", name, max_norm, shift, out_shift, flush=True)
    tensors = [draw(i, n, dtype=TYPE[t]) for i, (n, t) in enumerate(LISTS[name])]
    check_clip(tensors, max_norm, clip_all(stream, tensors, max_norm, shift=shift, out_shift=out_shift))


@pytest.mark.parametrize("name", ["short", "chunks", "many"])
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_clip_in_place(stream, name, max_norm):
    tensors = [draw(i, n, dtype=TYPE[t]) for i, (n, t) in enumerate(LISTS[name])]
    first = clip_all(stream, tensors, max_norm, in_place=True, shift=1)
    check_clip(tensors, max_norm, first)
    again = clip_all(stream, tensors, max_norm, shift=1)
    assert first[:2] == again[:2] and all(torch.equal(a, b) for a, b in zip(first[2], again[2]))


def test_clip_accumulates(stream):
    tensors = [draw(1, 300), draw(2, 20000, dtype=torch.bfloat16)]
    check_clip(tensors, 1.0, clip_all(stream, tensors, 1.0, accumulate=12345.678), 12345.678)


@pytest.mark.parametrize("size", [1e30, 1e-30, 3e38])
def test_clip_far_values(stream, size):
    """Squares far beyond the range of 32 bits."""
    tensors = [draw(1, 1000) .clamp(-1, 1) * size, torch.tensor([size])]
    check_clip(tensors, size, clip_all(stream, tensors, size))


def test_clip_not_finite(stream):
    bad = draw(1, 40)
    bad[7] = float("inf")
    norm, squares, (out, other) = clip_all(stream, [bad, draw(2, 5)], 1.0)
    assert np.isposinf(norm) and bool(torch.isnan(out[7])) and not out[:7].any() and not other.any()
    bad[7] = float("nan")
    norm, squares, (out, other) = clip_all(stream, [bad, draw(2, 5)], 1.0)
    assert np.isnan(norm) and bool(torch.isnan(out).all()) and bool(torch.isnan(other).all())


# ---- how they are called ------------------------------------------------------------------------------------------------------------

def calls(seed):
    """Every operator once: a function that queues it on a stream, and its outputs."""
    t, made = torch.bfloat16, []
    new = lambda *shape, dtype=t: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    x, r, dy = (draw(seed + i, 600, 1000, dtype=t).cuda() for i in range(3))
    s, y, q, scales, dx, dgain = new(600, 1000), new(600, 1000), new(600, 1024, dtype=torch.uint8), new(600, 8, dtype=torch.float32), new(600, 1000), new(1000, dtype=torch.float32)
    work = new(H.norm_rows_grad_workspace(600, 1000), dtype=torch.uint8)
    h, a, dh = draw(seed + 4, 600, 2000, dtype=t).cuda(), new(600, 1000), new(600, 2000)
    logits, bias = draw(seed + 5, 1500, 64).cuda(), draw(seed + 6, 64, scale=0.1).cuda()
    expert, weights, row_of = new(1500, 4, dtype=torch.int32), new(1500, 4, dtype=torch.float32), new(1500, 4, dtype=torch.int32)
    counts, offsets, dlogits, nb = new(65, dtype=torch.int32), new(65, dtype=torch.int32), new(1500, 64, dtype=torch.float32), new(64, dtype=torch.float32)
    need = H.expert_route_scored_workspace(1500, 64)
    work2 = new(need, dtype=torch.uint8)
    grads = [draw(seed + 7 + i, n, dtype=t).cuda() for i, n in enumerate((100, 70001, 3))]
    outs = [torch.zeros_like(g) for g in grads]
    table = H.grad_tensors([(g.data_ptr(), o.data_ptr(), g.numel(), dt(t)) for g, o in zip(grads, outs)])
    need3 = H.grad_squares_workspace(table, 3)
    work3, squares, norm = new(need3, dtype=torch.uint8), new(1, dtype=torch.float64), new(1, dtype=torch.float32)
    kept = (x, r, dy, work, h, logits, bias, work2, grads, work3, table)

    def queue(on):
        H.norm_rows(x.data_ptr(), dt(t), 600, 1000, on, residual=r.data_ptr(), sum=s.data_ptr(), y=y.data_ptr(), scale_type=1, q=q.data_ptr(), scales=scales.data_ptr())
        H.norm_rows_grad(dy.data_ptr(), s.data_ptr(), dt(t), 600, 1000, dx.data_ptr(), on, gain_grad=dgain.data_ptr(), workspace=work.data_ptr(),
                         workspace_bytes=work.numel())
        H.expert_gate(h.data_ptr(), dt(t), 600, 1000, a.data_ptr(), on)
        H.expert_gate_grad(dy.data_ptr(), h.data_ptr(), dt(t), 600, 1000, dh.data_ptr(), on)
        H.expert_route_scored(logits.data_ptr(), 4, 1500, 64, 4, 1, expert.data_ptr(), weights.data_ptr(), row_of.data_ptr(), counts.data_ptr(), offsets.data_ptr(),
                              work2.data_ptr(), need, on, bias=bias.data_ptr(), groups=8, groups_kept=3, renorm=True)
        H.expert_route_scored_grad(logits.data_ptr(), 4, 1500, 64, 4, 1, expert.data_ptr(), weights.data_ptr(), dlogits.data_ptr(), on, renorm=True)
        H.expert_bias(counts.data_ptr(), 64, 0.01, bias.data_ptr(), nb.data_ptr(), on)
        H.grad_squares(table, 3, squares.data_ptr(), work3.data_ptr(), need3, on)
        H.grad_clip(table, 3, squares.data_ptr(), 1.0, norm.data_ptr(), on)

    made += [s, y, q, scales, dx, dgain, a, dh, expert, weights, row_of, counts, offsets, dlogits, nb, squares, norm] + outs
    return queue, made, kept


def test_captured_and_replayed(stream):
    """A graph of all calls, replayed several times with eager work in between, its inputs changed, gives what the calls give."""
    queue, outs, kept = calls(100)
    other, _, kept_too = calls(200)
    ready()
    queue(stream.cuda_stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        queue(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        kept[0].copy_(draw(300 + i, 600, 1000, dtype=torch.bfloat16))
        kept[5].copy_(draw(400 + i, 1500, 64))
        kept[8][1].copy_(draw(500 + i, 70001, dtype=torch.bfloat16))
        ready()
        queue(stream.cuda_stream)
        stream.synchronize()
        want = [o.clone() for o in outs]
        for o in outs:
            o.zero_()
        other(stream.cuda_stream)
        ready()
        graph.replay()
        ready()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_two_streams_at_once():
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = [calls(100), calls(200)]
    ready()
    wants = []
    for (queue, outs, _), s in zip(sets, streams):
        queue(s.cuda_stream)
        ready()
        wants.append([o.clone() for o in outs])
        for o in outs:
            o.zero_()
    ready()
    for _ in range(5):
        for (queue, _, _), s in zip(sets, streams):
            queue(s.cuda_stream)
    ready()
    for (_, outs, _), want in zip(sets, wants):
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_far_into_memory(stream):
    """Rows more than 2^32 bytes apart."""
    far = (1 << 31) + 8
    room = torch.empty(2 * far + 4096, dtype=torch.bfloat16, device="cuda")      # 8.6 GB
    x = draw(1, 3, 512, dtype=torch.bfloat16)
    for i in range(3):
        room[i * far:i * far + 512] = x[i].cuda()
    y, out = torch.zeros(3, 512, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, 256, dtype=torch.bfloat16, device="cuda")
    want_y, want = torch.zeros_like(y), torch.zeros_like(out)
    near = x.cuda()
    table, squares = H.grad_tensors([(room.data_ptr(), None, 2 * far + 4096, dt(x.dtype))]), torch.zeros(1, dtype=torch.float64, device="cuda")
    work = torch.empty(H.grad_squares_workspace(table, 1), dtype=torch.uint8, device="cuda")
    ready()
    for src, stride, a, b in ((room, far, y, out), (near, 0, want_y, want)):
        H.norm_rows(src.data_ptr(), dt(x.dtype), 3, 512, stream.cuda_stream, y=a.data_ptr(), x_stride=stride)
        H.expert_gate(src.data_ptr(), dt(x.dtype), 3, 256, b.data_ptr(), stream.cuda_stream, h_stride=stride)
    stream.synchronize()
    assert torch.equal(y, want_y) and torch.equal(out, want)
    room.zero_()
    for i in range(3):
        room[i * far:i * far + 512] = x[i].cuda()
    ready()
    H.grad_squares(table, 1, squares.data_ptr(), work.data_ptr(), work.numel(), stream.cuda_stream)
    stream.synchronize()
    want = float((x.double() ** 2).sum())
    assert abs(float(squares) - want) <= 2000 * 2.0 ** -52 * want
