"""The experts' operators on the GPU against 64-bit references: sizes from one token up, odd and ragged ones, strides and
alignments, masks that leave rows, experts and groups empty, NaN and infinities in masked places, and the bytes around every output
untouched.  8-bit values, scales, choices, counts and rows are compared exactly; sums within bounds that follow from their length
(experts_reference.py)."""
import numpy as np
import pytest
import torch

import experts_reference as ref
from experts_reference import HALF, U, close, up128
from hccl_loader import load

pytestmark = pytest.mark.gpu
H = load()
TYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
KIND = {"fp32": ref.FP32, "e8m0": ref.E8M0}


def dt(t):
    return {torch.float32: H.HCCL_DATA_TYPE_FP32, torch.bfloat16: H.HCCL_DATA_TYPE_BFP16, torch.float16: H.HCCL_DATA_TYPE_FP16}[t]


class Out:
    """rows x width elements with a stride, in the middle of a buffer of canaries."""

    def __init__(self, rows, width, dtype, stride=0, shift=0):
        self.rows, self.width, self.stride, self.shift = rows, width, stride or width, shift
        unit = torch.empty(0, dtype=dtype).element_size()
        self.front = 64 + shift * unit
        self.raw = torch.full((self.front + rows * self.stride * unit + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        self.unit, self.dtype = unit, dtype
        body = self.raw[self.front:self.front + rows * self.stride * unit].clone()     # (torch wants aligned views)
        self.n = body.numel()

    @property
    def ptr(self):
        return self.raw.data_ptr() + self.front

    def fill(self, values):
        v = torch.full((self.rows, self.stride), 0, dtype=self.dtype, device="cuda")
        v.view(torch.uint8).fill_(0xA5)
        v[:, :self.width] = values
        self.raw[self.front:self.front + self.n] = v.reshape(-1).view(torch.uint8)
        return self

    def get(self):
        """The values; the bytes around them have to be canaries."""
        assert bool((self.raw[:self.front] == 0xA5).all()) and bool((self.raw[self.front + self.n:] == 0xA5).all())
        v = self.raw[self.front:self.front + self.n].clone().view(self.dtype).reshape(self.rows, self.stride)
        assert bool((v[:, self.width:].contiguous().view(torch.uint8) == 0xA5).all())
        return v[:, :self.width].contiguous()

    def numpy(self):
        v = self.get().cpu()
        return v.double().numpy() if v.is_floating_point() else v.numpy()


@pytest.fixture(scope="module")
def stream():
    return torch.cuda.Stream()


def done(stream):
    stream.synchronize()


def ready():
    torch.cuda.synchronize()


def canary(dtype, shape):
    return torch.full(shape, 0xA5, dtype=torch.uint8).view(dtype)


# ---- router -----------------------------------------------------------------------------------------------------------------

def run_route(stream, logits, topk, renorm, mask=None, stride=0, shift=0, dw=None, dl=None, loss_scale=0.01, out_stride=0):
    T, E = logits.shape
    ins = Out(T, E, logits.dtype, stride, shift).fill(logits)
    o = {"expert": Out(T, topk, torch.int32), "weights": Out(T, topk, torch.float32), "row_of": Out(T, topk, torch.int32),
         "counts": Out(1, E + 1, torch.int32), "offsets": Out(1, E + 1, torch.int32), "loss": Out(1, 1, torch.float32)}
    need = H.expert_route_workspace(T, E)
    work = torch.full((need + 64,), 0xC3, dtype=torch.uint8, device="cuda")
    m = None if mask is None else torch.from_numpy(mask).cuda()
    mp = None if m is None else m.data_ptr()
    grad = Out(T, E, logits.dtype, out_stride, shift)
    wg = None if dw is None else torch.from_numpy(dw.astype(np.float32)).cuda()
    lg = None if dl is None else torch.tensor([dl], dtype=torch.float32, device="cuda")
    ready()
    H.expert_route(ins.ptr, dt(logits.dtype), T, E, topk, o["expert"].ptr, o["weights"].ptr, o["row_of"].ptr, o["counts"].ptr, o["offsets"].ptr,
                   o["loss"].ptr, work.data_ptr() if need else None, need, stream.cuda_stream, renorm=renorm, mask=mp, loss_scale=loss_scale,
                   stride=stride)
    H.expert_route_grad(ins.ptr, dt(logits.dtype), T, E, topk, o["expert"].ptr, o["counts"].ptr, None if wg is None else wg.data_ptr(),
                        None if lg is None else lg.data_ptr(), grad.ptr, stream.cuda_stream, renorm=renorm, mask=mp, loss_scale=loss_scale,
                        stride=stride, grad_stride=out_stride)
    done(stream)
    assert bool((work[need:] == 0xC3).all())
    return {k: v.numpy() for k, v in o.items()}, grad.numpy()


def check_route(logits, topk, renorm, mask, got, grad, dw, dl, loss_scale=0.01):
    x = logits.double().cpu().numpy()
    T, E = x.shape
    r = ref.route(x, topk, renorm, mask, loss_scale)
    for k in ("expert", "row_of"):
        assert np.array_equal(got[k], r[k]), k
    assert np.array_equal(got["counts"][0], r["counts"]) and np.array_equal(got["offsets"][0], r["offsets"])
    # exp's argument is off by U times itself, exp by two units, the sum over the experts by E + 1, the quotient by one
    far = 0.0
    for t in range(T):
        f = x[t][np.isfinite(x[t])]
        if f.size and r["expert"][t, 0] >= 0:
            far = max(far, min(110.0, f.max() - f.min()))
    rel = (2 * far + E + 10) * U
    assert close(got["weights"], r["weights"], 2 * rel * np.abs(r["weights"]) + 1e-37)
    assert close(got["loss"][0], [r["loss"]], (rel + (T + 2 * E + 10) * U) * abs(r["loss"]))
    want, size = ref.route_grad(r, topk, renorm, loss_scale, dw, dl)
    assert close(grad, want, (4 * rel + 8 * U) * size + 1e-37, logits.dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tokens,experts,topk", [(1, 1, 1), (1, 64, 6), (3, 5, 5), (64, 8, 2), (65, 8, 2), (63, 60, 4), (200, 127, 7), (257, 256, 8),
                                                 (100, 257, 3), (33, 1000, 16), (17, 1024, 9), (1000, 16, 16), (4099, 64, 1), (48, 200, 8), (5003, 60, 4)])
def test_route(stream, dtype, tokens, experts, topk):
    rng = np.random.default_rng(tokens * 7 + experts)
    for renorm in (False, True):
        print("route", dtype, tokens, experts, topk, renorm, flush=True)
        logits = torch.from_numpy(2 * rng.standard_normal((tokens, experts)) + rng.standard_normal(experts)).to(TYPE[dtype])
        mask = (rng.random(tokens) > 0.2).astype(np.uint8) if renorm else None
        dw, dl = rng.standard_normal((tokens, topk)).astype(np.float32), 1.25
        got, grad = run_route(stream, logits, topk, renorm, mask, dw=dw, dl=dl)
        check_route(logits, topk, renorm, mask, got, grad, dw, dl)


def test_route_large(stream):
    """Enough tokens for tiles of 64; ties everywhere (few different values)."""
    rng = np.random.default_rng(5)
    logits = torch.from_numpy(rng.integers(0, 7, (16500, 24)) * 0.5).to(torch.bfloat16)
    dw, dl = rng.standard_normal((16500, 4)).astype(np.float32), -0.5
    got, grad = run_route(stream, logits, 4, True, None, dw=dw, dl=dl)
    check_route(logits, 4, True, None, got, grad, dw, dl)
    again, grad2 = run_route(stream, logits, 4, True, None, dw=dw, dl=dl)
    assert all(np.array_equal(got[k], again[k]) for k in got) and np.array_equal(grad, grad2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tokens,experts,topk", [(4200, 127, 7), (4200, 256, 8), (5000, 200, 16), (4500, 65, 2), (6000, 256, 3), (4300, 30, 16), (5000, 64, 8),
                                                 (70000, 16, 2), (140000, 8, 1), (66000, 256, 8), (17000, 300, 3), (40000, 1024, 4)])
def test_route_many_tokens(stream, dtype, tokens, experts, topk):
    """Beyond 4096 tokens, four lanes to a token, with up to 64 experts a lane and lists of every length; beyond 65536 (with more than 256 experts
    16384) workgroups of several tiles each."""
    rng = np.random.default_rng(tokens + experts)
    t = TYPE[dtype]
    for renorm in (False, True):
        print("route", dtype, tokens, experts, topk, renorm, flush=True)
        logits = torch.from_numpy((2 * rng.standard_normal((tokens, experts)) + rng.standard_normal(experts)).astype(np.float32)).to(t)
        mask = (rng.random(tokens) > 0.2).astype(np.uint8) if renorm else None
        dw, dl = rng.standard_normal((tokens, topk)).astype(np.float32), 1.25
        got, grad = run_route(stream, logits, topk, renorm, mask, dw=dw, dl=dl)
        x = logits.double().numpy()
        r, want, size = ref.route_finite(x, topk, renorm, mask, 0.01, dw.astype(np.float64), dl)
        for k in ("expert", "row_of"):
            assert np.array_equal(got[k], r[k]), k
        assert np.array_equal(got["counts"][0], r["counts"]) and np.array_equal(got["offsets"][0], r["offsets"])
        # (as for few tokens: exp's argument, the sum over the experts, the quotient; the loss adds up the tokens as well)
        rel = (2 * (x.max(1) - x.min(1)).max() + experts + 10) * U
        assert close(got["weights"], r["weights"], 2 * rel * np.abs(r["weights"]) + 1e-37)
        assert close(got["loss"][0], [r["loss"]], (rel + (tokens + 2 * experts + 10) * U) * abs(r["loss"]))
        assert close(grad, want, (4 * rel + 8 * U) * size + 1e-37, t)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("stride,shift", [(0, 1), (61, 0), (64, 3), (72, 0)])
def test_route_strides(stream, dtype, stride, shift):
    rng = np.random.default_rng(stride + shift)
    logits = torch.from_numpy(rng.standard_normal((90, 60))).to(TYPE[dtype])
    dw = rng.standard_normal((90, 5)).astype(np.float32)
    for dl in (None, 2.0):
        got, grad = run_route(stream, logits, 5, False, None, stride, shift, dw=dw, dl=dl, out_stride=stride)
        check_route(logits, 5, False, None, got, grad, dw, dl)
    got, grad = run_route(stream, logits, 5, True, None, stride, shift, dw=None, dl=2.0, out_stride=stride)
    check_route(logits, 5, True, None, got, grad, None, 2.0)


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_route_masked_places(stream, dtype, renorm):
    """Masked tokens full of NaN and infinities; rows with fewer experts than choices, with none, of the type's lowest value."""
    t = TYPE[dtype]
    rng = np.random.default_rng(3)
    logits = torch.from_numpy(rng.standard_normal((80, 20))).to(t)
    mask = np.ones(80, np.uint8)
    for i, v in ((0, float("nan")), (7, float("inf")), (63, -float("inf")), (64, float("nan"))):
        logits[i] = v
        mask[i] = 0
    logits[1] = -float("inf")
    logits[2] = -float("inf")
    logits[2, 3] = 0.5                       # one expert only
    logits[3] = torch.finfo(t).min           # all alike: the lowest experts
    logits[4, :] = torch.finfo(t).min
    logits[4, 5] = 1.0                       # one that counts, the others' weights are 0
    logits[79] = -float("inf")
    logits[79, 18:] = 0.0
    dw, dl = rng.standard_normal((80, 4)).astype(np.float32), 1.0
    got, grad = run_route(stream, logits, 4, renorm, mask, dw=dw, dl=dl)
    assert np.isfinite(got["loss"]).all() and np.isfinite(grad).all()
    check_route(logits, 4, renorm, mask, got, grad, dw, dl)
    assert (got["expert"][3] == [0, 1, 2, 3]).all() and (got["expert"][1] == -1).all()
    # nobody takes part: zeros
    got, grad = run_route(stream, logits, 4, renorm, np.zeros(80, np.uint8), dw=dw, dl=dl)
    assert not got["counts"].any() and not got["offsets"].any() and not got["loss"].any() and not grad.any() and (got["row_of"] == -1).all()


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("experts", [20, 127])
def test_route_masked_places_of_many_tokens(stream, dtype, renorm, experts):
    """The same in the form for many tokens: masked tokens of NaN and infinities, rows of few experts, of none, of the type's lowest value."""
    t, T = TYPE[dtype], 4200
    rng = np.random.default_rng(experts)
    logits = torch.from_numpy(rng.standard_normal((T, experts))).to(t)
    mask = np.ones(T, np.uint8)
    for i, v in ((0, float("nan")), (64, float("inf")), (2000, -float("inf")), (T - 1, float("nan"))):
        logits[i] = v
        mask[i] = 0
    logits[1] = -float("inf")
    logits[2] = -float("inf")
    logits[2, 3] = 0.5
    logits[3] = torch.finfo(t).min
    logits[4, :] = torch.finfo(t).min
    logits[4, 5] = 1.0
    logits[T - 2] = -float("inf")
    logits[T - 2, experts - 2:] = 0.0
    dw, dl = rng.standard_normal((T, 4)).astype(np.float32), 1.0
    got, grad = run_route(stream, logits, 4, renorm, mask, dw=dw, dl=dl)
    assert np.isfinite(got["loss"]).all() and np.isfinite(grad).all()
    check_route(logits, 4, renorm, mask, got, grad, dw, dl)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_route_zeros_of_both_signs_are_ties(stream, dtype):
    logits = torch.tensor([[-0.0, 0.0, -1.0, 0.0, -0.0, -2.0]] * 3).to(TYPE[dtype])
    logits[1] *= -1
    dw = np.ones((3, 4), np.float32)
    got, grad = run_route(stream, logits, 4, True, dw=dw, dl=1.0)
    check_route(logits, 4, True, None, got, grad, dw, 1.0)
    assert got["expert"][0].tolist() == [0, 1, 3, 4] and got["expert"][1].tolist() == [5, 2, 0, 1]


def test_route_nan_of_a_token_that_takes_part(stream):
    logits = torch.zeros(3, 8)
    logits[1, 2] = float("nan")
    logits[2, 4] = float("inf")
    got, _ = run_route(stream, logits, 2, True)
    assert (got["expert"] == [[0, 1], [0, 1], [4, 0]]).all()
    assert np.isnan(got["weights"][1]).all() and np.isnan(got["weights"][2]).all() and np.isnan(got["loss"]).all()
    assert np.isfinite(got["weights"][0]).all() and got["counts"][0].tolist() == [3, 2, 0, 0, 1, 0, 0, 0, 3]


def test_route_no_tokens(stream):
    o = [torch.full((n,), 9, dtype=torch.int32, device="cuda") for n in (9, 9)]
    loss = torch.full((1,), 9.0, device="cuda")
    ready()
    H.expert_route(None, H.HCCL_DATA_TYPE_FP32, 0, 8, 2, None, None, None, o[0].data_ptr(), o[1].data_ptr(), loss.data_ptr(), None, 0, stream.cuda_stream)
    done(stream)
    assert not o[0].any() and not o[1].any() and float(loss) == 0.0


@pytest.mark.parametrize("renorm", [False, True])
def test_route_gradient_against_differences(stream, renorm):
    rng = np.random.default_rng(11)
    T, E, k = 70, 12, 3
    logits = torch.from_numpy(np.stack([rng.permutation(E) * 0.4 for _ in range(T)]) + rng.uniform(0, 0.1, (T, E))).float()
    dw, dl = rng.standard_normal((T, k)).astype(np.float32), 3.0
    _, grad = run_route(stream, logits, k, renorm, dw=dw, dl=dl, loss_scale=1.0)
    x = logits.double().numpy()

    def value(x):
        r = ref.route(x, k, renorm, None, 1.0)
        return (r["weights"] * dw).sum() + dl * r["loss"]

    for i in range(8):
        step = rng.standard_normal(x.shape)
        h = 1e-5
        slope = (value(x + h * step) - value(x - h * step)) / (2 * h)
        # every one of the T E entries may be off by 200 U of values below 3; the differences by h^2 and 2^-53 / h times 1000
        assert abs(slope - (grad * step).sum()) < 200 * U * 3 * np.abs(step).sum() + 1e-6


# ---- rows into expert order and back --------------------------------------------------------------------------------------------

def some_rows(rng, tokens, topk, missing, spare=3):
    """row_of with some choices missing, and rows nobody names."""
    n = tokens * topk
    row = np.full(n, -1, np.int64)
    taken = rng.random(n) >= missing
    row[taken] = rng.permutation(taken.sum() + spare)[:taken.sum()]
    return row.reshape(tokens, topk).astype(np.int32), int(taken.sum()) + spare


def values(rng, shape, dtype, odd=False):
    x = torch.from_numpy(rng.standard_normal(shape) * np.exp(rng.standard_normal((shape[0], 1)))).to(dtype)
    if odd and x.numel() > 600:
        x[0, :200] = 0                                    # a whole block of zeros
        x[1, 3], x[1, 5], x[1, 6] = float("inf"), float("nan"), -float("inf")
        x[2, 130:135] = torch.finfo(dtype).max
        x[2, 0] = torch.finfo(dtype).tiny
    return x


SIZES = [(1, 1, 1), (1, 128, 1), (3, 127, 2), (2, 129, 8), (70, 520, 3), (64, 1024, 8), (5, 8192, 16), (33, 2001, 4), (300, 64, 6)]


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,width,topk", SIZES)
def test_pack_in_8_bits(stream, kind, dtype, tokens, width, topk):
    rng = np.random.default_rng(tokens + width)
    row, rows = some_rows(rng, tokens, topk, 0.2)
    x = values(rng, (tokens, width), TYPE[dtype], odd=True)
    for stride, shift, out_stride in ((0, 0, 0), (width + 3, 1, up128(width) + 16), (width + 8, 8, 0)):
        print("pack", kind, dtype, tokens, width, topk, stride, flush=True)
        xin = Out(tokens, width, TYPE[dtype], stride, shift).fill(x)
        q = Out(rows, up128(width), torch.uint8, out_stride)
        s = Out(rows, up128(width) // 128, torch.float32 if kind == "fp32" else torch.uint8, up128(width) // 128 + (1 if out_stride else 0))
        r = torch.from_numpy(row).cuda()
        ready()
        H.expert_pack(xin.ptr, dt(x.dtype), tokens, width, topk, r.data_ptr(), q.ptr, rows, stream.cuda_stream, scales=s.ptr, scale_type=KIND[kind],
                      x_stride=stride, out_stride=out_stride, scale_stride=s.stride)
        done(stream)
        codes, stored, _ = ref.quant_rows(x.float().numpy(), KIND[kind])
        got_q, got_s = q.get().cpu().numpy(), s.get().cpu().numpy()
        named = np.zeros(rows, bool)
        for t in range(tokens):
            for j in range(topk):
                if row[t, j] >= 0:
                    named[row[t, j]] = True
                    assert ref.same_codes(got_q[row[t, j]], codes[t]) and np.array_equal(got_s[row[t, j]], stored[t]), (t, j)
        assert (got_q[~named] == 0xA5).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,width,topk", SIZES)
def test_pack_copies_and_combine(stream, dtype, tokens, width, topk):
    """A copy, weights that sum rows up, and both gradients."""
    t = TYPE[dtype]
    rng = np.random.default_rng(tokens * 3 + width)
    row, rows = some_rows(rng, tokens, topk, 0.25)
    x = values(rng, (tokens, width), t)
    w = rng.standard_normal((tokens, topk)).astype(np.float32)
    w[row < 0] = np.nan                                   # weights of choices that are not there are not looked at
    back = values(rng, (rows, width), t)
    named = np.zeros(rows, bool)
    named[row[row >= 0]] = True
    back[~torch.from_numpy(named)] = float("nan")         # nor rows that nobody names
    dy = values(rng, (tokens, width), t)
    r, wg = torch.from_numpy(row).cuda(), torch.from_numpy(w).cuda()
    has = row >= 0
    for stride, shift in ((0, 0), (width + 1, 1), (width + 8, 8)):
        print("exchange", dtype, tokens, width, topk, stride, shift, flush=True)
        xin = Out(tokens, width, t, stride, shift).fill(x)
        packed = Out(rows, width, t, stride, shift)
        bin_ = Out(rows, width, t, stride, shift).fill(back)
        y, ysum = Out(tokens, width, t, stride, shift), Out(tokens, width, t, stride, shift)
        dyin = Out(tokens, width, t, stride, shift).fill(dy)
        dx, dwt = Out(rows, width, t, stride, shift), Out(tokens, topk, torch.float32)
        ready()
        S = stream.cuda_stream
        H.expert_pack(xin.ptr, dt(t), tokens, width, topk, r.data_ptr(), packed.ptr, rows, S, x_stride=stride, out_stride=stride)
        H.expert_combine(bin_.ptr, dt(t), rows, width, tokens, topk, r.data_ptr(), wg.data_ptr(), y.ptr, S, x_stride=stride, y_stride=stride)
        H.expert_combine(bin_.ptr, dt(t), rows, width, tokens, topk, r.data_ptr(), None, ysum.ptr, S, x_stride=stride, y_stride=stride)
        H.expert_combine_grad(dyin.ptr, bin_.ptr, dt(t), rows, width, tokens, topk, r.data_ptr(), wg.data_ptr(), dx.ptr, dwt.ptr, S,
                              y_grad_stride=stride, x_stride=stride, x_grad_stride=stride)
        done(stream)
        got = packed.get().cpu()
        gx = dx.get().cpu()
        X, B, D = x.double().numpy(), back.double().numpy(), dy.double().numpy()
        for i in range(tokens):
            for j in range(topk):
                if has[i, j]:
                    assert torch.equal(got[row[i, j]], x[i])
                    p = np.float64(w[i, j]) * D[i]
                    assert close(gx[row[i, j]].double().numpy(), p, U * np.abs(p), t)
        for buf in (got, gx):
            assert bool((buf[~torch.from_numpy(named)].contiguous().view(torch.uint8) == 0xA5).all())
        at = np.where(has, row, 0)
        terms = np.where(has[..., None], np.where(has, w, 0)[..., None] * np.nan_to_num(B[at]), 0)
        assert close(y.numpy(), terms.sum(1), (topk + 1) * U * np.abs(terms).sum(1), t)
        ones = np.where(has[..., None], np.nan_to_num(B[at]), 0)
        assert close(ysum.numpy(), ones.sum(1), (topk + 1) * U * np.abs(ones).sum(1), t)
        dots = np.where(has[..., None], D[:, None] * np.nan_to_num(B[at]), 0)
        assert close(dwt.numpy(), dots.sum(2), (width + 1) * U * np.abs(dots).sum(2))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shift", [0, 1])
def test_pack_copies_bits(stream, dtype, shift):
    """Every pattern of 16 bits, the NaN that signal among them, and of 32 bits those and random ones; aligned and off every boundary."""
    t = TYPE[dtype]
    if dtype == "fp32":
        high = np.arange(1 << 16, dtype=np.uint32) << 16
        bits = torch.from_numpy((high | np.random.default_rng(9).integers(0, 1 << 16, 1 << 16, dtype=np.uint32)).view(np.int32)).reshape(64, 1024)
    else:
        bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).reshape(64, 1024)
    row = torch.randperm(64, generator=torch.Generator().manual_seed(1)).int().reshape(64, 1)
    x, out, r = Out(64, 1024, bits.dtype, 1024 + shift, shift).fill(bits.cuda()), Out(64, 1024, bits.dtype, 1024 + shift, shift), row.cuda()
    ready()
    H.expert_pack(x.ptr, dt(t), 64, 1024, 1, r.data_ptr(), out.ptr, 64, stream.cuda_stream, x_stride=x.stride, out_stride=out.stride)
    done(stream)
    assert torch.equal(out.get().cpu()[row[:, 0].long()], bits)


def test_rows_without_a_map_and_rows_that_are_not_there(stream):
    """rowOf None: row t is token t.  Rows outside [0, rows) are skipped."""
    x = torch.randn(5, 256, device="cuda")
    q, s = Out(5, 256, torch.uint8), Out(5, 2, torch.float32)
    y = Out(5, 256, torch.float32)
    bad = torch.tensor([[0], [5], [-7], [2 ** 31 - 1], [4]], dtype=torch.int32, device="cuda")
    packed = Out(5, 256, torch.float32)
    dw = Out(5, 1, torch.float32)
    ready()
    S = stream.cuda_stream
    H.expert_pack(x.data_ptr(), H.HCCL_DATA_TYPE_FP32, 5, 256, 1, None, q.ptr, 5, S, scales=s.ptr, scale_type=H.HCCL_AMD_SCALE_FP32)
    H.expert_pack(x.data_ptr(), H.HCCL_DATA_TYPE_FP32, 5, 256, 1, bad.data_ptr(), packed.ptr, 5, S)
    H.expert_combine(x.data_ptr(), H.HCCL_DATA_TYPE_FP32, 5, 256, 5, 1, bad.data_ptr(), None, y.ptr, S)
    H.expert_combine_grad(x.data_ptr(), x.data_ptr(), H.HCCL_DATA_TYPE_FP32, 5, 256, 5, 1, bad.data_ptr(), None, None, dw.ptr, S)
    done(stream)
    codes, stored, _ = ref.quant_rows(x.cpu().numpy(), ref.FP32)
    assert np.array_equal(q.get().cpu().numpy(), codes) and np.array_equal(s.get().cpu().numpy(), stored)
    p, z = packed.get().cpu(), y.get().cpu()
    assert torch.equal(p[0], x[0].cpu()) and torch.equal(p[4], x[4].cpu()) and bool((p[1:4].view(torch.uint8) == 0xA5).all())
    assert torch.equal(z[0], x[0].cpu()) and torch.equal(z[4], x[4].cpu()) and not z[1:4].any()
    assert not dw.get().cpu()[1:4].any() and float(dw.get()[0]) > 0


# ---- 8-bit products ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("experts,n,k", [(1, 1, 1), (3, 128, 128), (2, 129, 255), (1, 300, 1000), (5, 64, 40)])
def test_quant_weights(stream, kind, dtype, experts, n, k):
    rng = np.random.default_rng(n + k)
    for stride, shift in ((0, 0), (k + 5, 1)):
        w = values(rng, (experts * n, k), TYPE[dtype], odd=True)
        win = Out(experts * n, k, TYPE[dtype], stride, shift).fill(w)
        real = torch.float32 if kind == "fp32" else torch.uint8
        q, qt = Out(experts * n, up128(k), torch.uint8), Out(experts * k, up128(n), torch.uint8)
        nb, kb = up128(n) // 128, up128(k) // 128
        s, st = Out(experts * nb, kb, real), Out(experts * kb, nb, real)
        ready()
        H.block_quant_weights(win.ptr, dt(w.dtype), experts, n, k, KIND[kind], q.ptr, s.ptr, qt.ptr, st.ptr, stream.cuda_stream, stride=stride)
        done(stream)
        codes, stored, _ = ref.quant_weights(w.float().numpy().reshape(experts, n, k), KIND[kind])
        assert ref.same_codes(q.get().cpu().numpy().reshape(codes.shape), codes) and np.array_equal(s.get().cpu().numpy().reshape(stored.shape), stored)
        tcodes = np.zeros((experts, k, up128(n)), np.uint8)
        tcodes[:, :, :n] = codes[:, :, :k].transpose(0, 2, 1)
        assert ref.same_codes(qt.get().cpu().numpy().reshape(tcodes.shape), tcodes)
        assert np.array_equal(st.get().cpu().numpy().reshape(experts, kb, nb), stored.transpose(0, 2, 1))


def some_groups(rng, rows, groups, skew=True):
    """Ascending offsets of groups, some of them empty."""
    if groups == 1:
        return np.array([0, rows], np.int32)
    w = rng.random(groups) ** (4 if skew else 1) * (rng.random(groups) > 0.25) + 1e-9
    n = np.floor(w / w.sum() * rows).astype(int)
    n[int(np.argmax(w))] += rows - n.sum()
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,width,groups", [(1, 1, 1), (128, 128, 1), (129, 130, 3), (700, 72, 70), (1000, 257, 5), (64, 1000, 200)])
def test_quant_columns(stream, kind, dtype, rows, width, groups):
    rng = np.random.default_rng(rows + width)
    offsets = some_groups(rng, rows, groups)
    columns = H.block_columns(rows, groups)
    for stride, shift in ((0, 0), (width + 3, 1)):
        x = values(rng, (rows, width), TYPE[dtype], odd=True)
        xin = Out(rows, width, TYPE[dtype], stride, shift).fill(x)
        q, s = Out(width, columns, torch.uint8), Out(columns // 128, width, torch.float32 if kind == "fp32" else torch.uint8)
        off = torch.from_numpy(offsets).cuda()
        ready()
        H.block_quant_columns(xin.ptr, dt(x.dtype), rows, width, groups, off.data_ptr(), KIND[kind], q.ptr, columns, s.ptr, stream.cuda_stream, stride=stride)
        done(stream)
        codes, stored, _ = ref.quant_columns(x.float().numpy(), offsets, KIND[kind])
        got_q, got_s = q.get().cpu().numpy(), s.get().cpu().numpy()
        used = codes.shape[1]
        assert ref.same_codes(got_q[:, :used], codes) and np.array_equal(got_s[:used // 128], stored)
        assert (got_q[:, used:] == 0xA5).all()


def check_matmul(stream, rng, rows, groups, experts, n, k, kind, dtype, owner=False, strides=False, offsets=None):
    offsets = some_groups(rng, rows, groups) if offsets is None else offsets
    own = rng.integers(0, experts, groups).astype(np.int32) if owner else None
    a = rng.standard_normal((rows, k)).astype(np.float32) * np.exp(rng.standard_normal((rows, 1))).astype(np.float32)
    w = rng.standard_normal((experts, n, k)).astype(np.float32)
    qa, sa, va = ref.quant_rows(a, KIND[kind])
    qw, sw, vw = ref.quant_weights(w, KIND[kind])
    t = TYPE[dtype]
    KP, KB = up128(k), up128(k) // 128
    more = 1 if strides else 0
    A = Out(rows, KP, torch.uint8, KP + 48 * more, 16 * more).fill(torch.from_numpy(qa).cuda())
    sdt = torch.float32 if kind == "fp32" else torch.uint8
    SA = Out(rows, KB, sdt, KB + more).fill(torch.from_numpy(sa.astype(np.float32) if kind == "fp32" else sa).cuda())
    W, SW = torch.from_numpy(qw).cuda(), torch.from_numpy(sw).cuda()
    y = Out(rows, n, t, n + 3 * more, more)
    off = torch.from_numpy(offsets).cuda()
    og = None if own is None else torch.from_numpy(own).cuda()
    ready()
    H.block_matmul(A.ptr, SA.ptr, rows, W.data_ptr(), SW.data_ptr(), experts, n, k, KIND[kind], y.ptr, dt(t), stream.cuda_stream, groups=groups,
                   offsets=off.data_ptr(), expert_of_group=None if og is None else og.data_ptr(), a_stride=A.stride if more else 0,
                   a_scale_stride=SA.stride, y_stride=y.stride)
    done(stream)
    got = y.get().cpu()
    va, vw = rows_ok(ref.rows_values(qa, va)[:, :k]), ref.weights_values(qw, vw)[:, :, :k]
    lo0, hi0 = offsets[0], offsets[-1]
    for g in range(groups):
        lo, hi = offsets[g], offsets[g + 1]
        if hi > lo:
            m = vw[own[g] if owner else g]
            want, size = va[lo:hi] @ m.T, np.abs(va[lo:hi]) @ np.abs(m).T
            # a sum of k products in 32 bits, each block's scaled once more; the matrix unit may cut off instead of rounding: twice
            assert close(got[lo:hi].double().numpy(), want, 2 * (k + 3 * KB + 2) * U * size, t), (g, lo, hi)
    for part in (got[:lo0], got[hi0:]):
        assert bool((part.contiguous().view(torch.uint8) == 0xA5).all())


def rows_ok(v):
    return v


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("rows,groups,experts,n,k", [
    (1, 1, 1, 1, 1), (1, 1, 1, 64, 128), (7, 1, 1, 65, 200), (16, 1, 1, 128, 384), (17, 3, 3, 100, 129), (8, 64, 64, 96, 256), (40, 200, 200, 33, 64),
    (64, 2, 2, 256, 1000), (130, 5, 5, 130, 640), (300, 1, 1, 300, 512), (33, 1, 1, 4000, 257), (130, 1, 1, 4100, 384), (70, 2, 2, 3900, 130), (513, 4, 4, 257, 300), (1000, 9, 9, 520, 1100)])
def test_matmul(stream, kind, rows, groups, experts, n, k):
    rng = np.random.default_rng(rows + n + k)
    for dtype in ("bf16", "fp16", "fp32"):
        print("matmul", kind, rows, groups, n, k, dtype, flush=True)
        check_matmul(stream, rng, rows, groups, experts, n, k, kind, dtype, strides=dtype != "bf16")


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("rows,groups,experts,n,k", [(90, 12, 3, 70, 260), (900, 16, 4, 300, 256), (2100, 6, 2, 600, 384)])
def test_matmul_groups_that_share_weights(stream, kind, rows, groups, experts, n, k):
    """What a receive buffer of an all-to-all-v looks like: source rank by source rank, each with all local experts; rows before the
    first and behind the last group belong to nobody."""
    rng = np.random.default_rng(rows)
    offsets = some_groups(rng, rows - 10, groups) + 4
    check_matmul(stream, rng, rows, groups, experts, n, k, kind, "bf16", owner=True, strides=True, offsets=offsets.astype(np.int32))


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("rows,n,k", [(2048, 2048, 512), (1500, 1111, 1300), (4100, 640, 128)])
def test_matmul_large(stream, kind, rows, n, k):
    rng = np.random.default_rng(rows)
    check_matmul(stream, rng, rows, 1, 1, n, k, kind, "bf16")
    check_matmul(stream, rng, rows, 8, 8, n // 2, k, kind, "fp32", strides=True)


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("rows,groups,n,k,dtype", [(4100, 1, 4100, 300, "bf16"), (4100, 1, 4104, 1000, "fp16"), (6000, 3, 2600, 513, "bf16")])
def test_matmul_many_tiles(stream, kind, rows, groups, n, k, dtype):
    """Enough for tiles of 256 x 256; groups whose last tile is nearly empty, odd and even numbers of blocks."""
    rng = np.random.default_rng(rows + k)
    check_matmul(stream, rng, rows, groups, groups, n, k, kind, dtype, strides=n % 8 != 0)


def run_matmul(stream, qa, sa, qw, sw, n, k, kind, dtype):
    """All rows in one group without offsets."""
    rows, t = qa.shape[0], TYPE[dtype]
    A, SA, W, SW = (torch.from_numpy(v).cuda() for v in (qa, sa, qw, sw))
    y = Out(rows, n, t)
    ready()
    H.block_matmul(A.data_ptr(), SA.data_ptr(), rows, W.data_ptr(), SW.data_ptr(), 1, n, k, KIND[kind], y.ptr, dt(t), stream.cuda_stream)
    done(stream)
    return y.numpy()


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n,k", [(40, 200, 1024), (16, 64, 384), (1000, 1100, 1024), (4100, 4100, 384), (4000, 4000, 640)])
def test_matmul_sums_are_in_32_bits(stream, kind, dtype, rows, n, k):
    """Two large products of every block cancel, what is left is 10^5 times smaller: sums of fewer bits lose it."""
    print("matmul, cancelling", kind, dtype, rows, n, k, flush=True)
    rng = np.random.default_rng(rows + k)
    a, w = (2 * rng.standard_normal((m, k)).astype(np.float32) for m in (rows, n))
    a[:, 0::128] = a[:, 1::128] = w[:, 0::128] = 448
    w[:, 1::128] = -448
    qa, sa, va = ref.quant_rows(a, KIND[kind])
    qw, sw, vw = ref.quant_weights(w[None], KIND[kind])
    got = run_matmul(stream, qa, sa, qw, sw, n, k, kind, dtype)
    want = ref.rows_values(qa, va) @ ref.weights_values(qw, vw)[0].T
    # the results' own rounding, and k roundings of partial sums up to 448^2, independent of each other: their 2-norm per result, four times
    room = HALF[TYPE[dtype]] * np.linalg.norm(want) + 4 * k ** 0.5 * U * 448 ** 2 * want.size ** 0.5
    assert np.linalg.norm(got - want) < room, (np.linalg.norm(got - want) / room)
    assert room < 0.04 * np.linalg.norm(want)


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("rows,n,k", [(24, 100, 1000), (700, 500, 1000), (4100, 4100, 260)])
def test_products_of_32_bits_as_a_whole(stream, kind, rows, n, k):
    """The 2-norm of all errors, which leaves no room for sums of fewer bits as the bounds for single results do: results and weights' gradient."""
    print("products of 32 bits", kind, rows, n, k, flush=True)
    rng = np.random.default_rng(rows + n)
    a, w = (rng.standard_normal((m, k)).astype(np.float32) for m in (rows, n))
    qa, sa, va = ref.quant_rows(a, KIND[kind])
    qw, sw, vw = ref.quant_weights(w[None], KIND[kind])
    got = run_matmul(stream, qa, sa, qw, sw, n, k, kind, "fp32")
    want = ref.rows_values(qa, va) @ ref.weights_values(qw, vw)[0].T

    def room(terms):
        # independent roundings, cut off at worst (2 U), of partial sums that grow as the root of their terms: 2 U sqrt(terms / 2) of the result
        return 2 * U * (terms / 2) ** 0.5 + 4 * U

    assert np.linalg.norm(got - want) < room(k) * np.linalg.norm(want)
    if rows * n > 1 << 20:
        return
    dy, x = (torch.from_numpy(rng.standard_normal((rows, c))).bfloat16() for c in (n, k))
    columns, sdt = H.block_columns(rows, 1), torch.float32 if kind == "fp32" else torch.uint8
    (qy, sy), (qx, sx) = ((Out(c, columns, torch.uint8), Out(columns // 128, c, sdt)) for c in (n, k))
    dw, ins = Out(n, k, torch.float32), [v.cuda() for v in (dy, x)]
    ready()
    S = stream.cuda_stream
    for v, q, s, c in ((ins[0], qy, sy, n), (ins[1], qx, sx, k)):
        H.block_quant_columns(v.data_ptr(), H.HCCL_DATA_TYPE_BFP16, rows, c, 1, None, KIND[kind], q.ptr, columns, s.ptr, S)
    H.block_matmul_grad_weight(qy.ptr, sy.ptr, qx.ptr, sx.ptr, columns, rows, n, k, KIND[kind], 1, None, 1, dw.ptr, H.HCCL_DATA_TYPE_FP32, S)
    done(stream)
    y64, x64 = (ref.from_fp8(q) * np.repeat(v.T, 128, 1) for q, _, v in (ref.quant_columns(t.float().numpy(), [0, rows], KIND[kind]) for t in (dy, x)))
    want = y64 @ x64.T
    assert np.linalg.norm(dw.numpy() - want) < room(rows) * np.linalg.norm(want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,groups,n,k", [(4000, 1, 4000, 640), (3999, 1, 4001, 700), (7600, 3, 4000, 1500)])
def test_matmul_large_tiles(stream, dtype, rows, groups, n, k):
    """Scales of powers of two and as many tiles of 256 x 256 as compute units: the form with those; odd and even numbers of blocks, rows and
    columns that end inside a tile, also on odd addresses."""
    print("matmul, large tiles", dtype, rows, groups, n, k, flush=True)
    rng = np.random.default_rng(rows + k)
    check_matmul(stream, rng, rows, groups, groups, n, k, "e8m0", dtype, strides=n % 8 != 0)


def test_matmul_of_many_small_groups_by_many_columns(stream):
    """So many groups and columns that a launch cannot hold a workgroup for every 16 of a group's rows: a form with larger tiles takes it."""
    print("matmul, 4096 groups by 65536 columns", flush=True)
    rng = np.random.default_rng(12)
    rows, groups, experts, n, k = 16384, 4096, 2, 65536, 128
    offsets = some_groups(rng, rows, groups, skew=False)
    own = rng.integers(0, experts, groups).astype(np.int32)
    qa, sa, va = ref.quant_rows(rng.standard_normal((rows, k)).astype(np.float32), ref.FP32)
    qw, sw, vw = ref.quant_weights(rng.standard_normal((experts, n, k)).astype(np.float32), ref.FP32)
    A, SA, W, SW, off, og = (torch.from_numpy(v).cuda() for v in (qa, sa, qw, sw, offsets, own))
    y = torch.full((rows, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    ready()
    H.block_matmul(A.data_ptr(), SA.data_ptr(), rows, W.data_ptr(), SW.data_ptr(), experts, n, k, ref.FP32, y.data_ptr(), H.HCCL_DATA_TYPE_BFP16,
                   stream.cuda_stream, groups=groups, offsets=off.data_ptr(), expert_of_group=og.data_ptr())
    done(stream)
    assert bool(torch.isfinite(y).all())
    group = np.searchsorted(offsets, np.arange(rows), side="right") - 1
    for r in [0, rows - 1] + rng.integers(0, rows, 30).tolist():
        e = own[group[r]]
        m = ref.from_fp8(qw[e]) * np.repeat(vw[e], 128, 0)
        x = ref.rows_values(qa[r:r + 1], va[r:r + 1])
        want, size = x @ m.T, np.abs(x) @ np.abs(m).T
        assert close(y[r:r + 1].double().cpu().numpy(), want, 2 * (k + 5) * U * size, torch.bfloat16), r
    del y
    torch.cuda.empty_cache()


def test_matmul_offsets_and_owners_that_point_outside(stream):
    """Whatever the device's offsets and owners hold, no row outside is written and no weights outside are read."""
    rng = np.random.default_rng(8)
    qa, sa, _ = ref.quant_rows(rng.standard_normal((50, 128)).astype(np.float32), ref.FP32)
    qw, sw, _ = ref.quant_weights(rng.standard_normal((2, 64, 128)).astype(np.float32), ref.FP32)
    A, SA, W, SW = (torch.from_numpy(v).cuda() for v in (qa, sa, qw, sw))
    for off, own in (([-5, 20, 70, 2 ** 31 - 1, -(2 ** 31)], [0, 1, 1, 0]), ([0, 10, 20, 30, 50], [-1, 2, 7, 2 ** 31 - 1]), ([40, 30, 20, 10, 0], [0, 0, 1, 1]),
                     ([0, 50, 0, 50, 50], [0, 0, 0, 1])):
        y = Out(50, 64, torch.float32)
        o, g = torch.tensor(off, dtype=torch.int32, device="cuda"), torch.tensor(own, dtype=torch.int32, device="cuda")
        ready()
        H.block_matmul(A.data_ptr(), SA.data_ptr(), 50, W.data_ptr(), SW.data_ptr(), 2, 64, 128, ref.FP32, y.ptr, H.HCCL_DATA_TYPE_FP32,
                       stream.cuda_stream, groups=4, offsets=o.data_ptr(), expert_of_group=g.data_ptr())
        done(stream)
        y.get()


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("rows,groups,experts,n,k,dtype", [
    (1, 1, 1, 1, 1, "fp32"), (5, 1, 1, 64, 64, "bf16"), (200, 3, 3, 65, 130, "fp32"), (300, 70, 70, 40, 33, "fp16"), (513, 4, 4, 257, 300, "fp32"),
    (1000, 9, 9, 128, 520, "bf16"), (700, 12, 3, 100, 200, "fp32"), (2500, 2, 2, 600, 700, "fp32")])
def test_grad_weight(stream, kind, rows, groups, experts, n, k, dtype):
    rng = np.random.default_rng(rows + n)
    offsets = some_groups(rng, rows, groups)
    own = rng.integers(0, experts, groups).astype(np.int32) if groups != experts else None
    dy, x = (values(rng, (rows, c), torch.bfloat16) for c in (n, k))
    columns = H.block_columns(rows, groups)
    sdt = torch.float32 if kind == "fp32" else torch.uint8
    t = TYPE[dtype]
    qy, qx = (Out(c, columns, torch.uint8) for c in (n, k))
    sy, sx = (Out(columns // 128, c, sdt) for c in (n, k))
    off = torch.from_numpy(offsets).cuda()
    og = None if own is None else torch.from_numpy(own).cuda()
    ins = [v.cuda() for v in (dy, x)]
    first = torch.from_numpy(rng.standard_normal((experts * n, k))).to(t)
    dw, more = Out(experts * n, k, t), Out(experts * n, k, t).fill(first.cuda())
    ready()
    S = stream.cuda_stream
    for v, q, s, c in ((ins[0], qy, sy, n), (ins[1], qx, sx, k)):
        H.block_quant_columns(v.data_ptr(), H.HCCL_DATA_TYPE_BFP16, rows, c, groups, off.data_ptr(), KIND[kind], q.ptr, columns, s.ptr, S)
    for out, add in ((dw, False), (more, True)):
        H.block_matmul_grad_weight(qy.ptr, sy.ptr, qx.ptr, sx.ptr, columns, rows, n, k, KIND[kind], groups, off.data_ptr(), experts, out.ptr, dt(t), S,
                                   expert_of_group=None if og is None else og.data_ptr(), accumulate=add)
    done(stream)
    vals = []
    for v in (dy, x):
        codes, _, scale = ref.quant_columns(v.float().numpy(), offsets, KIND[kind])
        vals.append(ref.from_fp8(codes) * np.repeat(scale.T, 128, 1))
    at, want, size, long = 0, np.zeros((experts, n, k)), np.zeros((experts, n, k)), 0
    for g in range(groups):
        m = up128(int(offsets[g + 1] - offsets[g]))
        e = g if own is None else own[g]
        a, b = (v[:, at:at + m] for v in vals)
        want[e] += a @ b.T
        size[e] += np.abs(a) @ np.abs(b).T
        at += m
        long = max(long, at)
    room = 2 * (long + 3 * long // 128 + 2) * U * size
    assert close(dw.numpy().reshape(want.shape), want, room, t)
    f = first.double().numpy().reshape(want.shape)
    assert close(more.numpy().reshape(want.shape), want + f, room + U * (np.abs(f) + np.abs(want)), t)


@pytest.mark.parametrize("kind", ["fp32", "e8m0"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("groups", [0, 3])
def test_grad_weight_without_rows(stream, kind, dtype, groups):
    """No row at all, the operands absent: zeros, or with accumulate what was there.  groups 0: no offsets, one group of all rows."""
    print("grad weight without rows", kind, dtype, groups, flush=True)
    experts, n, k, t = max(1, groups), 130, 200, TYPE[dtype]
    first = torch.randn(experts * n, k, device="cuda").to(t)
    dw, more = Out(experts * n, k, t), Out(experts * n, k, t).fill(first)
    off = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    ready()
    for out, add in ((dw, False), (more, True)):
        H.block_matmul_grad_weight(None, None, None, None, H.block_columns(0, experts), 0, n, k, KIND[kind], experts, off.data_ptr() if groups else None,
                                   experts, out.ptr, dt(t), stream.cuda_stream, accumulate=add)
    done(stream)
    assert not dw.get().any() and torch.equal(more.get(), first)


def test_products_in_a_graph(stream):
    """Captured calls, replayed with the program's own work between: every replay is the eager result."""
    torch.manual_seed(4)
    T, E, k, W, N = 96, 8, 2, 256, 192
    x = torch.randn(T, W, device="cuda").bfloat16()
    logits = torch.randn(T, E, device="cuda")
    w = torch.randn(E, N, W, device="cuda").bfloat16()
    o = {n: torch.zeros(T, k, dtype=d, device="cuda") for n, d in (("expert", torch.int32), ("weights", torch.float32), ("row", torch.int32))}
    counts, offsets, loss = (torch.zeros(E + 1, dtype=torch.int32, device="cuda"), torch.zeros(E + 1, dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda"))
    need = H.expert_route_workspace(T, E)
    work = torch.zeros(max(16, need), dtype=torch.uint8, device="cuda")
    q, s = torch.zeros(T * k, W, dtype=torch.uint8, device="cuda"), torch.zeros(T * k, W // 128, device="cuda")
    wq, ws = torch.zeros(E, N, W, dtype=torch.uint8, device="cuda"), torch.zeros(E, 2, W // 128, device="cuda")
    y, out = torch.zeros(T * k, N, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")
    P = lambda v: v.data_ptr()  # noqa: E731
    BF, F = H.HCCL_DATA_TYPE_BFP16, H.HCCL_DATA_TYPE_FP32

    def step(S):
        H.expert_route(P(logits), F, T, E, k, P(o["expert"]), P(o["weights"]), P(o["row"]), P(counts), P(offsets), P(loss), P(work), need, S, renorm=True)
        H.expert_pack(P(x), BF, T, W, k, P(o["row"]), P(q), T * k, S, scales=P(s), scale_type=ref.FP32)
        H.block_quant_weights(P(w), BF, E, N, W, ref.FP32, P(wq), P(ws), None, None, S)
        H.block_matmul(P(q), P(s), T * k, P(wq), P(ws), E, N, W, ref.FP32, P(y), BF, S, groups=E, offsets=P(offsets))
        H.expert_combine(P(y), BF, T * k, N, T, k, P(o["row"]), P(o["weights"]), P(out), S)

    ready()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            step(stream.cuda_stream)
    for i in range(4):
        logits.copy_(torch.randn(T, E, device="cuda"))
        x.copy_(torch.randn(T, W, device="cuda"))
        out.zero_()
        ready()
        graph.replay()
        ready()
        got, got_loss = out.clone(), loss.clone()
        out.zero_()
        ready()
        step(stream.cuda_stream)
        done(stream)
        assert torch.equal(got, out) and torch.equal(got_loss, loss) and bool(out.any())


def test_an_error_of_another_hip_call_is_none_of_theirs(stream):
    """A HIP call that failed before, on the host and without harm: every operator succeeds, does all of its work, and leaves that error to
    whoever asks for it."""
    torch.manual_seed(5)
    T, E, k, W, N = 900, 16, 2, 256, 192                      # (a router's call of three launches)
    x, logits, w = torch.randn(T, W, device="cuda").bfloat16(), torch.randn(T, E, device="cuda"), torch.randn(E, N, W, device="cuda").bfloat16()
    need = H.expert_route_workspace(T, E)
    columns = H.block_columns(T * k, E)
    dw_in, dl_in = torch.randn(T, k, device="cuda"), torch.ones(1, device="cuda")
    BF, F, K, P = H.HCCL_DATA_TYPE_BFP16, H.HCCL_DATA_TYPE_FP32, ref.FP32, lambda v: v.data_ptr()  # noqa: E731
    u8, i32, f32, bf = torch.uint8, torch.int32, torch.float32, torch.bfloat16
    shapes = {"expert": (T, k, i32), "weights": (T, k, f32), "row": (T, k, i32), "counts": (1, E + 1, i32), "offsets": (1, E + 1, i32), "loss": (1, 1, f32),
              "d_logits": (T, E, f32), "q": (T * k, W, u8), "s": (T * k, 2, f32), "wq": (E * N, W, u8), "ws": (E * 2, 2, f32), "y": (T * k, N, bf),
              "out": (T, N, bf), "dx": (T * k, N, bf), "dweights": (T, k, f32), "yt": (N, columns, u8), "yts": (columns // 128, N, f32), "xt": (N, columns, u8),
              "xts": (columns // 128, N, f32), "grad": (E * N, N, f32)}

    def run():
        o = {n: torch.zeros(a, b, dtype=t, device="cuda") for n, (a, b, t) in shapes.items()}
        work = torch.zeros(need, dtype=u8, device="cuda")
        ready()
        S = stream.cuda_stream
        calls = (
            lambda: H.expert_route(P(logits), F, T, E, k, P(o["expert"]), P(o["weights"]), P(o["row"]), P(o["counts"]), P(o["offsets"]), P(o["loss"]), P(work),
                                   need, S),
            lambda: H.expert_route_grad(P(logits), F, T, E, k, P(o["expert"]), P(o["counts"]), P(dw_in), P(dl_in), P(o["d_logits"]), S),
            lambda: H.expert_pack(P(x), BF, T, W, k, P(o["row"]), P(o["q"]), T * k, S, scales=P(o["s"]), scale_type=K),
            lambda: H.block_quant_weights(P(w), BF, E, N, W, K, P(o["wq"]), P(o["ws"]), None, None, S),
            lambda: H.block_matmul(P(o["q"]), P(o["s"]), T * k, P(o["wq"]), P(o["ws"]), E, N, W, K, P(o["y"]), BF, S, groups=E, offsets=P(o["offsets"])),
            lambda: H.expert_combine(P(o["y"]), BF, T * k, N, T, k, P(o["row"]), P(o["weights"]), P(o["out"]), S),
            lambda: H.expert_combine_grad(P(o["out"]), P(o["y"]), BF, T * k, N, T, k, P(o["row"]), P(o["weights"]), P(o["dx"]), P(o["dweights"]), S),
            lambda: H.block_quant_columns(P(o["dx"]), BF, T * k, N, E, P(o["offsets"]), K, P(o["yt"]), columns, P(o["yts"]), S),
            lambda: H.block_quant_columns(P(o["y"]), BF, T * k, N, E, P(o["offsets"]), K, P(o["xt"]), columns, P(o["xts"]), S),
            lambda: H.block_matmul_grad_weight(P(o["yt"]), P(o["yts"]), P(o["xt"]), P(o["xts"]), columns, T * k, N, N, K, E, P(o["offsets"]), E, P(o["grad"]), F, S))
        return o, calls

    hip = H.lib()                                             # (the runtime that the library has loaded)
    want, calls = run()
    for call in calls:
        call()
    done(stream)
    got, calls = run()
    for call in calls:
        try:
            failed = hip.hipSetDevice(9999)                   # no such device
            assert failed != 0
            call()
            assert hip.hipPeekAtLastError() == failed
        finally:
            hip.hipGetLastError()
    done(stream)
    for name in shapes:
        assert torch.equal(got[name].view(u8), want[name].view(u8)) and bool(want[name].any()), name


# ---- addresses beyond 2^32 bytes ------------------------------------------------------------------------------------------------------

def test_exchange_beyond_32_bits(stream):
    """Rows 3 GB apart, tokens likewise."""
    W, far = 264, 1_600_000_000
    big = torch.empty(far * 2 + W, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(3, W, device="cuda").bfloat16()
    row = torch.tensor([[2], [0], [1]], dtype=torch.int32, device="cuda")
    y, dw = torch.empty(3, W, dtype=torch.bfloat16, device="cuda"), torch.empty(3, 1, device="cuda")
    w = torch.tensor([[1.0], [2.0], [4.0]], device="cuda")
    q, s = torch.empty(3, up128(W), dtype=torch.uint8, device="cuda"), torch.empty(3, 3, device="cuda")
    ready()
    S = stream.cuda_stream
    BF = H.HCCL_DATA_TYPE_BFP16
    H.expert_pack(x.data_ptr(), BF, 3, W, 1, row.data_ptr(), big.data_ptr(), 3, S, out_stride=far)
    H.expert_combine(big.data_ptr(), BF, 3, W, 3, 1, row.data_ptr(), w.data_ptr(), y.data_ptr(), S, x_stride=far)
    H.expert_pack(big.data_ptr(), BF, 3, W, 1, None, q.data_ptr(), 3, S, scales=s.data_ptr(), scale_type=ref.FP32, x_stride=far)
    H.expert_combine_grad(x.data_ptr(), big.data_ptr(), BF, 3, W, 3, 1, row.data_ptr(), w.data_ptr(), None, dw.data_ptr(), S, x_stride=far)
    done(stream)
    for t in range(3):
        assert torch.equal(big[int(row[t]) * far:int(row[t]) * far + W], x[t])
    assert torch.equal(y, (x.float() * w).bfloat16())
    codes, stored, _ = ref.quant_rows(x[[1, 2, 0]].float().cpu().numpy(), ref.FP32)
    assert np.array_equal(q.cpu().numpy(), codes) and np.array_equal(s.cpu().numpy(), stored)
    X = x.double().cpu().numpy()
    assert close(dw.cpu().numpy()[:, 0], (X * X).sum(1), (W + 1) * U * (X * X).sum(1))
    del big
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,experts,n", [(300, 3, 200_064), (600_000, 2, 64)])
def test_matmul_beyond_32_bits(stream, rows, experts, n):
    """Weights, or rows, of more than 4 GiB; the last expert's and the last rows' results."""
    k = 8192
    g = torch.Generator(device="cuda").manual_seed(6)
    a = torch.randint(0, 120, (rows, k), generator=g, device="cuda", dtype=torch.uint8)
    w = torch.randint(0, 120, (experts, n, k), generator=g, device="cuda", dtype=torch.uint8)
    nb = (n + 127) // 128
    sa, sw = torch.rand((rows, k // 128), generator=g, device="cuda"), torch.rand((experts, nb, k // 128), generator=g, device="cuda")
    cut = rows - rows // 3
    off = torch.tensor([0] + [cut] * (experts - 1) + [rows], dtype=torch.int32, device="cuda")
    y = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
    ready()
    H.block_matmul(a.data_ptr(), sa.data_ptr(), rows, w.data_ptr(), sw.data_ptr(), experts, n, k, ref.FP32, y.data_ptr(), H.HCCL_DATA_TYPE_BFP16,
                   stream.cuda_stream, groups=experts, offsets=off.data_ptr())
    done(stream)
    value = lambda q, s: q.view(torch.float8_e4m3fn).double() * s.double().repeat_interleave(128, -1)  # noqa: E731
    for lo, e in ((cut - 20, 0), (rows - 20, experts - 1)):
        x = value(a[lo:lo + 20], sa[lo:lo + 20])
        m = value(w[e, n - 64:], sw[e, torch.arange(n - 64, n, device="cuda") // 128])
        want = x @ m.T                                     # (all values positive: the sum of the magnitudes is the sum)
        assert close(y[lo:lo + 20, n - 64:].double().cpu().numpy(), want.cpu().numpy(), 2 * (k + 3 * k // 128 + 2) * U * want.cpu().numpy(), torch.bfloat16)
    del a, w, y
    torch.cuda.empty_cache()
