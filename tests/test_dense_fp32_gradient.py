"""The gradient of an fp32 result (the router's logits): nothing of it vanishes or overflows in the operands' 16 bits."""
from __future__ import annotations

import importlib
import math

import pytest

from conftest import PKG_NAME
from test_dense_ops import BF16, F16, F32, F64, U32, act_reference, check, half_step, normal

torch = pytest.importorskip("torch")
tops = importlib.import_module(PKG_NAME + ".torch_ops")
opsm = importlib.import_module(PKG_NAME + ".ops")
pytestmark = pytest.mark.gpu


def exact_gradients(dy, x, w, pre, act):
    dz = dy.double()
    if pre is not None:
        z = pre.double().requires_grad_(True)
        dz, = torch.autograd.grad(act_reference(z, act), z, dz)
    return dz, dz @ w.double(), dz.t() @ x.double(), dz.sum(dim=0)


def grad32_check(ops, T, N, H, dtype, act="none", dy_scale=1.0, x_scale=1.0, w_scale=1.0, transposed=False, seed=0):
    """fp16's dz is scaled by a power of two that takes its largest value to [2^14, 2^15): values from 2^-28 of that on
    round by 2^-11 of themselves, smaller ones by half the type's smallest step, 2^-39 of the largest. bf16's rounds by 2^-8."""
    Z = 2 * N if act == "swiglu" else N
    dy = normal((T, N), F32, seed) * dy_scale
    x, w = normal((T, H), dtype, seed + 1, x_scale), normal((Z, H), dtype, seed + 2, w_scale)
    pre = None if act == "none" else normal((T, Z), dtype, seed + 3, 1.5)
    wd = w.t().contiguous().cuda().t() if transposed else w.cuda()
    gx, gw, gb = ops.MoeLinearGrad(dy.cuda(), x.cuda(), wd, None if pre is None else pre.cuda(), act, gradBias=True)
    assert gx.dtype == gw.dtype == gb.dtype == dtype
    dz, rx, rw, rb = exact_gradients(dy, x, w, pre, act)
    fp = torch.zeros_like(dz)
    if pre is not None:  # the slopes' own rounding, relative to their factors
        z = pre.double()
        fp = (1 + z.abs()) * (torch.cat([dy, dy], 1).double().abs() * (1 + z.abs().roll(N, 1)) if act == "swiglu"
                              else dy.double().abs() * 2) * 2 * 4 * 2.0**-23
    dzt = fp + (dz.abs() * 2.0**-8 if dtype == BF16 else dz.abs() * 2.0**-11 + dz.abs().max() * 2.0**-39)
    for name, got, ref, tol in (
            ("grad_x", gx, rx, dzt @ w.double().abs() + (Z + 1) * U32 * (dz.abs() @ w.double().abs())),
            ("grad_weight", gw, rw, dzt.t() @ x.double().abs() + (T + 1) * U32 * (dz.abs().t() @ x.double().abs())),
            ("grad_bias", gb, rb, (T + 1) * U32 * dz.abs().sum(dim=0) + fp.sum(dim=0))):
        if dtype == F16:  # a result of 65520 and more rounds to infinity (half a step past 65504), tol more or less
            inf = got.double().cpu() == ref.sign() * math.inf
            assert (inf | (ref.abs() - tol < 65520)).all() and (~inf | (ref.abs() + tol >= 65520)).all(), (name, T, N, H, act)
            ref, got = torch.where(inf, 0.0, ref), torch.where(inf.cuda(), 0.0, got)
        check(got, ref, tol + half_step(ref.abs() + tol, dtype), (name, T, N, H, act))


@pytest.mark.parametrize("T,N,H,act,transposed", [
    (1, 8, 64, "none", False), (500, 256, 512, "none", True), (300, 64, 136, "none", False), (37, 13, 65, "none", True),
    (37, 13, 65, "none", False), (130, 40, 72, "silu", False), (129, 33, 100, "swiglu", False), (70, 48, 64, "swiglu", True),
    (70, 7, 40, "gelu", True), (2100, 256, 1024, "none", True)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_fp32_gradients(ops, dtype, T, N, H, act, transposed):
    grad32_check(ops, T, N, H, dtype, act, transposed=transposed)
    grad32_check(ops, T, N, H, dtype, act, 1e-9, 300.0, 300.0, transposed, 10)  # below fp16's smallest value
    grad32_check(ops, T, N, H, dtype, act, 1e7, 1e-4, 1e-4, transposed, 20)  # above its largest


def test_fp32_gradients_on_large_tiles(ops):
    """2048 x 2048 x 2048 on the kernels of large tiles: sampled rows against 64 bits, with gradients of 1e-8."""
    T = N = H = 2048
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda shape, s, t: torch.empty(shape, dtype=t, device="cuda").normal_(0, s, generator=g)  # noqa: E731
    dy, x, w = new((T, N), 1e-8, F32), new((T, H), 30.0, F16), new((N, H), 30.0, F16)
    gx, gw, _ = ops.MoeLinearGrad(dy, x, w)
    dz = dy.double()
    dzt = dz.abs() * 2.0**-11 + dz.abs().max() * 2.0**-39
    at = torch.tensor([0, 1, 255, 256, T // 2, T - 1], device="cuda")
    ref = dz[at] @ w.double()
    tol = dzt[at] @ w.double().abs() + N * U32 * (dz[at].abs() @ w.double().abs())
    check(gx[at], ref.cpu(), (tol + half_step(ref.abs() + tol, F16)).cpu(), "grad_x")
    ref = dz[:, at].t() @ x.double()
    tol = dzt[:, at].t() @ x.double().abs() + T * U32 * (dz[:, at].abs().t() @ x.double().abs())
    check(gw[at], ref.cpu(), (tol + half_step(ref.abs() + tol, F16)).cpu(), "grad_weight")


def test_torch_gradient_of_fp32_logits_keeps_small_and_large_values(ops):
    """The router's path: y = linear(x, w_gate.t(), outDtype=float32), whose gradient arrives in fp32. One rounding of 2^-11
    in dz and one in the result, each at most that relative in the norm; a result below 2^-14 rounds by up to 2^-25 instead,
    half of fp16's smallest step, which is 2^-25 sqrt(values) in the norm."""
    for dy_scale, s in ((1e-9, 300.0), (1e7, 1e-4)):
        x = normal((400, 128), F16, 1, s).cuda().requires_grad_(True)
        w = normal((64, 128), F16, 2, s).cuda().requires_grad_(True)
        dy = (normal((400, 64), F32, 3) * dy_scale).cuda()
        tops.linear(x, w, outDtype=F32).backward(dy)
        for got, ref in ((x.grad, dy.double() @ w.double()), (w.grad, dy.double().t() @ x.double())):
            inf = ref.abs() >= 65000  # near 65520, from where a result rounds to infinity
            assert (got[inf].abs() >= 64900).all() and inf.double().mean() < 0.01
            err, ref = torch.where(inf, 0.0, got.double() - ref), torch.where(inf, 0.0, ref)
            assert err.norm() < 2 * 2.0**-11 * ref.norm() + 2.0**-25 * ref.numel()**0.5, dy_scale


def test_fp32_gradients_that_are_not_finite_or_zero(ops):
    x, w = normal((40, 64), F16, 1).cuda(), normal((24, 64), F16, 2).cuda()
    dy = normal((40, 24), F32, 3).cuda() * 1e-8
    want = ops.MoeLinearGrad(dy, x, w)[0]
    spoilt = dy.clone()
    spoilt[3, 5], spoilt[7, 0] = math.nan, math.inf
    got = ops.MoeLinearGrad(spoilt, x, w)[0]
    rows = torch.isfinite(got).all(dim=1)
    assert not rows[3] and not rows[7] and rows.sum() == 38
    assert torch.equal(got[rows], want[rows])  # the scale is the finite values'
    for g in ops.MoeLinearGrad(torch.zeros_like(dy), x, w, gradBias=True):
        assert (g == 0).all()
    gx, gw, gb = ops.MoeLinearGrad(dy[:0], x[:0], w, gradBias=True)
    assert gx.shape == (0, 64) and (gw == 0).all() and (gb == 0).all()


def test_fp32_gradients_of_strided_rows_and_replays(ops):
    x, w = normal((50, 64), F16, 1).cuda(), normal((20, 64), F16, 2).cuda()
    wide = normal((50, 33), F32, 3).cuda() * 1e-7
    want = ops.MoeLinearGrad(wide[:, 5:25].contiguous(), x, w, gradBias=True)
    for a, b in zip(ops.MoeLinearGrad(wide[:, 5:25], x, w, gradBias=True), want):
        assert torch.equal(a, b)
    static = wide.clone()
    ops.MoeLinearGrad(static[:, 5:25], x, w, gradBias=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.MoeLinearGrad(static[:, 5:25], x, w, gradBias=True)
    for k in range(4):
        static.copy_(wide * 10.0**(3 * k))
        graph.replay()
        eager = ops.MoeLinearGrad(static[:, 5:25].contiguous(), x, w, gradBias=True)
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b), k


def test_fp32_gradient_of_the_other_type_is_refused(ops):
    c = lambda *shape, dtype=F16: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    for dtype in (BF16, F64):
        with pytest.raises(opsm.MoeError) as e:
            ops.MoeLinearGrad(c(4, 8, dtype=dtype), c(4, 64), c(8, 64))
        assert e.value.status == 4
