"""The torch.library registration of the operators around the routed experts: shapes on fake tensors here, gradients
through torch's differentiation, opcheck and compilation on the GPU."""
from __future__ import annotations

import importlib

import pytest

from conftest import PKG_NAME

torch = pytest.importorskip("torch")
tops = importlib.import_module(PKG_NAME + ".torch_ops")
op = torch.ops.moe_mi355x
F16, F32 = torch.float16, torch.float32


def meta(*shape, dtype=F16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_meta_shapes():
    x, w = meta(7, 64), meta(24, 64)
    ids, wt = op.MoeRoutingGroupTopK(meta(7, 16, dtype=F32), None, 3, weightsDtype=F32)
    assert (ids.shape, ids.dtype, wt.shape, wt.dtype) == ((7, 3), torch.int32, (7, 3), F32)
    assert op.MoeRoutingGroupTopKGrad(wt, meta(7, 16, dtype=F32), ids).shape == (7, 16)
    y, pre = op.MoeLinear(x, w, activation="swiglu", outDtype=F32, returnPre=True)
    assert (y.shape, y.dtype, pre.shape, pre.dtype) == ((7, 12), F32, (7, 24), F16)
    assert op.MoeLinear(x, w)[1].numel() == 0
    gx, gw, gb = op.MoeLinearGrad(meta(7, 24), x, w, None, "none", True, True, False)
    assert gx.shape == (7, 64) and gw.shape == (24, 64) and gb.numel() == 0
    geo, gwt = op.MoeCombineGrad(meta(7, 64), meta(7, 2, 64), meta(7, 2))
    assert geo.shape == (7, 2, 64) and gwt.shape == (7, 2)
    with pytest.raises(RuntimeError, match="MoeLinear: x must be"):
        op.MoeLinear(meta(7, 32), w)


def test_cpu_tensors_have_no_kernel():
    with pytest.raises(NotImplementedError):
        op.MoeLinear(torch.zeros(4, 64, dtype=F16), torch.zeros(8, 64, dtype=F16))
    with pytest.raises(NotImplementedError):
        op.MoeRoutingGroupTopK(torch.zeros(4, 8))


def leaf(shape, seed, sigma=1.0, dtype=F16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0, sigma, generator=g).requires_grad_(True)


def dense_step(x, gu, down, bias, residual):
    return tops.linear(tops.linear(x, gu, bias, activation="swiglu"), down, residual=residual)


@pytest.mark.gpu
def test_gradients_through_torch(ops):
    x, gu, down = leaf((33, 64), 1), leaf((80, 64), 2, 0.125), leaf((48, 40), 3, 0.15)
    bias, residual = leaf((80,), 4), leaf((33, 48), 5)
    y = dense_step(x, gu, down, bias, residual)
    dy = leaf((33, 48), 6).detach()
    y.backward(dy)
    want = [t.detach().double().requires_grad_(True) for t in (x, gu, down, bias, residual)]
    z = want[0] @ want[1].t() + want[3]
    g, u = z.chunk(2, dim=1)
    ref = (g * torch.sigmoid(g) * u) @ want[2].t() + want[4]
    ref.backward(dy.double())
    for name, a, b in zip(("x", "gate_up", "down", "bias", "residual"), (x, gu, down, bias, residual), want):
        assert a.grad.dtype == F16
        # roundings of 2^-11 each: hidden, pre, its gradient, dz, the result
        assert (a.grad.double() - b.grad).norm() / b.grad.norm() < 5 * 2.0**-11, name

    logits, eo = leaf((33, 16), 7, dtype=F32), leaf((33, 3, 48), 8)
    ids, w = op.MoeRoutingGroupTopK(logits, None, 3, scoring="sigmoid", scale=2.0)
    assert not ids.requires_grad
    op.MoeCombine(eo, ids, w, 3).backward(dy)
    l64, e64 = logits.detach().double().requires_grad_(True), eo.detach().double().requires_grad_(True)
    s = torch.sigmoid(l64).gather(1, ids.long())
    ((e64 * (2.0 * s / s.sum(dim=1, keepdim=True)).unsqueeze(2)).sum(dim=1) * dy.double()).sum().backward()
    assert (logits.grad.double() - l64.grad).norm() / l64.grad.norm() < 3 * 2.0**-11
    assert (eo.grad.double() - e64.grad).norm() / e64.grad.norm() < 2 * 2.0**-11


@pytest.mark.gpu
def test_gradient_rules(ops):
    x, w = leaf((5, 16), 1), leaf((8, 16), 2)
    with pytest.raises(RuntimeError, match="returnPre"):
        op.MoeLinear(x, w, activation="silu")[0].sum().backward()
    y, pre = op.MoeLinear(x, w, activation="silu", returnPre=True)
    with pytest.raises(RuntimeError, match="through pre"):
        (y.sum() + pre.sum()).backward()
    frozen = w.detach()
    x.grad = None
    tops.linear(x, frozen, activation="gelu").sum().backward()
    assert x.grad is not None
    y32 = tops.linear(x, w, outDtype=F32)
    assert y32.dtype == F32
    y32.sum().backward()
    assert w.grad.dtype == F16


@pytest.mark.gpu
def test_opcheck_and_compile(ops):
    x, w, logits = leaf((9, 64), 1), leaf((32, 64), 2), leaf((9, 16), 3, dtype=F32)
    utils = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(op.MoeLinear, (x, w, None, None, "swiglu", None, True), test_utils=utils)
    torch.library.opcheck(op.MoeRoutingGroupTopK, (logits, None, 3), test_utils=utils)
    compiled = torch.compile(lambda a, b: tops.linear(a, b, activation="swiglu"), backend="aot_eager", fullgraph=True)
    with torch.no_grad():
        assert torch.equal(compiled(x, w), tops.linear(x, w, activation="swiglu"))


@pytest.mark.gpu
def test_captured_training_step_replays_on_changed_inputs(ops):
    """Forward and backward of a router, its experts' combine and a dense expert in one graph, against eager steps on
    leaves of their own."""
    shapes = dict(logits=((40, 16), F32), eo=((40, 3, 64), F16), x=((40, 64), F16), gu=((96, 64), F16), down=((64, 48), F16),
                  dy=((40, 64), F16))

    def fresh(seed):
        return {k: leaf(s, seed + n, 0.25, d).detach() for n, (k, (s, d)) in enumerate(shapes.items())}

    def step(v):
        leaves = [v[k].requires_grad_(True) for k in ("logits", "eo", "x", "gu", "down")]
        ids, w = op.MoeRoutingGroupTopK(leaves[0], None, 3, 4, 2, 2, "softmax")
        y = tops.linear(tops.linear(leaves[2], leaves[3], activation="swiglu"), leaves[4],
                        residual=op.MoeCombine(leaves[1], ids, w, 3))
        return (y.detach(),) + torch.autograd.grad(y, leaves, v["dy"])

    static = fresh(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for seed in range(100, 130, 10):
        now = fresh(seed)
        with torch.no_grad():
            for k, t in static.items():
                t.copy_(now[k])
        graph.replay()
        eager = step(now)
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert torch.equal(a, b)
