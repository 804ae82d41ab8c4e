"""The activations and their gradients over the whole range of their types: digits in the tail of GELU, limits at
infinities."""
from __future__ import annotations

import math

import pytest

from test_dense_ops import BF16, F16, F32, F64, half_step

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def forward_of(ops, z, act):
    """act(z) in fp32 of 16-bit values z, as a product with the matrix [1]."""
    one = torch.ones((1, 1), dtype=z.dtype, device="cuda")
    return ops.MoeLinear(z.reshape(-1, 1).cuda(), one, activation=act, outDtype=F32).double().cpu().flatten()


def slope_of(ops, z, act, up=None):
    """act'(z) rounded to z's type, as the gradient of that product's rows."""
    pre = z.reshape(-1, 1).cuda()
    if act == "swiglu":
        pre = torch.cat([pre, up.reshape(-1, 1).cuda()], dim=1).contiguous()
        w = torch.eye(2, dtype=z.dtype, device="cuda")
        x = torch.zeros((z.numel(), 2), dtype=z.dtype, device="cuda")
    else:
        w = torch.ones((1, 1), dtype=z.dtype, device="cuda")
        x = torch.zeros((z.numel(), 1), dtype=z.dtype, device="cuda")
    dy = torch.ones((z.numel(), 1), dtype=z.dtype, device="cuda")
    return ops.MoeLinearGrad(dy, x, w, pre, act)[0].cpu()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gelu_keeps_its_digits_in_the_tail(ops, dtype):
    """z Phi(z), relative to itself down to -12.5, where Phi is 4e-36. 2^-20: the polynomial's error is below 2^-22, e^(-z^2/2)
    is within 3 ulp by the two-part exponent, and five roundings of 2^-24 follow."""
    z = torch.cat([torch.linspace(-12.5, 12.5, 20001), torch.linspace(-0.01, 0.01, 101)]).to(dtype)
    zd = z.double()
    ref = zd * 0.5 * torch.erfc(-zd / math.sqrt(2.0))
    got = forward_of(ops, z, "gelu")
    rel = ((got - ref).abs() / ref.abs().clamp(min=1e-300))[ref != 0]
    assert rel.max() <= 2.0**-20, (float(rel.max()), float(zd[ref != 0][rel.argmax()]))


def test_gelu_slope_keeps_its_digits_in_the_tail(ops):
    """Phi(z) + z phi(z), away from its zero at -0.7518, rounded to bf16. Both terms are within 2^-20 of themselves; below
    -1.5 their difference is above a fifth of the larger one."""
    z = torch.linspace(-12.5, -1.5, 5001).to(BF16)
    zd = z.double()
    ref = 0.5 * torch.erfc(-zd / math.sqrt(2.0)) + zd * torch.exp(-0.5 * zd * zd) / math.sqrt(2 * math.pi)
    got = slope_of(ops, z, "gelu").double().flatten()
    tol = half_step(ref, BF16) + ref.abs() * 6 * 2.0**-20 * (1 + 2.0**-8)
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (zd[bad][:4].tolist(), got[bad][:4].tolist(), ref[bad][:4].tolist())


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_slopes_have_their_limits_at_the_ends(ops, act, dtype):
    """A sum that is finite in fp32 may be infinite in pre: its slope is the limit, 1 or 0. NaN stays NaN (relu's is 0)."""
    big = torch.finfo(dtype).max
    z = torch.tensor([math.inf, big, big / 2, 1000.0, -1000.0, -big / 2, -big, -math.inf, math.nan], dtype=dtype)
    got = slope_of(ops, z, act).flatten()
    assert got[:4].tolist() == [1.0] * 4 and got[4:8].abs().max() == 0.0, got.tolist()
    assert act == "relu" or torch.isnan(got[8])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cols", [1, 8])  # the paths of any width and of whole vectors
def test_swiglu_slopes_have_their_limits_at_the_ends(ops, dtype, cols):
    big = torch.finfo(dtype).max
    gate = torch.tensor([math.inf, big, -big, -math.inf], dtype=dtype)
    up = torch.tensor([2.0, 2.0, 2.0, 2.0], dtype=dtype)
    pre = torch.cat([gate.reshape(-1, 1).expand(4, cols), up.reshape(-1, 1).expand(4, cols)], dim=1).contiguous().cuda()
    w = torch.eye(2 * cols, dtype=dtype, device="cuda")
    x = torch.zeros((4, 2 * cols), dtype=dtype, device="cuda")
    dy = torch.ones((4, cols), dtype=dtype, device="cuda")
    _, _, gb = ops.MoeLinearGrad(dy[2:], x[2:], w, pre[2:].contiguous(), "swiglu", gradBias=True)
    assert gb.abs().max() == 0.0, gb.tolist()  # silu(gate) and its slope are 0
    _, _, gb = ops.MoeLinearGrad(dy[:1], x[:1], w, pre[:1].contiguous(), "swiglu", gradBias=True)
    assert (gb[:cols] == 2.0).all() and torch.isinf(gb[cols:]).all(), gb.tolist()
