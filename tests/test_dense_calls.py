"""Calls of the operators around the routed experts that their documentation allows."""
from __future__ import annotations

import pytest

from test_dense_limits import ones
from test_dense_ops import F16, F32

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [(1 << 24) + 3, (1 << 25) + 5, (1 << 26) + 9])
def test_combine_gradient_of_as_many_tokens_as_the_combine(ops, T):
    H, K = 8, 1
    eo, dy, w = ones((T, K, H), 1), ones((T, H), 2), ones((T, K), 3)
    y = ops.MoeCombine(eo, None, w, K)
    assert torch.equal(y, eo[:, 0] * w)
    geo, gw = ops.MoeCombineGrad(dy, eo, w)
    assert torch.equal(geo[:, 0], dy * w)
    assert torch.equal(gw[:, 0], (dy * eo[:, 0]).float().sum(dim=1).to(F16))


def test_results_are_seen_by_dispatch_modes(ops):
    """What a mode that follows torch's calls (a memory tracker) sees of an operator is its allocations."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.shapes = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if isinstance(out, torch.Tensor):
                self.shapes.append(tuple(out.shape))
            return out

    x, w, logits = ones((6, 64), 1), ones((40, 64), 2), ones((6, 16), 3, F32)
    with Seen() as seen:
        y = ops.MoeLinear(x, w)
        ids, wt = ops.MoeRoutingGroupTopK(logits, None, 3)
        gx, gw, _ = ops.MoeLinearGrad(y, x, w)
        geo, _ = ops.MoeCombineGrad(x, ones((6, 2, 64), 4), wt[:, :2].contiguous())
    for shape in ((6, 40), (6, 3), (6, 64), (40, 64), (6, 2, 64)):
        assert shape in seen.shapes, (shape, seen.shapes)


@pytest.mark.parametrize("T,N,H,transposed", [(4, 72, 8192, True), (4, 72, 8192, False), (130, 72, 8192, False),
                                              (40, 130, 4100, True)])
def test_split_sums_are_in_the_workspace_and_in_one_order(ops, T, N, H, transposed):
    """Where the plan splits k (all but few aligned rows of a weight by rows), the pieces' sums are in the workspace, within
    it, and every call adds them alike."""
    w = torch.randn((H, N) if transposed else (N, H), device="cuda", dtype=F16)
    w, x = w.t() if transposed else w, torch.randn((T, H), device="cuda", dtype=F16)
    need = ops.linear_workspace_bytes(T, N, H)
    got = []
    for _ in range(3):
        ws = torch.full((need + 256,), 0x7f, dtype=torch.uint8, device="cuda")
        got.append(ops.MoeLinear(x, w, outDtype=F32, workspace=ws))
        assert (ws[need:] == 0x7f).all()
        if transposed or T > 64:
            assert (ws[:need] != 0x7f).sum() > T * N * 4
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    ref = x.double() @ w.double().t()
    tol = (H + 1) * 2.0**-24 * (x.double().abs() @ w.double().abs().t())
    assert ((got[0].double() - ref).abs() <= tol + 2.0**-24 * ref.abs()).all()


@pytest.mark.parametrize("T,N,H,transposed", [(4097, 2056, 72, False), (3001, 3000, 200, False), (2049, 4104, 1032, True),
                                              (8191, 1400, 136, False), (4099, 1032, 1000, True), (260, 33000, 96, False),
                                              (300, 520, 4096, False), (1000, 733, 1056, True)])
def test_every_value_of_large_products(ops, T, N, H, transposed):
    """Operands -1, 0 and 1: sums below 2^24 are whole in fp32 in any order, so a lost or repeated term shows anywhere."""
    x, w, dy = ones((T, H), 1), ones((H, N) if transposed else (N, H), 2), ones((T, N), 3)
    w = w.t() if transposed else w
    assert torch.equal(ops.MoeLinear(x, w, outDtype=F32), x.float() @ w.float().t())
    gx, gw, gb = ops.MoeLinearGrad(dy, x, w, gradBias=True)
    assert torch.equal(gx, (dy.float() @ w.float()).to(F16))
    assert torch.equal(gw, (dy.float().t() @ x.float()).to(F16))
    assert torch.equal(gb, dy.float().sum(dim=0).to(F16))
