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
