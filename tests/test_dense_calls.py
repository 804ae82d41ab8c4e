"""Calls of the operators around the routed experts that their documentation allows."""
from __future__ import annotations

import pytest

from test_dense_limits import ones
from test_dense_ops import F16

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
