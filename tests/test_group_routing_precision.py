"""MoeRoutingGroupTopK where its values cancel: group scores that are small sums of large c."""
from __future__ import annotations

import pytest

from test_dense_ops import F16, F32, normal, route_reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def same_choice(ops, logits, bias, K, G, TG, scoring):
    ids, _ = ops.MoeRoutingGroupTopK(logits.cuda(), bias.cuda(), K, G, TG, 2, scoring, True, 1.0, F32)
    rid, _ = route_reference(logits, bias, K, G, TG, 2, scoring, True, 1.0)
    bad = (ids.cpu() != rid).any(dim=1)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].flatten().tolist(), ids.cpu()[bad][:2].tolist(),
                           rid[bad][:2].tolist())


@pytest.mark.parametrize("B", [16.0, 32.0, 40.0, 64.0, 100.0, 1000.0])
def test_two_best_of_opposite_signs(ops, B):
    """Group 0's two best add up to a 3.8e-6 more or less than group 1's: the float64 sums decide, whatever fp32 makes of
    sums whose terms are of the size of B."""
    rows = [[6.1035e-6, 6.1035e-6, 9.1553e-6, 0.0], [0.0, 9.1553e-6, 6.1035e-6, 6.1035e-6], [1e-6, -1e-6, 2e-6, 1e-6],
            [0.3, -0.7, 0.3, -0.7], [0.3, -0.7, 0.30001, -0.70001]]
    same_choice(ops, torch.tensor(rows), torch.tensor([B, -B, B, -B]), 2, 2, 1, "sigmoid")


@pytest.mark.parametrize("T,E,G,TG,K", [(64, 64, 8, 4, 6), (64, 256, 8, 4, 8), (64, 256, 128, 9, 8), (64, 65, 13, 5, 6),
                                        (2100, 256, 128, 9, 4), (2100, 48, 8, 3, 5)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("B", [1.0, 16.0, 64.0, 1000.0, 1e6])
def test_group_scores_that_cancel(ops, T, E, G, TG, K, scoring, B):
    """Groups of nearly the same logits; one expert of each has the bias +B, the others -B, so that every group's two best
    add up to nearly the same small sum. In every third group the biases are small: scores of the same size whose fp32
    errors are not. A group is closed by finite biases."""
    size = E // G
    for n, (spread, dtype) in enumerate([(1e-5, F32), (1e-3, F32), (1e-2, F16)]):
        base = normal((T, 1, size), F32, 7 + n)
        logits = (base + spread * normal((T, G, size), F32, 17 + n)).reshape(T, E).to(dtype)
        bias = torch.full((G, size), -B)
        bias[:, 0] = B
        bias[::3] = 0.0
        if G > 4:
            bias[4] = -1e9
        same_choice(ops, logits, bias.reshape(E).contiguous(), K, G, TG, scoring)
