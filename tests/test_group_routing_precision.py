"""MoeRoutingGroupTopK and its gradient where their values cancel: group scores that are small sums of large c, and the
gradients of rows that one expert dominates."""
from __future__ import annotations

import pytest

from test_dense_ops import F16, F32, F64, half_step, normal, route_grad_reference, route_reference

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


def dominated(T, E, seed, gap):
    """Logits N(0, 1), but for one expert of every row, which stands `gap` above the others."""
    logits = normal((T, E), F32, seed)
    at = torch.randint(0, E, (T,), generator=torch.Generator().manual_seed(seed + 1))
    logits[torch.arange(T), at] += gap
    return logits


@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True)])
@pytest.mark.parametrize("E,K", [(8, 2), (64, 6), (200, 20), (256, 8)])
@pytest.mark.parametrize("gap", [0.0, 6.0, 12.0, 20.0])
def test_gradient_of_dominated_rows(ops, scoring, renorm, E, K, gap):
    """dl_k = p_k sum_j p_j (g_k - g_j): every term counts, also where p_k is nearly 1 and g_k nearly the mean of g.

    Scores in fp32, relative to the largest: the exponent d = x - top rounds by |d| 2^-24, expf and a product are within
    4 ulp, so p_k p_j is within 2 (|d| + 16) 2^-24 of itself, |d| <= gap + 10 here; sums are in float64, here and in the
    reference: each of the mean's up to K + 5 roundings moves the difference by 2^-53 of the largest |g|, times p_k."""
    T = 70
    logits = dominated(T, E, 3, gap if scoring == "softmax" else -gap)
    if scoring == "sigmoid":  # far below zero a sigmoid is e^x
        logits = -logits.abs() - 5.0
    ids = logits.topk(K, dim=1)[1].to(torch.int32)
    gw = normal((T, K), F32, 5)
    grad = ops.MoeRoutingGroupTopKGrad(gw.cuda(), logits.cuda(), ids.cuda(), scoring, renorm, 2.5)
    ref = route_grad_reference(gw, logits, ids, scoring, renorm, 2.5)
    lg, at = logits.double(), ids.long()
    s = torch.softmax(lg, dim=1) if scoring == "softmax" else torch.sigmoid(lg)
    g = torch.zeros(T, E, dtype=F64).scatter_(1, at, 2.5 * gw.double())
    if renorm:
        chosen = torch.zeros(T, E, dtype=F64).scatter_(1, at, 1.0)
        p = s * chosen / (s * chosen).sum(dim=1, keepdim=True)
    else:
        p = s
    terms = p * (p.unsqueeze(1) * (g.unsqueeze(2) - g.unsqueeze(1)).abs()).sum(dim=2)
    sums = 2 * (K + 5) * 2.0**-53 * p * g.abs().amax(dim=1, keepdim=True)
    tol = terms * (2 * (gap + 10) + 32) * 2.0**-24 + sums + half_step(ref, F32)
    out = grad.double().cpu()
    bad = ~((out - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), out[bad][:4].tolist(), ref[bad][:4].tolist(), tol[bad][:4].tolist())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_gradient_of_a_single_renormalised_weight_is_zero(ops, scoring):
    """The weight is scale, whatever the logit."""
    logits, gw = normal((500, 64), F32, 1), normal((500, 1), F32, 2)
    ids = logits.argmax(dim=1, keepdim=True).to(torch.int32)
    grad = ops.MoeRoutingGroupTopKGrad(gw.cuda(), logits.cuda(), ids.cuda(), scoring, True, 2.5)
    assert (grad == 0).all(), float(grad.abs().max())


@pytest.mark.parametrize("T,E,G,TG,K", [(5, 48, 1, 1, 6), (5, 65, 5, 2, 20), (40, 200, 8, 3, 8), (70, 256, 1, 1, 8),
                                        (70, 256, 8, 4, 40), (5, 256, 1, 1, 256), (2100, 256, 8, 4, 8), (2100, 64, 1, 1, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_more_scores_than_fp32_tells_apart(ops, T, E, G, TG, K, scoring):
    """Equal scores, runs of equal ones, and biases beside which the scores keep few bits: the float64 values decide among
    all of a row's experts, the lowest index among equal ones."""
    logits = normal((T, E), F32, 23)
    logits[::3] = (logits[::3] * 2).round() / 2
    logits[1::7] = 0.0
    logits[2::11, ::2] = float("-inf")
    logits[3::13, 1:] = float("-inf")
    steps = (torch.arange(E) % 5).float() / 4
    signs = torch.where(torch.arange(E) % 2 == 0, 40.0, -40.0)
    for bias in (torch.zeros(E), torch.full((E,), 1e4), torch.full((E,), -3e3), steps, signs, 1e5 + signs):
        same_choice(ops, logits, bias, K, G, TG, scoring)
