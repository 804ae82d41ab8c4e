"""The operators around the routed experts: MoeRoutingGroupTopK, MoeLinear, MoeCombineGrad and the gradients, against
plain implementations in 64 bits.

Tolerances, from the arithmetic alone:
  a rounding to type t is off by at most eps(t) / 2 relative (fp16 2^-11, bf16 2^-8, fp32 2^-24), and by half the smallest
  subnormal step where the value is below the normal range (fp16: 2^-25);
  an fp32 sum of n products in any order is off by at most n 2^-24 times the sum of their magnitudes;
  expf, tanhf, erfcf and a division are counted with 4 * 2^-23 relative together (their documented errors are 1-4 ulp).
"""
from __future__ import annotations

import importlib
import itertools
import math

import pytest

from conftest import PKG_NAME

torch = pytest.importorskip("torch")
opsm = importlib.import_module(PKG_NAME + ".ops")
MoeError = opsm.MoeError
gpu = pytest.mark.gpu
F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
U32 = 2.0**-24
FN = 4 * 2.0**-23
NEG = float("-inf")


def half_step(t, dtype):
    """The most that rounding the values `t` (float64) to dtype moves them."""
    eps = torch.finfo(dtype).eps / 2
    return t.abs() * eps + (2.0**-25 if dtype == F16 else 1e-38)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(shape, dtype, seed, sigma=1.0):
    return (torch.randn(shape, generator=gen(seed), dtype=F32) * sigma).to(dtype)


def check(out, ref, tol, tag=""):
    out = out.double().cpu()
    assert out.shape == ref.shape, (tag, out.shape, ref.shape)
    bad = ~((out - ref).abs() <= tol)
    assert not bad.any(), (tag, int(bad.sum()), bad.nonzero()[:4].tolist(), out[bad][:4].tolist(), ref[bad][:4].tolist())


# ---------------------------------------------------------------------------------------------------------------------
# routing from logits
# ---------------------------------------------------------------------------------------------------------------------


def route_reference(logits, bias, K, G, TG, GT, scoring, renorm, scale):
    """Row by row in Python floats (64 bits), experts picked one after another."""
    T, E = logits.shape
    size = E // G
    ids, ws = [], []
    for row in logits.double().tolist():
        open_ = [v > NEG for v in row]
        top = max((v for v, o in zip(row, open_) if o), default=0.0)
        s = [0.0] * E
        for e, (v, o) in enumerate(zip(row, open_)):
            if o:
                if scoring == "sigmoid":
                    s[e] = 1.0 / (1.0 + math.exp(-v)) if v > -700 else 0.0
                else:
                    s[e] = 1.0 if v == top else math.exp(v - top)
        if scoring == "softmax":
            total = sum(s) or 1.0
            s = [v / total for v in s]
        c = [NEG] * E
        for e in range(E):
            if open_[e]:
                v = s[e] + (float(bias[e]) if bias is not None else 0.0)
                c[e] = v if v > NEG else NEG
        if TG < G:
            score = []
            for g in range(G):
                best = sorted((v for v in c[g * size:(g + 1) * size] if v > NEG), reverse=True)
                score.append(sum(best[:GT]) if best else NEG)
            keep = sorted(range(G), key=lambda g: (-score[g], g))[:TG]
            c = [v if e // size in keep else NEG for e, v in enumerate(c)]
        order = sorted(range(E), key=lambda e: (-c[e], e))[:K]
        pick = [e if c[e] > NEG else -1 for e in order]
        w = [s[e] if e >= 0 else 0.0 for e in pick]
        if renorm:  # s > 0 for every finite logit, so the quotient is taken in logarithms, where nothing underflows
            lw = [row[e] if scoring == "softmax" else min(row[e], 0.0) - math.log1p(math.exp(-abs(row[e])))
                  for e in pick if e >= 0]
            q = [1.0 if v == max(lw) else math.exp(v - max(lw)) for v in lw]
            w = [v / sum(q) for v in q] + [0.0] * (K - len(q))
        ids.append(pick)
        ws.append([v * scale for v in w])
    return torch.tensor(ids, dtype=torch.int32).view(T, K), torch.tensor(ws, dtype=F64).view(T, K)


def route_grad_reference(gw, logits, ids, scoring, renorm, scale):
    lg = logits.double()
    shut = ~(lg > NEG)
    empty = shut.all(dim=1, keepdim=True)
    leaf = torch.where(shut, 0.0, lg).requires_grad_(True)
    if renorm:  # a softmax over the picks' log scores: the same quotient, where nothing underflows
        ok = (ids >= 0) & (ids < lg.shape[1])
        at = ids.long().clamp(0, lg.shape[1] - 1)
        ok &= ~shut.gather(1, at)
        v = leaf.gather(1, at)
        v = torch.nn.functional.logsigmoid(v) if scoring == "sigmoid" else v
        none = ~ok.any(dim=1, keepdim=True)
        w = torch.softmax(torch.where(none, 0.0, torch.where(ok, v, NEG)), dim=1)
        grad, = torch.autograd.grad((torch.where(ok, w, 0.0) * scale * gw.double()).sum(), leaf)
        return torch.where(shut, 0.0, grad)
    if scoring == "sigmoid":
        s = torch.where(shut, 0.0, torch.sigmoid(leaf))
    else:
        s = torch.where(empty, 0.0, torch.softmax(torch.where(empty, 0.0, leaf.masked_fill(shut & ~empty, NEG)), dim=1))
    ok = (ids >= 0) & (ids < lg.shape[1])
    w = torch.where(ok, s.gather(1, ids.long().clamp(0, lg.shape[1] - 1)), 0.0)
    grad, = torch.autograd.grad((w * scale * gw.double()).sum(), leaf)
    return torch.where(shut, 0.0, grad)


ROUTES = [  # E, K, groups, top_groups, group_top
    (1, 1, 1, 1, 1), (2, 2, 1, 1, 1), (7, 3, 1, 1, 2), (16, 2, 4, 2, 1), (16, 16, 1, 1, 1), (24, 5, 8, 3, 2),
    (33, 4, 3, 2, 2), (64, 6, 1, 1, 1), (64, 6, 8, 3, 1), (65, 6, 13, 5, 2), (128, 8, 128, 9, 2), (160, 6, 8, 3, 1),
    (255, 9, 5, 4, 2), (256, 8, 8, 4, 2), (256, 256, 1, 1, 1), (256, 40, 2, 1, 1)]


@gpu
@pytest.mark.parametrize("E,K,G,TG,GT", ROUTES)
@pytest.mark.parametrize("scoring,renorm", list(itertools.product(("softmax", "sigmoid"), (True, False))))
def test_group_routing_against_the_definition(ops, E, K, G, TG, GT, scoring, renorm):
    for n, (T, dtype, with_bias) in enumerate([(1, F32, True), (37, F32, False), (50, F16, True), (33, BF16, False)]):
        logits = normal((T, E), dtype, 100 + n, 1.5)
        if n:
            shut = torch.rand((T, E), generator=gen(n)) < 0.2
            shut[3] = True  # a padded row
            shut[4, 1:] = True
            logits = logits.masked_fill(shut, NEG)
            logits[5] = torch.finfo(dtype).min  # masked by the type's lowest value: equal, available
            logits[6, E // 2] = float("nan")
            logits[7] = 0.25  # all equal
        bias = (torch.rand(E, generator=gen(50 + n)) - 0.5) * 0.2 if with_bias else None
        ids, w = ops.MoeRoutingGroupTopK(logits.cuda(), bias.cuda() if with_bias else None, K, G, TG, GT, scoring, renorm,
                                         2.5, F32 if n % 2 else F16)
        rid, rw = route_reference(logits, bias, K, G, TG, GT, scoring, renorm, 2.5)
        assert torch.equal(ids.cpu(), rid), (n, (ids.cpu() != rid).nonzero()[:4])
        check(w, rw, half_step(rw, w.dtype) + rw.abs() * FN)
        gw = normal((T, K), (F32, F16, BF16, F32)[n], 200 + n)
        grad = ops.MoeRoutingGroupTopKGrad(gw.cuda(), logits.cuda(), ids, scoring, renorm, 2.5)
        ref = route_grad_reference(gw, logits, rid, scoring, renorm, 2.5)
        # s, the K-term mean and the difference each round relative to the largest |g| s they are made of
        s_max = 2.5 * gw.double().abs().amax(dim=1, keepdim=True)
        check(grad, ref, half_step(ref, dtype) + s_max * (K + E / 16 + 20) * 2.0**-23)


@gpu
def test_group_routing_rows_of_a_padded_tensor_and_closed_experts(ops):
    wide = normal((70, 80), F32, 1).cuda()
    logits = wide[:, 3:67]
    bias = torch.zeros(64)
    bias[5], bias[9], bias[11] = NEG, float("nan"), float("inf")  # two experts switched off, one always first
    a = ops.MoeRoutingGroupTopK(logits, bias.cuda(), 6, 4, 2, 2, "sigmoid", True, 1.0, F32)
    b = ops.MoeRoutingGroupTopK(logits.contiguous(), bias.cuda(), 6, 4, 2, 2, "sigmoid", True, 1.0, F32)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    rid, rw = route_reference(logits.cpu(), bias, 6, 4, 2, 2, "sigmoid", True, 1.0)
    assert torch.equal(a[0].cpu(), rid)
    assert not ((rid == 5) | (rid == 9)).any() and (rid[:, 0] == 11).all()
    gw = normal((70, 6), F32, 2).cuda()
    assert torch.equal(ops.MoeRoutingGroupTopKGrad(gw, logits, a[0]),
                       ops.MoeRoutingGroupTopKGrad(gw, logits.contiguous(), a[0]))


@gpu
def test_group_routing_ties_in_fp32_scores_are_ordered_by_the_logits(ops):
    """Logits a last bit apart have sigmoids that agree in fp32: the choice is still the definition's."""
    base = torch.linspace(3, 9, 40).view(-1, 1).repeat(1, 64)
    step = torch.arange(64, dtype=F32)[torch.randperm(64, generator=gen(3))]
    logits = torch.nextafter(base, torch.tensor(100.0))
    for _ in range(3):
        logits = torch.where(step % 4 > 0, torch.nextafter(logits, torch.tensor(100.0)), logits)
        step = step - (step % 4 > 0).float()
    for scoring in ("sigmoid", "softmax"):
        ids, _ = ops.MoeRoutingGroupTopK(logits.cuda(), None, 8, 1, 1, 1, scoring)
        rid, _ = route_reference(logits, None, 8, 1, 1, 1, scoring, True, 1.0)
        assert torch.equal(ids.cpu(), rid)
        bias = torch.full((64,), 0.125)
        ids, _ = ops.MoeRoutingGroupTopK(logits.cuda(), bias.cuda(), 8, 8, 4, 2, scoring)
        rid, _ = route_reference(logits, bias, 8, 8, 4, 2, scoring, True, 1.0)
        assert torch.equal(ids.cpu(), rid)


@gpu
def test_group_routing_infinite_logits_and_far_picks(ops):
    logits = torch.tensor([[1.0, float("inf"), 2.0, float("inf")], [-90.0, -95.0, -200.0, -91.0]]).cuda()
    ids, w = ops.MoeRoutingGroupTopK(logits, None, 2, scoring="softmax", weightsDtype=F32)
    assert ids[0].tolist() == [1, 3] and w[0].tolist() == [0.5, 0.5]
    ids, w = ops.MoeRoutingGroupTopK(logits, None, 3, scoring="sigmoid", weightsDtype=F32)
    assert ids.tolist() == [[1, 3, 2], [0, 3, 1]]
    rid, rw = route_reference(logits.cpu(), None, 3, 1, 1, 1, "sigmoid", True, 1.0)
    check(w, rw, half_step(rw, F32) + rw * FN)
    gw = normal((2, 3), F32, 8)
    grad = ops.MoeRoutingGroupTopKGrad(gw.cuda(), logits, ids, "sigmoid")
    ref = route_grad_reference(gw, logits.cpu(), rid, "sigmoid", True, 1.0)
    check(grad, ref, gw.double().abs().max() * 40 * 2.0**-23)


@gpu
@pytest.mark.parametrize("scoring,renorm", list(itertools.product(("softmax", "sigmoid"), (True, False))))
def test_group_routing_gradient_against_differences(ops, scoring, renorm):
    """Central differences of the operator itself, h = 2^-6: the third derivative of these weights is below 2, so the
    truncation is below h^2 / 3 = 8.2e-5, and the fp32 weights' rounding (2^-22 each) below 2^-22 / h = 1.6e-5."""
    T, E, K, h = 3, 12, 4, 2.0**-6
    logits = (torch.randint(-96, 96, (T, E), generator=gen(4)).float() / 64)
    gw = normal((T, K), F32, 5)
    bias = torch.linspace(-2, 2, E).cuda()  # keeps the choice where it is
    bias[:8] -= 10.0
    ids, _ = ops.MoeRoutingGroupTopK(logits.cuda(), bias, K, 1, 1, 1, scoring, renorm, 1.0, F32)
    order = ids.cpu()
    grad = ops.MoeRoutingGroupTopKGrad(gw.cuda(), logits.cuda(), ids, scoring, renorm).cpu().double()
    for e in range(E):
        d = torch.zeros_like(logits)
        d[:, e] = h
        lo, hi = (ops.MoeRoutingGroupTopK((logits + s * d).cuda(), bias, K, 1, 1, 1, scoring, renorm, 1.0, F32)
                  for s in (-1, 1))
        assert (lo[0].cpu().sort(dim=1)[0] == order.sort(dim=1)[0]).all()
        num = torch.zeros(T, dtype=F64)
        for sign, (i, w) in ((-1, lo), (1, hi)):
            at = (i.cpu().unsqueeze(2) == order.unsqueeze(1)).double()  # the pick's slot in the first order
            num += sign * (w.cpu().double().unsqueeze(2) * at * gw.double().unsqueeze(1)).sum(dim=(1, 2))
        tol = gw.double().abs().sum(dim=1) * (8.2e-5 + 1.6e-5)
        assert ((num / (2 * h) - grad[:, e]).abs() <= tol).all()


@gpu
def test_group_routing_gradient_of_a_repeated_and_an_outside_id(ops):
    logits = normal((5, 16), F32, 6)
    ids = torch.tensor([[3, 3], [2, -1], [16, 4], [-7, 99], [0, 15]], dtype=torch.int32)
    gw = normal((5, 2), F32, 7)
    for scoring, renorm in itertools.product(("softmax", "sigmoid"), (True, False)):
        grad = ops.MoeRoutingGroupTopKGrad(gw.cuda(), logits.cuda(), ids.cuda(), scoring, renorm)
        check(grad, route_grad_reference(gw, logits, ids, scoring, renorm, 1.0), 40 * 2.0**-23 * gw.double().abs().max())


# ---------------------------------------------------------------------------------------------------------------------
# combine's gradient
# ---------------------------------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("T,H,K", [(1, 8, 1), (1, 2048, 2), (3, 520, 5), (130, 1056, 3), (129, 64, 9), (2047, 256, 6),
                                   (2048, 8, 2), (2051, 264, 4), (1, 7168, 8), (4100, 72, 13)])
def test_combine_gradient(ops, T, H, K):
    dy, eo = normal((T, H), F16, 1), normal((T, K, H), F16, 2)
    w = torch.rand((T, K), generator=gen(3)).to(F16)
    geo, gw = ops.MoeCombineGrad(dy.cuda(), eo.cuda(), w.cuda())
    ref = w.double().unsqueeze(2) * dy.double().unsqueeze(1)
    check(geo, ref, half_step(ref, F16))  # the product of two fp16 values is exact in fp32
    prod = eo.double() * dy.double().unsqueeze(1)
    ref = prod.sum(dim=2)
    acc = prod.abs().sum(dim=2) * H * U32
    check(gw, ref, acc + half_step(ref.abs() + acc, F16))
    again = ops.MoeCombineGrad(dy.cuda(), eo.cuda(), w.cuda())
    assert torch.equal(geo, again[0]) and torch.equal(gw, again[1])


@gpu
def test_combine_gradient_against_differences(ops):
    """y is linear in each weight and in expert_out: differences at fp16 values are exact but for y's rounding."""
    T, H, K = 4, 16, 3
    eo = (torch.randint(-8, 8, (T, K, H), generator=gen(1)).float() / 8).to(F16)
    w = (torch.randint(1, 8, (T, K), generator=gen(2)).float() / 8).to(F16)
    dy = (torch.randint(-8, 8, (T, H), generator=gen(3)).float() / 8).to(F16)
    geo, gw = (t.cpu().double() for t in ops.MoeCombineGrad(dy.cuda(), eo.cuda(), w.cuda()))

    def f(eo, w):
        return (ops.MoeCombine(eo.cuda(), None, w.cuda(), K).cpu().double() * dy.double()).sum(dim=1)

    for k in range(K):
        d = torch.zeros_like(w)
        d[:, k] = 0.125
        assert torch.equal((f(eo, w + d) - f(eo, w - d)) / 0.25, gw[:, k])  # multiples of 2^-9 far below 2^11 steps
        d = torch.zeros_like(eo)
        d[:, k, 5] = 0.125
        assert torch.equal((f(eo + d, w) - f(eo - d, w)) / 0.25, geo[:, k, 5])


# ---------------------------------------------------------------------------------------------------------------------
# dense product
# ---------------------------------------------------------------------------------------------------------------------


def act_reference(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "swiglu":
        g, u = z.chunk(2, dim=1)
        return g * torch.sigmoid(g) * u
    return z


def linear_check(ops, T, N, H, dtype, act="none", bias=False, residual=False, out=None, pre=False, transposed=False,
                 x=None, w=None, seed=0, workspace=None):
    Z = 2 * N if act == "swiglu" else N
    out = out or dtype
    x = normal((T, H), dtype, seed) if x is None else x
    w = normal((Z, H), dtype, seed + 1, 1 / math.sqrt(H)) if w is None else w
    b = normal((Z,), dtype, seed + 2) if bias else None
    r = normal((T, N), out, seed + 3) if residual else None
    wd = w.t().contiguous().cuda().t() if transposed else w.cuda()
    got = ops.MoeLinear(x.cuda(), wd, None if b is None else b.cuda(), None if r is None else r.cuda(), act, out, pre,
                        workspace)
    y, z16 = got if pre else (got, None)
    xd, wd64 = x.double(), w.double()
    z = xd @ wd64.t()
    zt = (H + 1) * U32 * (xd.abs() @ wd64.abs().t())
    if bias:
        z = z + b.double()
        zt = zt + U32 * z.abs()
    if pre:
        check(z16, z, zt + half_step(z.abs() + zt, dtype), "pre")
    ref = act_reference(z, act)
    if act == "swiglu":  # |silu'| <= 1.1
        g, u = z.chunk(2, dim=1)
        gt, ut = zt.chunk(2, dim=1)
        tol = 1.1 * gt * (u.abs() + ut) + g.abs() * ut + FN * ref.abs()
    elif act == "none":
        tol = zt
    else:  # slopes up to 1.13; the activations' own rounding
        tol = 1.13 * zt + FN * z.abs()
    if residual:
        ref = ref + r.double()
        tol = tol + U32 * ref.abs()
    check(y, ref, tol + half_step(ref.abs() + tol, out), (T, N, H, act))
    return y


ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu", "swiglu"]
# one token to several tiles, at and beside the edges of tiles, stages and 16-byte rows
LINEAR_SIZES = [(1, 1, 1), (1, 8, 8), (2, 3, 5), (1, 16, 2048), (3, 130, 64), (16, 40, 96), (17, 129, 65), (31, 7, 333),
                (32, 256, 1056), (33, 64, 72), (64, 200, 128), (100, 128, 63), (127, 257, 264), (128, 128, 64),
                (129, 100, 200), (255, 33, 1000), (256, 256, 128), (257, 513, 520), (300, 24, 2056), (513, 640, 192)]


@gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_linear_sizes(ops, dtype, act):
    for n, (T, N, H) in enumerate(LINEAR_SIZES):
        print(f"[linear] {T} {N} {H} {dtype} {act}", flush=True)
        linear_check(ops, T, N, H, dtype, act, bias=n % 2 == 0, residual=n % 3 == 0, out=F32 if n % 4 == 1 else dtype,
                     pre=n % 5 == 0, transposed=False, seed=n)
        linear_check(ops, T, N, H, dtype, act, bias=n % 3 == 0, residual=n % 2 == 0, out=F32 if n % 4 == 0 else dtype,
                     pre=n % 4 == 0, transposed=True, seed=n)


def random_rows_check(ops, T, N, H, dtype, act, transposed, seed, rows=24, residual=False, out=None):
    """A product too large for the CPU: every value against fp32 sums on the device, sampled rows against 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    Z = 2 * N if act == "swiglu" else N
    x = torch.empty((T, H), dtype=dtype, device="cuda").normal_(generator=g)
    w = torch.empty((H, Z) if transposed else (Z, H), dtype=dtype, device="cuda").normal_(0, H**-0.5, generator=g)
    w = w.t() if transposed else w
    b = torch.empty((Z,), dtype=dtype, device="cuda").normal_(generator=g)
    out = out or dtype
    r = torch.empty((T, N), dtype=out, device="cuda").normal_(generator=g) if residual else None
    y, pre = ops.MoeLinear(x, w, b, r, act, out, True)
    at = torch.randint(0, T, (rows,), generator=gen(seed))
    at[0], at[1] = 0, T - 1
    z = x[at.cuda()].double() @ w.double().t() + b.double()
    zt = (H + 2) * U32 * (x[at.cuda()].double().abs() @ w.double().abs().t() + b.double().abs())
    check(pre[at.cuda()], z.cpu(), (zt + half_step(z.abs() + zt, dtype)).cpu(), "pre")
    ref = act_reference(z, act)
    if act == "swiglu":
        (gz, uz), (gt, ut) = z.chunk(2, dim=1), zt.chunk(2, dim=1)
        tol = 1.1 * gt * (uz.abs() + ut) + gz.abs() * ut + FN * ref.abs()
    else:
        tol = 1.13 * zt + FN * z.abs()
    if residual:
        ref = ref + r[at.cuda()].double()
        tol = tol + U32 * ref.abs()
    check(y[at.cuda()], ref.cpu(), (tol + half_step(ref.abs() + tol, out)).cpu(), (T, N, H, act))
    zf = x.float() @ w.float().t() + b.float()  # all values: two fp32 sums, each within 2 H 2^-24 of |x| |w|
    # and a rounding; |x| |w| is below 2 sqrt(H) sigma for these distributions, so 2^-8 covers fp16 with room
    yf = act_reference(zf, act) + (0 if r is None else r.float())
    err = (y.float() - yf).abs()
    assert (err <= 2.0**-6 + torch.finfo(dtype).eps * yf.abs()).all(), (T, N, H, act, float(err.max()))
    return y


@gpu
@pytest.mark.parametrize("T,N,H,act,transposed,out", [
    (4096, 2048, 64, "none", False, None), (4097, 2056, 72, "gelu", False, None), (2049, 4104, 128, "silu", True, None),
    (3001, 3000, 200, "relu", False, F32), (8191, 1400, 136, "swiglu", False, None), (4099, 1032, 1000, "swiglu", True, None),
    (33000, 264, 520, "gelu_tanh", True, F32), (260, 33000, 96, "none", False, None), (2300, 2306, 1544, "none", False, None)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_linear_large_tiles(ops, dtype, T, N, H, act, transposed, out):
    print(f"[linear large] {T} {N} {H} {act} {transposed} {dtype}", flush=True)
    random_rows_check(ops, T, N, H, dtype, act, transposed, T + N, residual=N % 16 == 8, out=out)


@gpu
@pytest.mark.parametrize("T,N,H,act,transposed", [
    (4097, 2056, 2056, "none", False), (2049, 2100, 4104, "silu", True), (8200, 1032, 2048, "swiglu", False),
    (100, 4100, 4096, "gelu", False)])
def test_linear_gradient_large_tiles(ops, T, N, H, act, transposed):
    print(f"[linear grad large] {T} {N} {H} {act} {transposed}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T)
    Z = 2 * N if act == "swiglu" else N
    new = lambda shape, s: torch.empty(shape, dtype=F16, device="cuda").normal_(0, s, generator=g)  # noqa: E731
    dy, x, w = new((T, N), 1), new((T, H), 1), new((Z, H), H**-0.5)
    pre = None if act == "none" else new((T, Z), 1)
    gx, gw, gb = ops.MoeLinearGrad(dy, x, w.t().contiguous().t() if transposed else w, pre, act, gradBias=True)
    dz = dy.double()
    if pre is not None:
        z = pre.double().requires_grad_(True)
        dz, = torch.autograd.grad(act_reference(z, act), z, dz)
    dzt = 2 * half_step(dz, F16) + 2.0**-20 * (0 if pre is None else 1)
    rows = torch.tensor([0, 1, T // 2, T - 1], device="cuda")
    cols = torch.tensor([0, Z // 2 - 1, Z // 2, Z - 1], device="cuda")
    wd, xd = w.double(), x.double()
    ref = dz[rows] @ wd
    tol = dzt[rows] @ wd.abs() + Z * U32 * (dz[rows].abs() @ wd.abs())
    check(gx[rows], ref.cpu(), (tol + half_step(ref.abs() + tol, F16)).cpu(), "grad_x")
    ref = dz[:, cols].t() @ xd
    tol = dzt[:, cols].t() @ xd.abs() + T * U32 * (dz[:, cols].abs().t() @ xd.abs())
    check(gw[cols], ref.cpu(), (tol + half_step(ref.abs() + tol, F16)).cpu(), "grad_weight")
    for got, ref in ((gx, dz.float() @ w.float()), (gw, dz.t().float() @ x.float())):  # every value, loosely
        assert ((got.float() - ref).norm() / ref.norm()) < 3 * 2.0**-11
        assert ((got.float() - ref).abs() <= 2.0**-5 * ref.abs() + 2.0**-4 * ref.square().mean().sqrt()).all()
    ref = dz.sum(dim=0)
    tol = (T + 1) * U32 * dz.abs().sum(dim=0) + T * 2.0**-20
    check(gb, ref.cpu(), (tol + half_step(ref.abs() + tol, F16)).cpu(), "grad_bias")


@gpu
def test_linear_strides_and_alignment(ops):
    """Rows of wider tensors, bases off 16 bytes, rows off 16 bytes, a transposed view: the same values as contiguous."""
    T, N, H = 70, 96, 136
    for dtype in (F16, BF16):
        xw, ww = normal((T, 200), dtype, 1).cuda(), normal((N, 160), dtype, 2, 0.1).cuda()
        for xo, wo in ((0, 0), (8, 16), (1, 0), (0, 3), (5, 7)):
            x, w = xw[:, xo:xo + H], ww[:, wo:wo + H]
            y = linear_check(ops, T, N, H, dtype, x=x.cpu(), w=w.cpu())
            assert torch.equal(ops.MoeLinear(x, w), y), (xo, wo)
        odd = normal((T, H + 1), dtype, 3).cuda()[:, :H]  # rows 2 bytes off
        assert torch.equal(ops.MoeLinear(odd, ww[:, :H]), ops.MoeLinear(odd.contiguous(), ww[:, :H].contiguous()))
        wt = normal((H, 101), dtype, 4, 0.1).cuda()[:, 2:98].t()  # [96, 136], contiguous along the 96
        x = xw[:, :H]
        linear_check(ops, T, N, H, dtype, x=x.cpu(), w=wt.cpu(), transposed=True)
        got = ops.MoeLinear(x, wt).double().cpu()
        ref = x.double().cpu() @ wt.double().cpu().t()
        tol = (H + 1) * U32 * (x.double().cpu().abs() @ wt.double().cpu().abs().t())
        check(got, ref, tol + half_step(ref.abs() + tol, dtype))


@gpu
def test_linear_reads_nothing_past_the_operands(ops):
    """NaN in the columns beside the operands, before and after their rows: no result takes any of it."""
    for T, N, H in ((5, 40, 72), (40, 130, 200), (150, 72, 88), (1, 24, 1000)):
        def framed(rows, cols):
            t = torch.full((rows + 2, cols + 16), float("nan"), dtype=F16)
            t[1:rows + 1, 8:cols + 8] = normal((rows, cols), F16, rows + cols)
            return t.cuda()[1:rows + 1, 8:cols + 8]

        x, w = framed(T, H), framed(N, H)
        wt = framed(H, N).t()
        dy = framed(T, N)
        assert torch.isfinite(ops.MoeLinear(x, w)).all() and torch.isfinite(ops.MoeLinear(x, wt)).all()
        for weight in (w, wt):
            for g in ops.MoeLinearGrad(dy, x, weight, gradBias=True):
                assert torch.isfinite(g).all()


@gpu
def test_linear_inf_and_nan_stay_in_their_row(ops):
    x = normal((40, 128), F16, 1)
    x[3, 5], x[7, 0] = float("nan"), float("inf")
    w = normal((64, 128), F16, 2)
    y = ops.MoeLinear(x.cuda(), w.cuda()).cpu()
    rows = torch.isfinite(y).all(dim=1)
    assert not rows[3] and not rows[7] and rows.sum() == 38


@gpu
def test_linear_split_over_k_is_deterministic_and_takes_its_workspace(ops):
    T, N, H = 4, 72, 8192
    need = ops.linear_workspace_bytes(T, N, H)
    assert need > 0
    ws = torch.full((need + 64,), 0x7f, dtype=torch.uint8, device="cuda")
    y = linear_check(ops, T, N, H, F16, bias=True, residual=True, workspace=ws)
    assert (ws[need:] == 0x7f).all()
    assert torch.equal(y, linear_check(ops, T, N, H, F16, bias=True, residual=True))
    with pytest.raises(MoeError) as e:
        ops.MoeLinear(torch.zeros(T, H, dtype=F16, device="cuda"), torch.zeros(N, H, dtype=F16, device="cuda"),
                      workspace=ws[:need - 16])
    assert e.value.status == 5


@gpu
@pytest.mark.parametrize("T,N,H,act,transposed", [
    (3, 40, 333, "none", False), (70, 41, 64, "swiglu", True), (70, 41, 65, "swiglu", True), (300, 130, 2049, "silu", False),
    (300, 130, 2049, "silu", True), (1, 7, 4099, "swiglu", False)])
def test_odd_sizes_keep_within_their_workspace(ops, T, N, H, act, transposed):
    need = ops.linear_workspace_bytes(T, N, H, act)
    ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    linear_check(ops, T, N, H, F16, act, bias=True, transposed=transposed, workspace=ws[:need])
    assert (ws[need:] == 0x5a).all()
    need = ops.linear_grad_workspace_bytes(T, N, H, act)
    ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    grad_check(ops, T, N, H, BF16, act, transposed=transposed, workspace=ws[:need])
    assert (ws[need:] == 0x5a).all()


def grad_check(ops, T, N, H, dtype, act, transposed=False, seed=0, dy=None, x=None, w=None, workspace=None):
    Z = 2 * N if act == "swiglu" else N
    dy = normal((T, N), dtype, seed) if dy is None else dy
    x = normal((T, H), dtype, seed + 1) if x is None else x
    w = normal((Z, H), dtype, seed + 2, 1 / math.sqrt(H)) if w is None else w
    pre = None if act == "none" else normal((T, Z), dtype, seed + 3, 1.5)
    wd = w.t().contiguous().cuda().t() if transposed else w.cuda()
    gx, gw, gb = ops.MoeLinearGrad(dy.cuda(), x.cuda(), wd, None if pre is None else pre.cuda(), act, gradBias=True,
                                   workspace=workspace)
    if pre is None:
        dz, dzt = dy.double(), torch.zeros(T, N, dtype=F64)
    else:
        z = pre.double().requires_grad_(True)
        dz, = torch.autograd.grad(act_reference(z, act), z, dy.double())
        z = z.detach()
        # the factors of a slope round relative to 1 and |z| (SwiGLU: times the other half), then dz to its type
        scale = (1 + z.abs()) * (torch.cat([dy, dy], 1).double().abs() * (1 + z.abs().roll(N, 1)) if act == "swiglu"
                                 else dy.double().abs() * 2)
        fp = scale * 2 * FN
        dzt = fp + half_step(dz.abs() + fp, dtype)
        bt = fp
    xd, wd64 = x.double(), w.double()
    ref = dz @ wd64
    tol = dzt @ wd64.abs() + (Z + 1) * U32 * ((dz.abs() + dzt) @ wd64.abs())
    check(gx, ref, tol + half_step(ref.abs() + tol, dtype), "grad_x")
    ref = dz.t() @ xd
    tol = dzt.t() @ xd.abs() + (T + 1) * U32 * ((dz.abs() + dzt).t() @ xd.abs())
    check(gw, ref, tol + half_step(ref.abs() + tol, dtype), "grad_weight")
    ref = dz.sum(dim=0)
    tol = (T + 1) * U32 * dz.abs().sum(dim=0) + (0 if pre is None else bt.sum(dim=0))
    check(gb, ref, tol + half_step(ref.abs() + tol, dtype), "grad_bias")
    return gx, gw, gb


@gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_linear_gradient_sizes(ops, dtype, act):
    for n, (T, N, H) in enumerate(LINEAR_SIZES):
        print(f"[linear grad] {T} {N} {H} {dtype} {act}", flush=True)
        grad_check(ops, T, N, H, dtype, act, transposed=n % 2 == 1, seed=10 * n)


@gpu
def test_linear_gradient_strides_and_parts(ops):
    T, N, H = 70, 96, 136
    dyw, xw, ww = normal((T, 121), F16, 1).cuda(), normal((T, 200), F16, 2).cuda(), normal((N, 160), F16, 3).cuda()
    pre = normal((T, N), F16, 4).cuda()
    for dy, x, w in ((dyw[:, :N], xw[:, 8:H + 8], ww[:, :H]), (dyw[:, 1:N + 1], xw[:, 1:H + 1], ww[:, 3:H + 3]),
                     (dyw[:, :N].contiguous(), xw[:, 8:H + 8], ww[:, 8:H + 8])):
        for act in ("none", "silu"):
            whole = ops.MoeLinearGrad(dy, x, w, pre, act, gradBias=True)
            flat = ops.MoeLinearGrad(dy.contiguous(), x.contiguous(), w.contiguous(), pre, act, gradBias=True)
            for a, b in zip(whole, flat):
                assert torch.equal(a, b)
            for k in range(3):  # each part alone
                part = ops.MoeLinearGrad(dy, x, w, pre, act, k == 0, k == 1, k == 2)
                assert torch.equal(part[k], whole[k]) and sum(p is not None for p in part) == 1


@gpu
def test_linear_gradient_against_differences(ops):
    """Central differences of MoeLinear's fp32 result along directions of +-1, h = 2^-5. Operands are multiples of 2^-5,
    so x + h d is exact; |d^3 silu / dz^3| < 1 and a direction moves z by at most h s with s = |w| or |x| summed over
    the direction, so the truncation is below sum |dy| (h s)^3 / 6 / h."""
    T, N, H, h = 6, 10, 16, 2.0**-5
    grid = lambda shape, seed: (torch.randint(-16, 17, shape, generator=gen(seed)).float() / 32).to(F16)  # noqa: E731
    x, w, dy = grid((T, H), 1), grid((N, H), 2), grid((T, N), 3)
    b = grid((N,), 4)

    def f(x, w, b):
        return (ops.MoeLinear(x.cuda(), w.cuda(), b.cuda(), None, "silu", F32).cpu().double() * dy.double()).sum()

    _, pre = ops.MoeLinear(x.cuda(), w.cuda(), b.cuda(), None, "silu", returnPre=True)
    gx, gw, gb = (g.cpu().double() for g in ops.MoeLinearGrad(dy.cuda(), x.cuda(), w.cuda(), pre, "silu", gradBias=True))
    dsum = dy.double().abs().sum()
    for seed in range(5):
        sign = lambda shape, s: torch.randint(0, 2, shape, generator=gen(s)).double() * 2 - 1  # noqa: E731
        dx, dw, db = sign((T, H), seed), sign((N, H), 50 + seed), sign((N,), 90 + seed)
        for (a, c, e), got, s in (((dx, 0 * dw, 0 * db), (gx * dx).sum(), w.double().abs().sum(dim=1).max()),
                                  ((0 * dx, dw, 0 * db), (gw * dw).sum(), x.double().abs().sum(dim=1).max()),
                                  ((0 * dx, 0 * dw, db), (gb * db).sum(), 1.0)):
            hi, lo = (f((x.double() + q * h * a).to(F16), (w.double() + q * h * c).to(F16), (b.double() + q * h * e).to(F16))
                      for q in (1, -1))
            # pre, dz and the gradient are rounded to fp16: three times 2^-11 of sum |dy| s
            tol = dsum * (float(h * s) ** 3 / 6 / h) + 3 * 2.0**-11 * dsum * s + dsum * 40 * U32 / h
            assert abs((hi - lo) / (2 * h) - got) <= tol


@gpu
def test_no_tokens(ops):
    x, w = torch.empty(0, 64, dtype=F16, device="cuda"), normal((24, 64), F16, 1).cuda()
    assert ops.MoeLinear(x, w).shape == (0, 24)
    gx, gw, gb = ops.MoeLinearGrad(torch.empty(0, 24, dtype=F16, device="cuda"), x, w, gradBias=True)
    assert gx.shape == (0, 64) and gw.abs().max() == 0 and gb.abs().max() == 0
    gx, gw, gb = ops.MoeLinearGrad(torch.empty(0, 24, dtype=F16, device="cuda"), x, w,
                                   torch.empty(0, 24, dtype=F16, device="cuda"), "gelu", gradBias=True)
    assert gw.abs().max() == 0 and gb.abs().max() == 0
    ids, wt = ops.MoeRoutingGroupTopK(torch.empty(0, 8, device="cuda"), None, 2)
    assert ids.shape == (0, 2) and wt.shape == (0, 2)
    assert ops.MoeRoutingGroupTopKGrad(wt, torch.empty(0, 8, device="cuda"), ids).shape == (0, 8)
    geo, gw = ops.MoeCombineGrad(torch.empty(0, 8, dtype=F16, device="cuda"), torch.empty(0, 2, 8, dtype=F16, device="cuda"),
                                 torch.empty(0, 2, dtype=F16, device="cuda"))
    assert geo.shape == (0, 2, 8) and gw.shape == (0, 2)


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------


def layer_inputs(T=45, H=128, E=16, I=96, S=72, dtype=F16):
    return dict(x=normal((T, H), dtype, 1), w_gate=normal((H, E), dtype, 2, H**-0.5),
                expert_weights=torch.cat([normal((E, 2 * I, H), dtype, 3, H**-0.5),
                                          normal((E, I, H), dtype, 4, I**-0.5)], dim=1),
                gate_up=normal((2 * S, H), dtype, 5, H**-0.5), down=normal((H, S), dtype, 6, S**-0.5),
                bias=(torch.rand(E, generator=gen(7)) - 0.5) * 0.1)


@gpu
def test_shared_layer_is_its_parts_and_matches_64_bits(ops):
    v = {k: t.cuda() for k, t in layer_inputs().items()}
    attrs = dict(topK=4, bias=v["bias"], numGroups=4, topGroups=2, groupTop=2, scoring="sigmoid", scale=2.5)
    y, ids, w, eo = ops.moe_layer_shared(v["x"], v["w_gate"], v["expert_weights"], v["gate_up"], v["down"], **attrs)
    logits = ops.MoeLinear(v["x"], v["w_gate"].t(), outDtype=F32)
    rid, rw = route_reference(logits.cpu(), v["bias"].cpu(), 4, 4, 2, 2, "sigmoid", True, 2.5)
    assert torch.equal(ids.cpu(), rid)
    check(w, rw, half_step(rw, F16) + rw * FN)
    assert torch.equal(eo, ops.MoeExpertFFN(v["x"], ids, w, v["expert_weights"]))
    routed = ops.MoeCombine(eo, ids, w, 4)
    plain = ops.moe_layer_shared(v["x"], v["w_gate"], v["expert_weights"], **attrs)
    assert torch.equal(plain[0], routed)
    gu = v["x"].double() @ v["gate_up"].double().t()
    hid = gu[:, :72] * torch.sigmoid(gu[:, :72]) * gu[:, 72:]
    ref = hid @ v["down"].double().t() + routed.double()
    err = (y.double() - ref).abs()
    # hidden is rounded once (2^-11 of each |hidden|), y once
    tol = 1.1 * 2.0**-11 * (hid.abs() @ v["down"].double().abs().t()) + half_step(ref, F16) + 1e-4
    assert (err <= tol).all()


@gpu
def test_router_training_step_through_the_operators(ops):
    """The chain of gradients from y to w_gate, x and the dense expert against 64-bit differentiation, with the routed
    experts' outputs held fixed."""
    v = layer_inputs()
    d = {k: t.cuda() for k, t in v.items()}
    T, H = v["x"].shape
    logits = ops.MoeLinear(d["x"], d["w_gate"].t(), outDtype=F32)
    ids, w = ops.MoeRoutingGroupTopK(logits, None, 4, scoring="softmax", scale=1.5)
    eo = ops.MoeExpertFFN(d["x"], ids, w, d["expert_weights"])
    hid, pre = ops.MoeLinear(d["x"], d["gate_up"], activation="swiglu", returnPre=True)
    dy = normal((T, H), F16, 9).cuda()
    _, gw = ops.MoeCombineGrad(dy, eo, w)
    gl = ops.MoeRoutingGroupTopKGrad(gw, logits, ids, scale=1.5)
    gx1, ggate, _ = ops.MoeLinearGrad(gl.to(F16), d["x"], d["w_gate"].t())
    ghid, gdown, _ = ops.MoeLinearGrad(dy, hid, d["down"])
    gx2, ggu, _ = ops.MoeLinearGrad(ghid, d["x"], d["gate_up"], pre, "swiglu")

    leaf = {k: v[k].double().requires_grad_(True) for k in ("x", "w_gate", "gate_up", "down")}
    p = torch.softmax(leaf["x"] @ leaf["w_gate"], dim=1).gather(1, ids.cpu().long())
    p = 1.5 * p / p.sum(dim=1, keepdim=True)
    z = leaf["x"] @ leaf["gate_up"].t()
    y = (eo.cpu().double() * p.unsqueeze(2)).sum(dim=1) + act_reference(z, "swiglu") @ leaf["down"].t()
    y.backward(dy.cpu().double())
    for name, got in (("w_gate", ggate.t()), ("x", gx1.float() + gx2.float()), ("gate_up", ggu), ("down", gdown)):
        ref = leaf[name].grad
        # a chain of at most 6 roundings of 2^-11 each, relative to the gradient's size
        rel = float((got.cpu().double() - ref).norm() / ref.norm())
        assert rel < 6 * 2.0**-11, (name, rel)


@gpu
def test_calls_on_other_streams_and_graph_replays(ops):
    v = {k: t.cuda() for k, t in layer_inputs(T=200, H=256).items()}
    x, gu = v["x"], v["gate_up"]
    logits = ops.MoeLinear(x, v["w_gate"].t(), outDtype=F32)
    dy = normal((200, 72), F16, 3).cuda()
    pre = normal((200, 144), F16, 4).cuda()
    ws = torch.empty(ops.linear_workspace_bytes(200, 72, 256, "swiglu") + 1, dtype=torch.uint8, device="cuda")
    gws = torch.empty(ops.linear_grad_workspace_bytes(200, 72, 256, "swiglu"), dtype=torch.uint8, device="cuda")

    def step(stream=None):
        ids, w = ops.MoeRoutingGroupTopK(logits, v["bias"], 3, 4, 2, 2, "sigmoid", stream=stream)
        gl = ops.MoeRoutingGroupTopKGrad(w, logits, ids, "sigmoid", stream=stream)
        y = ops.MoeLinear(x, gu, None, None, "swiglu", workspace=ws, stream=stream)
        return (ids, w, gl, y) + ops.MoeLinearGrad(dy, x, gu, pre, "swiglu", gradBias=True, workspace=gws, stream=stream)

    eager = [t.clone() for t in step()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other = step(s)
    s.synchronize()
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        for t in out:
            t.zero_()
        if n == 2:
            step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------------------------
# refusals (no GPU needed: every check is before the first launch)
# ---------------------------------------------------------------------------------------------------------------------


def refused(status, fn, *args, **kw):
    with pytest.raises(MoeError) as e:
        fn(*args, **kw)
    assert e.value.status == status, e.value
    assert e.value.message


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64, dtype=F16), torch.zeros(8, 64, dtype=F16)
    refused(4, opsm.MoeLinear, x, w)
    refused(4, opsm.MoeLinearGrad, torch.zeros(4, 8, dtype=F16), x, w)
    refused(4, opsm.MoeRoutingGroupTopK, torch.zeros(4, 8))
    refused(4, opsm.MoeRoutingGroupTopKGrad, torch.zeros(4, 2), torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32))
    refused(4, opsm.MoeCombineGrad, torch.zeros(4, 8, dtype=F16), torch.zeros(4, 2, 8, dtype=F16),
            torch.zeros(4, 2, dtype=F16))
    refused(1, opsm.MoeLinear, [1.0], w)
    refused(4, opsm.MoeLinear, x, w, activation="tanh")


def test_library_refuses_bad_sizes_before_any_launch():
    lib = importlib.import_module(PKG_NAME + "._lib").load()

    def route(T=4, E=16, K=2, G=1, TG=1, GT=1, ld=16, lt=0, wt=1, scoring=0, scale=1.0, ptr=16):
        return lib.moe_routing_group_topk(ptr, ld, lt, None, ptr, ptr, wt, T, E, K, G, TG, GT, scoring, 1, scale, None)

    assert route(T=0) == 0
    for kw, status in ((dict(T=-1), 4), (dict(E=0), 4), (dict(K=0), 4), (dict(K=17), 4), (dict(E=257, ld=257), 6),
                       (dict(G=3), 4), (dict(G=0), 4), (dict(TG=2), 4), (dict(G=4, TG=0), 4), (dict(G=4, TG=1, K=5), 4),
                       (dict(GT=3), 4), (dict(GT=0), 4), (dict(ld=15), 4), (dict(lt=3), 4), (dict(wt=27), 4),
                       (dict(scoring=2), 4), (dict(scale=float("nan")), 4), (dict(scale=float("inf")), 4),
                       (dict(T=1 << 40), 6), (dict(ptr=None), 1)):
        assert route(**kw) == status, kw
        assert lib.moe_last_error()

    def grad(T=4, E=16, K=2, ld=16, lt=0, wt=0, scoring=0, ptr=16):
        return lib.moe_routing_group_topk_grad(ptr, wt, ptr, ld, lt, ptr, ptr, T, E, K, scoring, 1, 1.0, None)

    for kw, status in ((dict(K=17), 4), (dict(ld=8), 4), (dict(wt=3), 4), (dict(lt=-1), 4), (dict(scoring=-1), 4),
                       (dict(ptr=None), 1), (dict(E=300, ld=300), 6)):
        assert grad(**kw) == status, kw

    def combine(T=4, H=64, K=2, ptr=16):
        return lib.moe_combine_grad(ptr, ptr, ptr, ptr, ptr, T, H, K, None)

    for kw, status in ((dict(T=-1), 4), (dict(H=0), 4), (dict(K=0), 4), (dict(H=60), 6), (dict(T=1 << 30, K=2), 6),
                       (dict(ptr=None), 1), (dict(ptr=8), 6)):
        assert combine(**kw) == status, kw

    def linear(T=4, N=8, H=64, act=0, dt=1, out=1, ldx=64, ldw=64, tr=0, ptr=16, ws=None, wsb=0):
        return lib.moe_linear(ptr, ldx, ptr, ldw, tr, None, None, ptr, None, ws, wsb, T, N, H, act, dt, out, None)

    assert linear(T=0) == 0
    for kw, status in ((dict(T=-1), 4), (dict(N=0), 4), (dict(H=0), 4), (dict(act=6), 4), (dict(act=-1), 4), (dict(dt=0), 4),
                       (dict(out=27), 4), (dict(ldx=63), 4), (dict(ldw=10), 4), (dict(tr=1, ldw=7), 4), (dict(ptr=None), 1),
                       (dict(N=(1 << 20) + 1), 6), (dict(T=1 << 40), 6), (dict(T=1 << 30, N=1 << 20), 6),
                       (dict(T=4, N=8, H=65536, ldx=65536, ldw=65536), 5), (dict(act=5, tr=1, ldw=8), 4)):
        assert linear(**kw) == status, kw

    def lgrad(T=4, N=8, H=64, act=0, dt=1, ldy=8, ldx=64, ldw=64, ptr=16, pre=16, ws=16, wsb=1 << 30):
        return lib.moe_linear_grad(ptr, ldy, ptr, ldx, ptr, ldw, 0, pre, 16, 16, 16, ws, wsb, T, N, H, act, dt, None)

    for kw, status in ((dict(act=4, pre=None), 1), (dict(ws=None), 5), (dict(wsb=16), 5), (dict(ldy=7), 4), (dict(ldx=8), 4),
                       (dict(ldw=8), 4), (dict(ptr=None), 1), (dict(ws=24), 6), (dict(dt=0), 4)):
        assert lgrad(**kw) == status, kw
    assert lib.moe_linear_workspace_bytes(-1, 8, 8, 0) == 0 and lib.moe_linear_grad_workspace_bytes(4, 0, 8, 0) == 0


@gpu
def test_refusals_on_device_tensors(ops):
    c = lambda *shape, dtype=F16: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    refused(4, ops.MoeLinear, c(4, 64), c(8, 64, dtype=BF16))
    refused(4, ops.MoeLinear, c(4, 64, dtype=F32), c(8, 64, dtype=F32))
    refused(3, ops.MoeLinear, c(4, 64), c(8, 32))
    refused(2, ops.MoeLinear, c(4, 4, 64), c(8, 64))
    refused(3, ops.MoeLinear, c(4, 64), c(7, 64), activation="swiglu")
    refused(3, ops.MoeLinear, c(4, 64), c(8, 64), c(4))
    refused(3, ops.MoeLinear, c(4, 64), c(8, 64), None, c(4, 7))
    refused(4, ops.MoeLinear, c(4, 64), c(8, 64), None, c(4, 8), outDtype=F32)
    refused(4, ops.MoeLinear, c(64, 4).t(), c(8, 64))
    refused(4, ops.MoeLinear, c(4, 64), c(8, 128)[:, ::2])
    refused(4, ops.MoeLinear, c(1, 64).expand(4, 64), c(8, 64))
    refused(4, ops.MoeLinear, c(4, 64), c(8, 64), outDtype=BF16)
    refused(1, ops.MoeLinearGrad, c(4, 8), c(4, 64), c(8, 64), None, "silu")
    refused(3, ops.MoeLinearGrad, c(4, 8), c(4, 64), c(8, 64), c(4, 7), "silu")
    refused(3, ops.MoeLinearGrad, c(3, 8), c(4, 64), c(8, 64))
    refused(4, ops.MoeRoutingGroupTopK, c(4, 8, dtype=torch.int32))
    refused(4, ops.MoeRoutingGroupTopK, c(8, 4).t())
    refused(4, ops.MoeRoutingGroupTopK, c(4, 8), c(8))
    refused(3, ops.MoeRoutingGroupTopK, c(4, 8), c(7, dtype=F32))
    refused(4, ops.MoeRoutingGroupTopK, c(4, 8), None, 9)
    refused(4, ops.MoeRoutingGroupTopK, c(4, 8), None, 2, scoring="relu")
    refused(4, ops.MoeRoutingGroupTopK, c(4, 8), None, 2, weightsDtype=BF16)
    refused(3, ops.MoeRoutingGroupTopKGrad, c(4, 3), c(4, 8), c(4, 2, dtype=torch.int32))
    refused(3, ops.MoeCombineGrad, c(4, 16), c(4, 2, 8), c(4, 2))
    refused(3, ops.moe_layer_shared, c(4, 64), c(64, 8), c(4, 96, 64))
    refused(1, ops.moe_layer_shared, c(4, 64), c(64, 8), c(8, 96, 64), c(16, 64))
