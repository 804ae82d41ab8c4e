"""The operators on rows (MoeAddRmsNorm, MoeAddRmsNormQuant, MoeAddRmsNormGrad, MoeQuantize, MoePermute, MoeUnpermute,
MoeUnpermuteGrad) against plain implementations in 64 bits.

Tolerances, from the arithmetic alone: a rounding is off by at most half a step (half_step), an fp32 operation by 2^-24
relative, an fp32 sum of n products in any order by n 2^-24 times the sum of their magnitudes. The 8-bit integers are
computed here by the same fp32 operations and have to be equal."""
from __future__ import annotations

import pytest

from test_dense_ops import BF16, F16, F32, F64, U32, MoeError, check, gen, gpu, half_step, normal, opsm

torch = pytest.importorskip("torch")
lib = opsm._lib
EPS = 1e-5
TYPES = (F16, BF16, F32)


def norm_reference(x, gamma, residual, eps=EPS):
    """v, r and y of the definition, in 64 bits."""
    v = x.double() + (0 if residual is None else residual.double())
    r = 1 / torch.sqrt(v.square().mean(dim=1, keepdim=True) + eps)
    return v, r, v * r * gamma.double()


def quant_reference(p):
    """The 8-bit form of fp32 rows by the definition's fp32 operations."""
    top = p.abs().amax(dim=1, keepdim=True)
    fine = torch.isfinite(top)
    up = torch.where(top < 2.0**-60, 2.0**64, 1.0)
    inverse = torch.where(fine & (top > 0), torch.tensor(127.0) / (top * up), 0.0)  # (a number / a tensor is two roundings)
    return torch.round(torch.where(fine, p * up, 0.0) * inverse).to(torch.int8), torch.where(fine, top, float("nan"))[:, 0]


def cuda(t):
    return None if t is None else t.cuda()


NORMS = [  # T, H: rows of one lane's step, ragged ends, a wave, 4 and 16 waves, several steps, rows read twice
    (1, 1), (5, 3), (4, 7), (3, 8), (6, 9), (1, 64), (9, 511), (130, 512), (7, 513), (1, 1056), (2050, 40), (2049, 1000),
    (2048, 2048), (33, 2047), (1, 4100), (2051, 4104), (2, 7168), (1, 8193), (2, 16385), (2, 32768), (3, 40003)]


@gpu
@pytest.mark.parametrize("T,H", NORMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_against_the_definition(ops, T, H, dtype):
    for n, (gdt, with_res) in enumerate(((dtype, True), (F32, False))):
        x, gamma = normal((T, H), dtype, 10 + n), (1 + 0.3 * normal((H,), F32, 20 + n)).to(gdt)
        res = normal((T, H), dtype, 30 + n, 2.0) if with_res else None
        if T > 2:
            x[1] = 0  # a row of zeros
            if res is not None:
                res[1] = 0
        v, _, ref = norm_reference(x, gamma, res)
        # v, the factor (conversion, root, quotient) and two products
        tol = half_step(ref, dtype) + ref.abs() * 8 * U32
        y, total = ops.MoeAddRmsNorm(x.cuda(), gamma.cuda(), cuda(res), EPS)
        check(y, ref, tol, (n, "y"))
        if with_res:
            check(total, v, half_step(v, dtype) * (1 + U32) + v.abs() * U32, (n, "sum"))
        else:
            assert total is None
        q, scale, y2, total2 = ops.MoeAddRmsNormQuant(x.cuda(), gamma.cuda(), cuda(res), EPS, returnNorm=bool(n))
        v32 = x.float() + (0 if res is None else res.float())
        rq, _ = quant_reference(v32 * gamma.float())
        assert torch.equal(q.cpu(), rq)
        rs = ref.abs().amax(dim=1) / 127
        check(scale, rs, rs * 10 * U32, (n, "scale"))
        assert (y2 is None) == (not n) and (y2 is None or torch.equal(y2, y))
        assert total is None or torch.equal(total, total2)


@gpu
@pytest.mark.parametrize("T,H", [(3, 5), (9, 511), (257, 2048), (2050, 1000), (1, 4100), (3, 16384)])
def test_rows_any_stride_and_alignment_apart(ops, T, H):
    wide, r = normal((T, H + 13), F16, 1).cuda(), normal((T, H + 5), F16, 2).cuda()
    gamma = normal((H + 1,), F16, 3).cuda()[1:]
    x, res = wide[:, 3:3 + H], r[:, 1:1 + H]
    for a, b in zip(ops.MoeAddRmsNormQuant(x, gamma, res, EPS, True),
                    ops.MoeAddRmsNormQuant(x.contiguous(), gamma.clone(), res.contiguous(), EPS, True)):
        assert torch.equal(a, b)
    for a, b in zip(ops.MoeQuantize(x), ops.MoeQuantize(x.contiguous())):
        assert torch.equal(a, b)
    gy = normal((T, H + 3), F16, 4).cuda()[:, 2:2 + H]
    for a, b in zip(ops.MoeAddRmsNormGrad(gy, x, gamma, res, EPS),
                    ops.MoeAddRmsNormGrad(gy.contiguous(), x.contiguous(), gamma.clone(), res.contiguous(), EPS)):
        assert torch.equal(a, b)
    ids = torch.randint(-1, 4, (T, 3), generator=gen(5), dtype=torch.int32).cuda()
    for a, b in zip(ops.MoePermute(x, ids, 4), ops.MoePermute(x.contiguous(), ids, 4)):
        assert a is b is None or torch.equal(a, b)
    position = ops.MoePermute(x, ids, 4)[2]
    rows, w = normal((3 * T, H), F16, 6).cuda(), normal((T, 3), F32, 7).cuda()
    for a, b in zip(ops.MoeUnpermuteGrad(x, rows, position, w), ops.MoeUnpermuteGrad(x.contiguous(), rows, position, w)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("H", [7, 64, 2049, 9000, 40000])
def test_rows_of_extreme_values(ops, H):
    """The largest, the smallest and subnormal values keep their digits; an infinity or a NaN stays in its row."""
    x = normal((10, H), F32, 1)
    for i, power in enumerate((127, 100, 63, -63, -100, -126, -140)):
        x[i] = (x[i] / x[i].abs().max()).double().mul(2.0**power).float()
    x[7, H // 2] = float("inf")
    x[8, H - 1] = float("nan")
    gamma = torch.ones(H)
    q, scale = ops.MoeQuantize(x.cuda())
    rq, top = quant_reference(x)
    assert torch.equal(q.cpu(), rq)
    rs = top.double() / 127
    fine = torch.isfinite(rs)
    check(scale[fine.cuda()], rs[fine], rs[fine] * U32 + 2.0**-150, "scale")  # half a subnormal step
    assert torch.isnan(scale[7:9]).all() and torch.equal(fine, torch.tensor([True] * 7 + [False] * 2 + [True]))
    nq, nscale, y, _ = ops.MoeAddRmsNormQuant(x.cuda(), gamma.cuda(), None, 2.0**-140, True)
    assert torch.equal(nq.cpu(), rq)
    _, _, ref = norm_reference(x, gamma, None, 2.0**-140)
    rows = [0, 1, 2, 3, 4, 5, 6, 9]
    check(y[rows], ref[rows], ref[rows].abs() * 8 * U32 + 2.0**-149)
    check(nscale[rows], ref[rows].abs().amax(dim=1) / 127, ref[rows].abs().amax(dim=1) / 127 * 10 * U32 + 2.0**-149)
    assert torch.isnan(nscale[7:9]).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H", [(1, 1), (3, 5), (5, 9), (1, 64), (131, 512), (70, 1000), (33, 1025), (2049, 2048),
                                 (9, 4096), (600, 4100), (2, 8192), (3, 8193), (2, 16384)])
def test_norm_gradient(ops, T, H, dtype):
    for n, (gdt, with_sum) in enumerate(((F32, True), (dtype, False))):
        v, gy = normal((T, H), dtype, 40 + n, 1.5), normal((T, H), dtype, 50 + n)
        gamma = (1 + 0.3 * normal((H,), F32, 60 + n)).to(gdt)
        gs = normal((T, H), dtype, 70 + n) if with_sum else None
        leaf, g64 = v.double().requires_grad_(True), gamma.double().requires_grad_(True)
        y = leaf / torch.sqrt(leaf.square().mean(dim=1, keepdim=True) + EPS) * g64
        rx, rg = torch.autograd.grad(y, (leaf, g64), gy.double())
        rx = rx + (0 if gs is None else gs.double())
        _, r, _ = norm_reference(v, gamma, None)
        u, d = v.double() * r, gy.double() * gamma.double()
        # each of the three terms: its factors' roundings (at most 12 together) and the additions'
        terms = r * d.abs() + r * u.abs() * (d * u).abs().mean(dim=1, keepdim=True) + (0 if gs is None else gs.double().abs())
        gx, gg = ops.MoeAddRmsNormGrad(gy.cuda(), v.cuda(), gamma.cuda(), cuda(gs), EPS)
        check(gx, rx, half_step(rx, dtype) * (1 + U32) + terms * 14 * U32, (n, "grad_x"))
        check(gg, rg, half_step(rg, gdt) * (1 + U32) + (gy.double() * u).abs().sum(dim=0) * (T + 8) * U32, (n, "grad_gamma"))
        only_x, none = ops.MoeAddRmsNormGrad(gy.cuda(), v.cuda(), gamma.cuda(), cuda(gs), EPS, gradGamma=False)
        none2, only_g = ops.MoeAddRmsNormGrad(gy.cuda(), v.cuda(), gamma.cuda(), cuda(gs), EPS, gradX=False)
        assert none is none2 is None and torch.equal(only_x, gx) and torch.equal(only_g, gg)


@gpu
def test_norm_gradient_against_differences(ops):
    """Directional differences of the 64-bit norm (step 1e-4: error 1e-8 of it) along random directions."""
    x, gamma, gy = normal((6, 96), F32, 1), 1 + 0.2 * normal((96,), F32, 2), normal((6, 96), F32, 3)
    gx, gg = ops.MoeAddRmsNormGrad(gy.cuda(), x.cuda(), gamma.cuda(), None, EPS)
    for seed in range(4):
        dx, dg = normal((6, 96), F64, 10 + seed), normal((96,), F64, 20 + seed)
        h = 1e-4
        up = norm_reference(x.double() + h * dx, gamma.double() + h * dg, None)[2]
        down = norm_reference(x.double() - h * dx, gamma.double() - h * dg, None)[2]
        want = float(((up - down) / (2 * h) * gy.double()).sum())
        got = float((gx.double().cpu() * dx).sum() + (gg.double().cpu() * dg).sum())
        assert abs(got - want) <= 1e-4 * 6 * 96**0.5, (got, want)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,H", [(1, 1), (3, 6), (5, 17), (1, 8192), (2100, 1408), (70, 2047), (2049, 8000), (2, 20000),
                                 (2, 50000)])
def test_quantize(ops, R, H, dtype):
    x = normal((R, H), dtype, 3, 0.7)
    q, scale = ops.MoeQuantize(x.cuda())
    rq, top = quant_reference(x.float())
    assert torch.equal(q.cpu(), rq)
    check(scale, top.double() / 127, top.double() / 127 * U32)


@gpu
def test_quantize_ties_go_to_even_and_weights_by_channel(ops):
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5]])
    q, scale = ops.MoeQuantize(x.cuda())
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, -2, 126, -126]] and scale.tolist() == [1.0]
    w = normal((3, 10, 24), F16, 1).cuda()
    q, scale = ops.MoeQuantize(w)
    for e in range(3):
        a, b = ops.MoeQuantize(w[e])
        assert torch.equal(q[e], a) and torch.equal(scale[e], b)


def permute_reference(ids, E):
    """(slots in the order of their experts, offsets, position), one pick after another."""
    T, K = ids.shape
    flat = ids.reshape(-1).tolist()
    bucket = [e if 0 <= e < E else E for e in flat]
    order = sorted(range(T * K), key=lambda s: (bucket[s], s))
    offsets = [sum(b < e for b in bucket) for e in range(E + 1)]
    position = [0] * (T * K)
    for place, s in enumerate(order):
        position[s] = place if bucket[s] < E else -1 - place
    return order, torch.tensor(offsets, dtype=torch.int32), torch.tensor(position, dtype=torch.int32).view(T, K)


SORTS = [  # T, H, E, K: one workgroup's slots and several chunks of them, whole tokens a chunk, the most experts and picks
    (1, 1, 1, 1), (1, 8, 256, 256), (3, 7, 5, 2), (128, 64, 16, 2), (1000, 17, 64, 4), (511, 40, 256, 8), (1366, 5, 3, 3),
    (4097, 9, 2, 1), (1400, 33, 7, 3), (2050, 24, 64, 6), (40, 12, 255, 130), (3000, 16, 256, 8), (20000, 3, 17, 1),
    (1024, 10, 5, 1), (1025, 10, 5, 1), (1024, 9, 64, 8), (1025, 9, 64, 8), (33, 9, 256, 256), (40000, 8, 33, 7)]


@gpu
@pytest.mark.parametrize("T,H,E,K", SORTS)
def test_permute_and_back(ops, T, H, E, K):
    for n, dtype in enumerate((F16, F32, torch.int8)):
        ids = torch.randint(0, E, (T, K), generator=gen(n), dtype=torch.int32)
        if n:  # picks of no expert, a token without any, one expert that all others share
            ids[torch.rand((T, K), generator=gen(9)) < 0.2] = -1
            ids[T // 2] = E + 3
            ids[ids % 3 == 1] = E // 2
        x = torch.randint(-127, 128, (T, H), generator=gen(5)).to(dtype)
        scale = torch.rand(T, generator=gen(6)) if n else None
        rows, offsets, position, rscale = ops.MoePermute(x.cuda(), ids.cuda(), E, cuda(scale))
        order, roff, rpos = permute_reference(ids, E)
        assert torch.equal(offsets.cpu(), roff) and torch.equal(position.cpu(), rpos)
        token, live = torch.tensor(order) // K, torch.arange(T * K) < roff[-1]
        want = torch.where(live[:, None], x[token], torch.zeros((), dtype=dtype))
        assert torch.equal(rows.cpu(), want)
        assert rscale is None if scale is None else torch.equal(rscale.cpu(), torch.where(live, scale[token], 0.0))
        if dtype == torch.int8:
            continue
        w = torch.rand((T, K), generator=gen(7), dtype=F64).to((F16, F32)[n])
        y, plain = ops.MoeUnpermute(rows, position, w.cuda()), ops.MoeUnpermute(rows, position)
        on = (rpos >= 0).double()
        ref = (on * w.double()).sum(dim=1, keepdim=True) * x.double()
        size = (on * w.double()).sum(dim=1, keepdim=True) * x.double().abs()
        check(y, ref, half_step(ref, dtype) * (1 + U32) + size * (K + 1) * U32)
        ref = on.sum(dim=1, keepdim=True) * x.double()
        check(plain, ref, half_step(ref, dtype) * (1 + U32) + ref.abs() * K * U32)


@gpu
@pytest.mark.parametrize("T,H,E,K", [(1, 1, 1, 1), (5, 7, 3, 2), (33, 9, 8, 8), (130, 1056, 64, 6), (2049, 264, 16, 3),
                                     (2100, 129, 5, 4), (9, 4100, 256, 17)])
@pytest.mark.parametrize("dtype", TYPES)
def test_unpermute_gradient(ops, T, H, E, K, dtype):
    for n, wdt in enumerate((F32, F16, BF16)):
        ids = torch.randint(-1 if n else 0, E, (T, K), generator=gen(n), dtype=torch.int32)
        _, _, rpos = permute_reference(ids, E)
        rows, gy, w = normal((T * K, H), dtype, 1), normal((T, H), dtype, 2), normal((T, K), wdt, 3)
        grad_rows, grad_w = ops.MoeUnpermuteGrad(gy.cuda(), rows.cuda(), rpos.cuda(), w.cuda())
        live, at = rpos >= 0, torch.where(rpos >= 0, rpos, -1 - rpos).long()
        want = torch.zeros((T * K, H), dtype=F64)
        want[at.reshape(-1)] = ((w.double() * live)[:, :, None] * gy.double()[:, None, :]).view(T * K, H)
        check(grad_rows, want, half_step(want, dtype) * (1 + U32) + want.abs() * U32)
        products = rows.double()[at] * gy.double()[:, None, :] * live[:, :, None]
        ref = products.sum(dim=2)
        check(grad_w, ref, half_step(ref, wdt) * (1 + U32) + products.abs().sum(dim=2) * (H + 1) * U32)
        only, none = ops.MoeUnpermuteGrad(gy.cuda(), None, rpos.cuda())
        want[at.reshape(-1)] = (live[:, :, None] * gy.double()[:, None, :]).view(T * K, H)
        assert none is None and torch.equal(only.double().cpu(), want)


@gpu
def test_values_of_picks_of_no_expert_do_not_reach_a_result(ops):
    """NaN and infinities in the rows and weights of picks of no expert, and positions outside the rows."""
    ids = torch.tensor([[0, -1], [2, 1], [-1, -1], [7, 0]], dtype=torch.int32)
    _, _, pos = permute_reference(ids, 3)
    rows, w = normal((8, 24), F16, 1), normal((4, 2), F32, 2)
    clean, cw = rows.clone(), w.clone()
    rows[4:] = float("nan")
    w[ids < 0] = float("inf")
    w[3, 0] = float("nan")
    y = ops.MoeUnpermute(rows.cuda(), pos.cuda(), w.cuda())
    assert torch.equal(y, ops.MoeUnpermute(clean.cuda(), pos.cuda(), cw.cuda())) and torch.isfinite(y).all()
    assert (y[2] == 0).all()
    gy = normal((4, 24), F16, 3).cuda()
    for a, b in zip(ops.MoeUnpermuteGrad(gy, rows.cuda(), pos.cuda(), w.cuda()),
                    ops.MoeUnpermuteGrad(gy, clean.cuda(), pos.cuda(), cw.cuda())):
        assert torch.equal(a, b)
    outside = pos.clone()
    outside[1] = torch.tensor([8, 2**31 - 1])
    assert (ops.MoeUnpermute(clean.cuda(), outside.cuda(), cw.cuda())[1] == 0).all()


@gpu
def test_no_tokens(ops):
    x, gamma, ids = torch.empty((0, 48), dtype=F16).cuda(), torch.ones(48).cuda(), torch.empty((0, 2), dtype=torch.int32).cuda()
    y, total = ops.MoeAddRmsNorm(x, gamma, x)
    assert y.shape == total.shape == (0, 48)
    q, scale, _, _ = ops.MoeAddRmsNormQuant(x, gamma)
    assert q.shape == (0, 48) and scale.shape == (0,)
    gx, gg = ops.MoeAddRmsNormGrad(x, x, gamma)
    assert gx.shape == (0, 48) and torch.equal(gg, torch.zeros(48).cuda())
    assert ops.MoeQuantize(x)[0].shape == (0, 48)
    rows, offsets, position, rs = ops.MoePermute(x, ids, 5, torch.empty(0).cuda())
    assert rows.shape == (0, 48) and offsets.tolist() == [0] * 6 and position.shape == (0, 2) and rs.shape == (0,)
    assert ops.MoeUnpermute(rows, position).shape == (0, 48)
    gr, gw = ops.MoeUnpermuteGrad(x, rows, position, torch.empty((0, 2)).cuda())
    assert gr.shape == (0, 48) and gw.shape == (0, 2)


@gpu
def test_row_operators_captured_with_changed_inputs(ops):
    """A norm, sort and way back with their gradients in one graph, replayed on changed inputs among eager calls."""
    T, H, E, K = 2500, 264, 16, 4  # several chunks of slots: with a workspace
    x, res, gamma = normal((T, H), F16, 1).cuda(), normal((T, H), F16, 2).cuda(), normal((H,), F32, 3).cuda()
    ids = torch.randint(-1, E, (T, K), generator=gen(4), dtype=torch.int32).cuda()
    w, gy = normal((T, K), F32, 5).cuda(), normal((T, H), F16, 6).cuda()

    def step():
        q, scale, y, v = ops.MoeAddRmsNormQuant(x, gamma, res, EPS, True)
        rows, offsets, position, _ = ops.MoePermute(y, ids, E)
        qrows, _, _, rscale = ops.MoePermute(q, ids, E, scale)
        out = ops.MoeUnpermute(rows, position, w)
        grows, gw = ops.MoeUnpermuteGrad(gy, rows, position, w)
        gx, gg = ops.MoeAddRmsNormGrad(ops.MoeUnpermute(grows, position), v, gamma, gy, EPS)
        return q, scale, y, v, rows, offsets, position, qrows, rscale, out, grows, gw, gx, gg

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(4):
        x.copy_(normal((T, H), F16, 20 + n))
        ids.copy_(torch.randint(-1, E, (T, K), generator=gen(30 + n), dtype=torch.int32))
        graph.replay()
        for i, (a, b) in enumerate(zip(got, step())):
            assert torch.equal(a, b), (n, i)
        torch.cuda.synchronize()


@gpu
def test_row_operators_on_another_stream(ops):
    T, H, E, K = 300, 520, 8, 2
    x, ids = normal((T, H), F16, 1).cuda(), torch.randint(0, E, (T, K), generator=gen(2), dtype=torch.int32).cuda()
    gamma, w = normal((H,), F16, 3).cuda(), normal((T, K), F32, 4).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def run(stream):
        q, scale, y, _ = ops.MoeAddRmsNormQuant(x, gamma, None, EPS, True, stream=stream)
        rows, offsets, position, _ = ops.MoePermute(y, ids, E, stream=stream)
        back = ops.MoeUnpermute(rows, position, w, stream=stream)
        grows, gw = ops.MoeUnpermuteGrad(y, rows, position, w, stream=stream)
        gx, gg = ops.MoeAddRmsNormGrad(back, x, gamma, None, EPS, stream=stream)
        return (q, scale, y, rows, offsets, position, back, grows, gw, gx, gg, *ops.MoeQuantize(back, stream=stream))

    got = run(side)
    side.synchronize()
    for a, b in zip(got, run(None)):
        assert torch.equal(a, b)


@gpu
def test_offsets_past_32_bits(ops):
    """Rows whose elements lie past 2^31: the last ones are as those of the same rows alone."""
    T, H = 70000, 32768  # 2.3e9 values
    x = torch.empty((T, H), dtype=F16, device="cuda")
    x[:4], x[-4:] = normal((4, H), F16, 1).cuda(), normal((4, H), F16, 2).cuda()
    gamma = normal((H,), F16, 3).cuda()
    q, scale, y, _ = ops.MoeAddRmsNormQuant(x, gamma, None, EPS, True)
    tail = x[-4:].contiguous()
    for a, b in zip((q[-4:], scale[-4:], y[-4:]), ops.MoeAddRmsNormQuant(tail, gamma, None, EPS, True)):
        assert torch.equal(a, b)
    del q, scale
    a, b = ops.MoeQuantize(x), ops.MoeQuantize(tail)
    assert torch.equal(a[0][-4:], b[0]) and torch.equal(a[1][-4:], b[1])
    del a, y
    ids = (torch.arange(T, dtype=torch.int32) * 7 % 3 - 1).view(T, 1).cuda()
    rows, offsets, position, _ = ops.MoePermute(x, ids, 2)
    assert offsets[-1] < T
    at = position[-4:, 0].long()
    assert torch.equal(rows[torch.where(at >= 0, at, -1 - at)], torch.where(at[:, None] >= 0, x[-4:], 0))
    back = ops.MoeUnpermute(rows, position)
    assert torch.equal(back[-4:], torch.where(at[:, None] >= 0, x[-4:], 0)) and torch.equal(back[2], rows[position[2, 0].item()])


@gpu
@pytest.mark.parametrize("T,H,K,dtype", [(6000, 2049, 6, F16), (9000, 1003, 8, BF16), (3001, 2051, 6, F32)])
def test_unpermute_gradient_of_rows_past_the_caches(ops, T, H, K, dtype):
    """Rows of more than 128 MB, which are read and written past the caches, with picks of no expert."""
    E = 16
    ids = torch.randint(-1, E, (T, K), generator=gen(1), dtype=torch.int32).cuda()
    gy, w = normal((T, H), dtype, 2).cuda(), normal((T, K), F32, 3).cuda()
    _, _, position, _ = ops.MoePermute(gy, ids, E)
    g = torch.Generator("cuda").manual_seed(4)
    rows = torch.randn((T * K, H), generator=g, device="cuda", dtype=F32).to(dtype)
    grad_rows, grad_w = ops.MoeUnpermuteGrad(gy, rows, position, w)
    only, none = ops.MoeUnpermuteGrad(gy, None, position)
    assert none is None
    live, at = position >= 0, torch.where(position >= 0, position, -1 - position).long()
    assert torch.equal(at.flatten().sort()[0], torch.arange(T * K, device="cuda"))  # every row is compared
    for k in range(K):
        on, d = live[:, k, None], gy.double()
        assert torch.equal(only[at[:, k]], torch.where(on, gy, 0)), k
        want = torch.where(on, w[:, k, None].double() * d, 0.0)
        off = (grad_rows[at[:, k]].double() - want).abs()
        assert (off <= half_step(want, dtype) * (1 + U32) + want.abs() * U32).all(), k
        products = torch.where(on, rows[at[:, k]].double() * d, 0.0)
        off = (grad_w[:, k].double() - products.sum(dim=1)).abs()
        assert (off <= products.abs().sum(dim=1) * (H + 2) * U32).all(), k


@gpu
def test_gradients_past_32_bits(ops):
    """Rows whose elements lie past 2^31, in both gradients: the last tokens'."""
    T, H = 70000, 32768
    gy = torch.empty((T, H), dtype=F16, device="cuda")
    gy[-4:] = normal((4, H), F16, 1).cuda()
    rows = torch.empty_like(gy)
    ids = (torch.arange(T, dtype=torch.int32) * 7 % 3 - 1).view(T, 1).cuda()
    position = ops.MoePermute(gy[:, :8].contiguous(), ids, 2)[2]
    at, on = position[-4:, 0].long(), position[-4:] >= 0
    at = torch.where(at >= 0, at, -1 - at)
    rows[at] = normal((4, H), F16, 2).cuda()
    w = normal((T, 1), F32, 3).cuda()
    grad_rows, grad_w = ops.MoeUnpermuteGrad(gy, rows, position, w)
    want = torch.where(on, w[-4:].double() * gy[-4:].double(), 0.0)
    assert ((grad_rows[at].double() - want).abs() <= half_step(want, F16) * (1 + U32) + want.abs() * U32).all()
    products = torch.where(on, rows[at].double() * gy[-4:].double(), 0.0)
    assert ((grad_w[-4:, 0].double() - products.sum(dim=1)).abs() <= products.abs().sum(dim=1) * (H + 2) * U32).all()
    del gy, rows, grad_rows
    T, H = 140000, 16384
    v, grad_y = torch.ones((T, H), dtype=F16, device="cuda"), torch.zeros((T, H), dtype=F16, device="cuda")
    v[-4:], grad_y[-4:] = normal((4, H), F16, 4).cuda(), normal((4, H), F16, 5).cuda()
    gamma = normal((H,), F32, 6).cuda()
    gx, gg = ops.MoeAddRmsNormGrad(grad_y, v, gamma, grad_y, EPS)
    tail, dtail = v[-4:].contiguous(), grad_y[-4:].contiguous()
    assert torch.equal(gx[-4:], ops.MoeAddRmsNormGrad(dtail, tail, gamma, dtail, EPS)[0])
    assert (gx[:8] == 0).all()
    terms = dtail.double() * norm_reference(tail, gamma, None)[1] * tail.double()  # the other rows add zeros
    assert ((gg.double() - terms.sum(dim=0)).abs() <= terms.abs().sum(dim=0) * (4 + 8) * U32).all()


# ---------------------------------------------------------------------------------------------------------------------
# refusals, on the CPU: every check runs before anything is launched
# ---------------------------------------------------------------------------------------------------------------------

P = 1 << 20  # an address that no check reads
ARG, NULL, WS, UNSUPPORTED = 4, 1, 5, 6


def norm_call(T=4, H=64, eps=1e-6, dtype=1, gtype=0, x=P, gamma=P, y=P, q=None, scale=None, xs=64, res=None, rs=0):
    return lib.load().moe_add_rms_norm(x, xs, res, rs, gamma, gtype, y, None, q, scale, T, H, eps, dtype, None)


def grad_call(T=4, H=64, eps=1e-6, dtype=1, gtype=0, gy=P, gx=P, gg=P, ws=P, wb=1 << 30, ys=64, gs=None, gss=0):
    return lib.load().moe_add_rms_norm_grad(gy, ys, P, H, P, gtype, gs, gss, gx, gg, ws, wb, T, H, eps, dtype, None)


def quantize_call(R=4, H=64, dtype=1, x=P, q=P, scale=P, xs=64):
    return lib.load().moe_quantize(x, xs, q, scale, R, H, dtype, None)


def permute_call(T=4, H=64, E=8, K=2, dtype=1, x=P, ids=P, rows=P, offsets=P, position=P, ws=P, wb=1 << 30, xs=64, sx=None,
                 sr=None):
    return lib.load().moe_permute(x, xs, sx, ids, rows, sr, offsets, position, ws, wb, T, H, E, K, dtype, None)


def unpermute_call(T=4, H=64, K=2, R=8, dtype=1, rows=P, position=P, w=P, wtype=0, y=P):
    return lib.load().moe_unpermute(rows, R, position, w, wtype, y, T, H, K, dtype, None)


def ungrad_call(T=4, H=64, K=2, dtype=1, gy=P, rows=P, position=P, w=P, wtype=0, gr=P, gw=P, ys=64):
    return lib.load().moe_unpermute_grad(gy, ys, rows, position, w, wtype, gr, gw, T, H, K, dtype, None)


NAN = float("nan")


@pytest.mark.parametrize("call,changes", [
    (norm_call, [(dict(T=-1), ARG), (dict(H=0), ARG), (dict(H=(1 << 20) + 1), UNSUPPORTED), (dict(eps=0.0), ARG),
                 (dict(eps=-1.0), ARG), (dict(eps=NAN), ARG), (dict(eps=float("inf")), ARG), (dict(dtype=2), ARG),
                 (dict(dtype=3), ARG), (dict(gtype=27), ARG), (dict(dtype=0, gtype=1), ARG), (dict(x=None), NULL),
                 (dict(gamma=None), NULL), (dict(q=P), NULL), (dict(scale=P), NULL), (dict(xs=63), ARG),
                 (dict(xs=-64), ARG), (dict(xs=1 << 41), ARG), (dict(res=P, rs=60), ARG), (dict(T=1 << 31), UNSUPPORTED)]),
    (grad_call, [(dict(T=-1), ARG), (dict(H=16385, ys=16385), UNSUPPORTED), (dict(eps=0.0), ARG), (dict(dtype=2), ARG),
                 (dict(gtype=27), ARG), (dict(gy=None), NULL), (dict(ws=None), WS), (dict(wb=255), WS),
                 (dict(ws=P + 2), UNSUPPORTED), (dict(ys=60), ARG), (dict(gs=P, gss=3), ARG)]),
    (quantize_call, [(dict(R=-1), ARG), (dict(H=0), ARG), (dict(H=(1 << 20) + 1), UNSUPPORTED), (dict(dtype=2), ARG),
                     (dict(x=None), NULL), (dict(q=None), NULL), (dict(scale=None), NULL), (dict(xs=1), ARG)]),
    (permute_call, [(dict(T=-1), ARG), (dict(K=0), ARG), (dict(K=9), ARG), (dict(E=257), UNSUPPORTED), (dict(E=0), ARG),
                    (dict(T=1 << 30), UNSUPPORTED), (dict(dtype=3), ARG), (dict(x=None), NULL), (dict(ids=None), NULL),
                    (dict(rows=None), NULL), (dict(offsets=None), NULL), (dict(position=None), NULL), (dict(sx=P), NULL),
                    (dict(sr=P), NULL), (dict(T=5000, ws=None), WS), (dict(T=5000, wb=16), WS),
                    (dict(T=5000, ws=P + 1), UNSUPPORTED), (dict(xs=63), ARG)]),
    (unpermute_call, [(dict(T=-1), ARG), (dict(K=0), ARG), (dict(R=-1), ARG), (dict(R=1 << 31), ARG), (dict(dtype=2), ARG),
                      (dict(wtype=3), ARG), (dict(rows=None), NULL), (dict(position=None), NULL), (dict(y=None), NULL),
                      (dict(T=1 << 30), UNSUPPORTED)]),
    (ungrad_call, [(dict(T=-1), ARG), (dict(K=0), ARG), (dict(dtype=2), ARG), (dict(wtype=2), ARG), (dict(gy=None), NULL),
                   (dict(rows=None), NULL), (dict(position=None), NULL), (dict(gr=None), NULL), (dict(gw=None), NULL),
                   (dict(ys=63), ARG), (dict(T=1 << 30), UNSUPPORTED)]),
])
def test_refusals(call, changes):
    assert call(T=0) == 0 if call not in (quantize_call, permute_call, grad_call) else True  # nothing to do
    for change, status in changes:
        assert call(**change) == status, (change, lib.load().moe_last_error())
        assert lib.load().moe_last_error()


def test_workspace_queries():
    L = lib.load()
    assert L.moe_permute_workspace_bytes(1024, 64, 8) == 0
    assert L.moe_permute_workspace_bytes(1025, 64, 8) == (9 * 65 + 1025 * 8) * 4
    assert L.moe_permute_workspace_bytes(-1, 64, 8) == 0 and L.moe_permute_workspace_bytes(1 << 30, 64, 8) == 0
    assert L.moe_add_rms_norm_grad_workspace_bytes(4, 16385) == 0
    assert L.moe_add_rms_norm_grad_workspace_bytes(0, 100) == 400


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros((4, 8), dtype=F16), torch.zeros((4, 2), dtype=torch.int32)
    for call in (lambda: opsm.MoeAddRmsNorm(x, x[0]), lambda: opsm.MoeAddRmsNormQuant(x, x[0]), lambda: opsm.MoeQuantize(x),
                 lambda: opsm.MoeAddRmsNormGrad(x, x, x[0]), lambda: opsm.MoePermute(x, ids, 4),
                 lambda: opsm.MoeUnpermute(x, ids), lambda: opsm.MoeUnpermuteGrad(x, None, ids)):
        with pytest.raises(MoeError, match="device tensor"):
            call()


@gpu
def test_python_refusals(ops):
    x, g, ids = normal((4, 16), F16, 1).cuda(), normal((16,), F16, 2).cuda(), torch.zeros((4, 2), dtype=torch.int32).cuda()
    pos, rows, w = ops.MoePermute(x, ids, 4)[2], normal((8, 16), F16, 3).cuda(), normal((4, 2), F32, 4).cuda()
    for call in (lambda: ops.MoeAddRmsNorm(x, g.to(BF16)), lambda: ops.MoeAddRmsNorm(x, g[:15]),
                 lambda: ops.MoeAddRmsNorm(x, g.repeat(2)[::2]), lambda: ops.MoeAddRmsNorm(x, g, x[:3]),
                 lambda: ops.MoeAddRmsNorm(x, g, x.float()), lambda: ops.MoeAddRmsNorm(x, g, eps=0.0),
                 lambda: ops.MoeAddRmsNorm(x.t(), g[:4]), lambda: ops.MoeAddRmsNorm(x[0], g),
                 lambda: ops.MoeAddRmsNormGrad(None, x, g), lambda: ops.MoeAddRmsNormGrad(x[:2], x, g),
                 lambda: ops.MoeAddRmsNormGrad(x, x, g, workspace=torch.empty(8, dtype=torch.uint8, device="cuda")),
                 lambda: ops.MoeQuantize(ids), lambda: ops.MoeQuantize(x.t()),
                 lambda: ops.MoeQuantize(rows.view(2, 4, 16).transpose(0, 1)), lambda: ops.MoePermute(x, ids[:3], 4),
                 lambda: ops.MoePermute(x, ids.long(), 4), lambda: ops.MoePermute(x, ids, 1),
                 lambda: ops.MoePermute(x, ids, 0), lambda: ops.MoePermute(x, ids, 4, w[:, 0]),
                 lambda: ops.MoePermute(x, ids[0], 4), lambda: ops.MoeUnpermute(rows, pos, w[:3]),
                 lambda: ops.MoeUnpermute(rows.t(), pos), lambda: ops.MoeUnpermute(rows, pos, w.t().contiguous().t()),
                 lambda: ops.MoeUnpermuteGrad(x, None, pos, w), lambda: ops.MoeUnpermuteGrad(x, rows[:7], pos, w),
                 lambda: ops.MoeUnpermuteGrad(x, rows, pos[:2], w)):
        with pytest.raises(MoeError):
            call()
