"""Quantised and permuted expert layers through torch: shapes on fake tensors here; gradients, opcheck, compilation and
the whole layer on the GPU."""
from __future__ import annotations

import importlib

import pytest

from conftest import PKG_NAME
from test_dense_ops import BF16, F16, F32, F64, U32, check, gen, gpu, half_step, normal

torch = pytest.importorskip("torch")
tops = importlib.import_module(PKG_NAME + ".torch_ops")
op = torch.ops.moe_mi355x


def meta(*shape, dtype=F16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_meta_shapes():
    x, g, ids = meta(7, 64), meta(64), meta(7, 3, dtype=torch.int32)
    y, v = op.MoeAddRmsNorm(x, g, x)
    assert y.shape == v.shape == (7, 64) and op.MoeAddRmsNorm(x, g)[1].numel() == 0
    q, s, y, v = op.MoeAddRmsNormQuant(x, g, None, 1e-6, True)
    assert (q.dtype, s.dtype, s.shape, y.shape, v.numel()) == (torch.int8, F32, (7,), (7, 64), 0)
    gx, gg = op.MoeAddRmsNormGrad(x, x, g, None, 1e-6, True, False)
    assert gx.shape == (7, 64) and gg.numel() == 0
    q, s = op.MoeQuantize(meta(4, 10, 64))
    assert q.shape == (4, 10, 64) and s.shape == (4, 10)
    rows, off, pos, rs = op.MoePermute(q[0], meta(10, 2, dtype=torch.int32), 5, s[0])
    assert (rows.shape, rows.dtype, off.shape, pos.shape, rs.shape) == ((20, 64), torch.int8, (6,), (10, 2), (20,))
    y = op.MoeUnpermute(meta(21, 64), ids, meta(7, 3))
    assert y.shape == (7, 64)
    gr, gw = op.MoeUnpermuteGrad(y, meta(21, 64), ids, meta(7, 3, dtype=F32))
    assert (gr.shape, gr.dtype, gw.shape, gw.dtype) == ((21, 64), F16, (7, 3), F32)
    y = op.MoeLinearInt8(rows, rs, meta(5, 24, 64, dtype=torch.int8), meta(5, 24, dtype=F32), off, activation="swiglu")
    assert (y.shape, y.dtype) == ((20, 12), F16)
    for call in (lambda: op.MoeAddRmsNorm(x, meta(63)), lambda: op.MoePermute(x, meta(6, 2, dtype=torch.int32), 4),
                 lambda: op.MoeLinearInt8(rows, rs, meta(24, 63, dtype=torch.int8), s), lambda: op.MoeQuantize(g),
                 lambda: op.MoeUnpermute(x, ids, meta(7, 2))):
        with pytest.raises(RuntimeError):
            call()


def test_cpu_tensors_have_no_kernel():
    with pytest.raises(NotImplementedError):
        op.MoeQuantize(torch.zeros(4, 64))
    with pytest.raises(NotImplementedError):
        op.MoeAddRmsNorm(torch.zeros(4, 64), torch.ones(64))


def leaf(t):
    return t.cuda().requires_grad_(True)


def inputs(T=45, H=96, E=8, K=3, dtype=F32):
    ids = torch.stack([torch.randperm(E, generator=gen(t))[:K] for t in range(T)]).to(torch.int32)
    ids[5, 1] = -1
    return (normal((T, H), dtype, 1), normal((T, H), dtype, 2), 1 + 0.2 * normal((H,), F32, 3), ids,
            torch.rand((T, K), generator=gen(4)))


def sorted_layer(x, res, gamma, ids, w, E):
    """A norm, the tokens by expert, something that differs by expert, and back; the sum goes on beside it."""
    y, v = op.MoeAddRmsNorm(x, gamma, res, 1e-5)
    rows, offsets, position, _ = op.MoePermute(y, ids, E)
    return op.MoeUnpermute(rows * rows, position, w) + v


@gpu
def test_gradients_through_torch(ops):
    """Against torch's differentiation of the definition in 64 bits. fp32 throughout: each value passes at most about 40
    roundings (norm 8, square 1, sum 4, their gradients twice that), and those of grad_gamma T sums more."""
    x, res, gamma, ids, w = inputs()
    args = [leaf(t) for t in (x, res, gamma, w)]
    dy = normal(x.shape, F32, 9)
    out = sorted_layer(args[0], args[1], args[2], ids.cuda(), args[3], 8)
    got = torch.autograd.grad(out, args, dy.cuda())
    a, b, g, k = (t.double().requires_grad_(True) for t in (x, res, gamma, w))
    v = a + b
    n = v / torch.sqrt(v.square().mean(dim=1, keepdim=True) + 1e-5) * g
    ref = n * n * (k * (ids >= 0)).sum(dim=1, keepdim=True) + v
    want = torch.autograd.grad(ref, (a, b, g, k), dy.double())
    scale = [float(t.abs().max()) for t in want]
    assert (out.double().cpu() - ref).abs().max() <= 40 * 2.0**-24 * float(ref.detach().abs().max())
    for u, r, s, n in zip(got, want, scale, (1, 1, 45, 96)):
        assert (u.double().cpu() - r).abs().max() <= (60 + n) * 2.0**-24 * s * 4
    assert torch.equal(got[0], got[1])


@gpu
def test_parts_that_need_no_gradient(ops):
    x, res, gamma, ids, w = inputs()
    X, R, G = leaf(x), leaf(res), leaf(gamma)
    y, v = op.MoeAddRmsNorm(X, G, R)
    gx, gr = torch.autograd.grad(v.sum(), (X, R), retain_graph=True)  # the sum alone
    assert torch.equal(gx, torch.ones_like(gx)) and torch.equal(gr, gx)
    gx, = torch.autograd.grad(y.sum() + v.sum(), X, retain_graph=True)
    gy, = torch.autograd.grad(y.sum(), X)
    assert torch.allclose(gx - 1, gy, atol=1e-5)  # 1 + gy rounded to fp32: within 2^-24 of at most 16
    y, _ = op.MoeAddRmsNorm(x.cuda(), G)
    assert torch.autograd.grad(y.sum(), G)[0].shape == G.shape
    rows, _, position, _ = op.MoePermute(leaf(x), ids.cuda(), 8)
    g, = torch.autograd.grad(op.MoeUnpermute(rows, position).sum(), rows)
    live = (ids >= 0).sum()
    assert g[:live].eq(1).all() and g[live:].eq(0).all()
    with pytest.raises(RuntimeError, match="one for each pick"):
        more = leaf(torch.zeros(200, 96))
        torch.autograd.grad(op.MoeUnpermute(more, position).sum(), more)


@gpu
@pytest.mark.parametrize("dtype", [torch.int8, F16, F32])
def test_scales_sorted_with_their_rows_have_a_gradient(ops, dtype):
    """Of a loss that takes row_scale: the sum over a token's picks, those of no expert left out (K - 1 fp32 additions)."""
    T, H, E, K = 45, 24, 8, 3
    ids = torch.randint(-1, E, (T, K), generator=gen(1), dtype=torch.int32)
    x = torch.randint(-127, 128, (T, H), generator=gen(2)).to(dtype)
    scale, d = leaf(torch.rand(T, generator=gen(3))), normal((T * K,), F32, 4)
    X = x.cuda() if dtype == torch.int8 else leaf(x)
    rows, _, position, row_scale = op.MoePermute(X, ids.cuda(), E, scale)
    at = torch.where(ids >= 0, position.cpu(), 0).long()
    terms = d.double()[at] * (ids >= 0)
    got, = torch.autograd.grad(row_scale, scale, d.cuda(), retain_graph=True)
    check(got, terms.sum(dim=1), terms.abs().sum(dim=1) * K * U32)
    if dtype == torch.int8:
        return
    dr = normal((T * K, H), dtype, 5)
    both = torch.autograd.grad((rows, row_scale), (X, scale), (dr.cuda(), d.cuda()), retain_graph=True)
    assert torch.equal(both[1], got)
    alone, = torch.autograd.grad(rows, X, dr.cuda(), retain_graph=True)
    assert torch.equal(both[0], alone)
    assert torch.autograd.grad(row_scale, X, d.cuda(), allow_unused=True, retain_graph=True)[0] is None
    assert torch.autograd.grad(rows, scale, dr.cuda(), allow_unused=True)[0] is None


def any_positions(T, K, kind):
    """Positions that MoeUnpermute takes and MoePermute does not give."""
    position = torch.randperm(T * K, generator=gen(T)).to(torch.int32).view(T, K)
    u = torch.rand((T, K), generator=gen(K))
    if kind == "masked":  # no expert's without a place, and past the rows
        position[u < 0.2], position[u > 0.9], position[u > 0.95] = -1, T * K, 2**31 - 1
        position[0] = -2**31
    elif kind == "shared":
        position = torch.where(u < 0.5, position // 3, position)
    elif kind == "one row":
        position[:] = T * K - 1
    else:
        position //= kind
    return position


@gpu
@pytest.mark.parametrize("T,H,K,dtype", [(1, 1, 1, F32), (40, 7, 3, BF16), (33, 9, 8, F16), (300, 1056, 4, BF16),
                                         (2049, 264, 3, F32), (130, 2051, 6, F16), (5000, 72, 2, F32)])
@pytest.mark.parametrize("kind", ["masked", "shared", 2, 63, 64, 65, "one row"])
def test_way_back_has_the_gradient_of_any_positions(ops, T, H, K, dtype, kind):
    """Rows that no pick, one or many name, against 64-bit sums: a row's is of at most T K products in fp32."""
    position = any_positions(T, K, kind)
    rows, dy = normal((T * K, H), dtype, 1), normal((T, H), dtype, 2)
    on = (position >= 0) & (position < T * K)
    at = torch.where(on, position, 0).long()
    for wdt in (None, F32, F16):
        w = None if wdt is None else normal((T, K), wdt, 3)
        args = [leaf(t) for t in (rows, w) if t is not None]
        y = op.MoeUnpermute(args[0], position.cuda(), *args[1:])
        got = torch.autograd.grad(y, args, dy.cuda())
        terms = on[:, :, None] * (1.0 if w is None else w.double()[:, :, None]) * dy.double()[:, None]
        want = torch.zeros((T * K, H), dtype=F64).index_add_(0, at.flatten(), terms.flatten(0, 1))
        size = torch.zeros((T * K, H), dtype=F64).index_add_(0, at.flatten(), terms.abs().flatten(0, 1))
        many = torch.bincount(at[on], minlength=T * K)[:, None]
        check(got[0], want, half_step(want, dtype) * (1 + U32) + size * (many + 1) * U32, "rows")
        if w is not None:
            products = on[:, :, None] * rows.double()[at] * dy.double()[:, None]
            ref = products.sum(dim=2)
            check(got[1], ref, half_step(ref, wdt) * (1 + U32) + products.abs().sum(dim=2) * (H + 1) * U32, "weights")
        y = op.MoeUnpermute(args[0], position.cuda(), *args[1:])
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, args, dy.cuda()), got))


@gpu
@pytest.mark.parametrize("T,H,E,K,dtype", [(45, 96, 8, 3, F32), (2100, 1031, 16, 4, BF16), (1, 5, 2, 2, F16)])
def test_gradient_of_any_positions_is_that_of_sorted_ones(ops, T, H, E, K, dtype):
    ids = torch.randint(-1, E, (T, K), generator=gen(1), dtype=torch.int32).cuda()
    dy, w = normal((T, H), dtype, 2).cuda(), normal((T, K), F32, 3).cuda()
    rows, _, position, _ = ops.MoePermute(normal((T, H), dtype, 4).cuda(), ids, E)
    need = ops.unpermute_grad_any_workspace_bytes(T, K)
    assert need == 8 * T * K
    room = torch.full((need + 64,), 0x7f, dtype=torch.uint8, device="cuda")
    for a, b in zip(ops.MoeUnpermuteGrad(dy, rows, position, w),
                    ops.MoeUnpermuteGrad(dy, rows, position, w, anyPosition=True, workspace=room)):
        assert torch.equal(a, b)
    assert (room[need:] == 0x7f).all()
    assert torch.equal(ops.MoeUnpermuteGrad(dy, None, position)[0],
                       ops.MoeUnpermuteGrad(dy, None, position, anyPosition=True)[0])
    with pytest.raises(ops.MoeError):
        ops.MoeUnpermuteGrad(dy, rows, position, w, anyPosition=True, workspace=room[:need - 4])


@gpu
def test_gradient_of_any_positions_captured_with_changed_ones(ops):
    """On another stream, with rows of an odd length and gradients any stride apart; every replay against an eager call."""
    T, H, K = 700, 333, 4
    dy, rows = normal((T, H + 5), F16, 1).cuda()[:, 2:2 + H], normal((T * K, H), F16, 2).cuda()
    position, w = any_positions(T, K, "masked").cuda(), normal((T, K), F32, 3).cuda()

    def step(stream=None):
        return ops.MoeUnpermuteGrad(dy, rows, position, w, stream, True)

    want, side = step(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for kind in ("shared", 65, "masked", "one row"):
        position.copy_(any_positions(T, K, kind))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), kind
        torch.cuda.synchronize()


def test_gradient_of_any_positions_refuses_like_the_other():
    L, P = tops.ops._lib.load(), 1 << 20

    def call(T=4, H=64, K=2, dtype=1, gy=P, rows=P, position=P, w=P, wtype=0, gr=P, gw=P, ys=64, ws=P, wb=1 << 30):
        return L.moe_unpermute_grad_any(gy, ys, rows, position, w, wtype, gr, gw, ws, wb, T, H, K, dtype, None)

    assert call(T=0, gy=None, gr=None, ws=None) == 0
    for change, status in ((dict(T=-1), 4), (dict(K=0), 4), (dict(dtype=2), 4), (dict(wtype=2), 4), (dict(gy=None), 1),
                           (dict(rows=None), 1), (dict(position=None), 1), (dict(gr=None), 1), (dict(gw=None), 1),
                           (dict(ys=63), 4), (dict(T=1 << 30), 6), (dict(ws=None), 5), (dict(wb=63), 5),
                           (dict(ws=P + 2), 6)):
        assert call(**change) == status, (change, L.moe_last_error())
    assert L.moe_unpermute_grad_any_workspace_bytes(4, 2) == 64
    assert L.moe_unpermute_grad_any_workspace_bytes(-1, 2) == L.moe_unpermute_grad_any_workspace_bytes(1 << 30, 2) == 0


@gpu
def test_opcheck(ops):
    x, res, gamma, ids, w = (t.cuda() for t in inputs(dtype=F16))
    # with results of whole numbers torch's own test of the traced gradient adds their sums to those of floats, and fails
    utils = ("test_schema", "test_faketensor", "test_autograd_registration")

    def check(fn, args, utils=utils):
        torch.library.opcheck(fn, args, test_utils=utils)

    for args in ((leaf(x), leaf(gamma), leaf(res), 1e-5), (leaf(x), leaf(gamma))):
        check(op.MoeAddRmsNorm, args, utils + ("test_aot_dispatch_dynamic",))
    check(op.MoeAddRmsNormQuant, (x, gamma, res, 1e-5, True))
    check(op.MoeQuantize, (x,))
    check(op.MoePermute, (leaf(x), ids, 8))
    q, s = op.MoeQuantize(x)
    check(op.MoePermute, (q, ids, 8, s))
    rows, off, pos, rs = op.MoePermute(q, ids, 8, s)
    check(op.MoeUnpermute, (leaf(rows.half()), pos, leaf(w)), utils + ("test_aot_dispatch_dynamic",))
    wq, ws = op.MoeQuantize(normal((8, 40, 96), F16, 5).cuda())
    check(op.MoeLinearInt8, (rows, rs, wq, ws, off, None, None, "swiglu", BF16))


def layer_inputs(T, H, E, I, dtype):
    gate_up = normal((E, 2 * I, H), dtype, 5, H**-0.5)
    down = normal((E, H, I), dtype, 6, I**-0.5)
    return (normal((T, H), dtype, 1), normal((T, H), dtype, 2), 1 + 0.2 * normal((H,), F32, 3),
            normal((H, E), dtype, 4, 2 * H**-0.5), gate_up, down)


@gpu
@pytest.mark.parametrize("T,H,E,I,K,dtype", [(1, 256, 8, 128, 2, F16), (45, 96, 16, 80, 3, BF16), (700, 512, 8, 384, 2, BF16),
                                             (2500, 256, 64, 144, 6, F16)])
def test_int8_layer_is_its_parts_and_near_the_definition(ops, T, H, E, I, K, dtype):
    x, res, gamma, w_gate, gate_up, down = (t.cuda() for t in layer_inputs(T, H, E, I, dtype))
    (gq, gs), (dq, ds) = ops.MoeQuantize(gate_up), ops.MoeQuantize(down)
    y, v, ids, w = ops.moe_layer_int8(x, gamma, w_gate, gq, gs, dq, ds, res, K, scoring="sigmoid", eps=1e-5)
    q, qs, n, v2 = ops.MoeAddRmsNormQuant(x, gamma, res, 1e-5, True)
    rows, off, pos, rs = ops.MoePermute(q, ids, E, qs)
    hidden = ops.MoeLinearInt8(rows, rs, gq, gs, off, activation="swiglu", outDtype=dtype)
    hq, hs = ops.MoeQuantize(hidden)
    part = ops.MoeLinearInt8(hq, hs, dq, ds, off, outDtype=dtype)
    assert torch.equal(y, ops.MoeUnpermute(part, pos, w)) and torch.equal(v, v2)
    # the layer that its 8-bit weights and inputs stand for, in 64 bits, from the ids and weights chosen
    W1, W2 = gq.double() * gs.double()[:, :, None], dq.double() * ds.double()[:, :, None]
    a, h8 = q.double() * qs.double()[:, None], torch.zeros((T, K, H), dtype=F64, device="cuda")
    for e in range(E):
        t, k = (ids == e).nonzero(as_tuple=True)
        if len(t):
            g, u = (a[t] @ W1[e].t()).chunk(2, dim=1)
            h = g * torch.sigmoid(g) * u
            step = h.abs().amax(dim=1, keepdim=True) / 127
            # rounded to dtype before it is quantised: a quantised value may be one step off near a border
            h8[t, k] = torch.round(h / step) * step @ W2[e].t()
    ref = (h8 * w.double()[:, :, None]).sum(dim=1)
    # a step of hidden (1/127 of its row's largest value, some 3.5 of its rms) off by half in the rare value, the rounding of
    # hidden to dtype moving a share of 127 eps of them over a border: sqrt(127 eps) / 127 * 3.5 of the result, its own
    # rounding and that of the products' results eps / 2 each; compared by their root mean squares, twice that
    eps = torch.finfo(dtype).eps
    off_by = float((y.double() - ref).norm() / ref.norm())
    assert off_by <= 2 * ((min(1.0, 127 * eps)) ** 0.5 / 127 * 3.5 + 2 * eps), off_by


@gpu
def test_int8_layer_captured_and_compiled(ops):
    x, res, gamma, w_gate, gate_up, down = (t.cuda() for t in layer_inputs(200, 128, 8, 96, F16))
    (gq, gs), (dq, ds) = ops.MoeQuantize(gate_up), ops.MoeQuantize(down)

    def step():
        return ops.moe_layer_int8(x, gamma, w_gate, gq, gs, dq, ds, res, 2)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(3):
        x.copy_(normal(x.shape, F16, 50 + n))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), n
        torch.cuda.synchronize()

    def through_torch(x):
        q, s, y, v = op.MoeAddRmsNormQuant(x, gamma, res, 1e-6, True)
        ids, w = op.MoeRoutingGroupTopK(op.MoeLinear(y, w_gate.t(), outDtype=F32)[0], topK=2, weightsDtype=F32)
        rows, off, pos, rs = op.MoePermute(q, ids, 8, s)
        h, hs = op.MoeQuantize(op.MoeLinearInt8(rows, rs, gq, gs, off, activation="swiglu"))
        return op.MoeUnpermute(op.MoeLinearInt8(h, hs, dq, ds, off), pos, w), v

    want = step()
    for fn in (through_torch, torch.compile(through_torch, fullgraph=True)):
        assert all(torch.equal(a, b) for a, b in zip(fn(x), want[:2]))


@gpu
def test_training_step_in_a_graph(ops):
    """Forward and backward as a whole, captured after warm-up steps whose results are dropped."""
    x, res, gamma, ids, w = inputs(T=64)
    ids = ids.cuda()
    leaves = [leaf(t) for t in (x, res, gamma, w)]

    def step():
        grads = torch.autograd.grad(sorted_layer(leaves[0], leaves[1], leaves[2], ids, leaves[3], 8).square().sum(), leaves)
        return [g.clone() for g in grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(3):
        with torch.no_grad():
            leaves[0].copy_(normal(x.shape, F32, 70 + n))
        graph.replay()
        torch.cuda.synchronize()
        kept = [g.clone() for g in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, step())), n


@gpu
def test_layer_refusals(ops):
    x, res, gamma, w_gate, gate_up, down = (t.cuda() for t in layer_inputs(4, 64, 4, 32, F16))
    (gq, gs), (dq, ds) = ops.MoeQuantize(gate_up), ops.MoeQuantize(down)
    with pytest.raises(ops.MoeError):
        ops.moe_layer_int8(x, gamma, w_gate, gq[:3], gs, dq, ds, res)
    with pytest.raises(ops.MoeError):
        ops.moe_layer_int8(x, gamma, w_gate, gq, gs[:3], dq, ds, res)


@gpu
@pytest.mark.parametrize("T,H,E,I,K", [(0, 64, 4, 32, 2), (1, 64, 1, 16, 1), (7, 100, 4, 33, 2), (300, 257, 8, 129, 3)])
def test_layer_of_odd_sizes_on_another_stream(ops, T, H, E, I, K):
    """Rows on odd addresses; a layer without a residual is the one with a residual of zeros."""
    x, _, gamma, w_gate, gate_up, down = (t.cuda() for t in layer_inputs(T, H, E, I, BF16))
    wide = torch.empty((T, H + 8), dtype=BF16, device="cuda")
    wide[:, 3:H + 3] = x
    (gq, gs), (dq, ds) = ops.MoeQuantize(gate_up), ops.MoeQuantize(down)
    y, v, ids, w = ops.moe_layer_int8(x, gamma, w_gate, gq, gs, dq, ds, None, K)
    assert v is None and y.shape == (T, H) and ids.shape == w.shape == (T, K) and y.isfinite().all()
    zeros, side = torch.zeros_like(x), torch.cuda.Stream()
    torch.cuda.synchronize()
    other = ops.moe_layer_int8(wide[:, 3:H + 3], gamma, w_gate, gq, gs, dq, ds, zeros, K, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(y, other[0]) and torch.equal(other[1], x) and torch.equal(ids, other[2])
