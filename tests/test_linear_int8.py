"""MoeLinearInt8, one product and those of experts, against 64-bit sums of the same integers.

Tolerances: the int32 sums are exact; their conversion to fp32, the product with the row's scale and that with the
column's round once each (3 * 2^-24 of the scaled sum), the bias's addition and the residual's once; activations as in
test_dense_ops (FN and their slopes); the result's rounding is half a step of its type."""
from __future__ import annotations

import math

import pytest

from test_dense_ops import BF16, F16, F32, FN, U32, MoeError, act_reference, check, gen, gpu, half_step, normal, opsm
from test_row_ops import ARG, NULL, UNSUPPORTED, WS, P

torch = pytest.importorskip("torch")
lib = opsm._lib
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu", "swiglu")


def int8(shape, seed, low=-127):
    return torch.randint(low, 128, shape, generator=gen(seed)).to(torch.int8)


def scales(shape, seed, H):
    return (0.5 + torch.rand(shape, generator=gen(seed))) / (60 * H**0.25)


def operands(T, Z, H, E, out, seed, bias, residual, N):
    lead = (E,) if E else ()
    return dict(x=int8((T, H), seed), xs=scales((T,), seed + 1, H), w=int8((*lead, Z, H), seed + 2),
                ws=scales((*lead, Z), seed + 3, H), bias=normal((*lead, Z), out, seed + 4) if bias else None,
                residual=normal((T, N), out, seed + 5) if residual else None)


def reference(x, xs, w, ws, bias, residual, act):
    """(result, its tolerance before the last rounding) in 64 bits, on the tensors' device."""
    z = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    zt = 3 * U32 * z.abs()
    if bias is not None:
        z = z + bias.double()
        zt = zt + U32 * z.abs()
    ref = act_reference(z, act)
    if act == "swiglu":  # |silu'| <= 1.1
        (g, u), (gt, ut) = z.chunk(2, dim=1), zt.chunk(2, dim=1)
        tol = 1.1 * gt * (u.abs() + ut) + g.abs() * ut + FN * ref.abs()
    else:
        tol = zt if act == "none" else 1.13 * zt + FN * z.abs()
    if residual is not None:
        ref = ref + residual.double()
        tol = tol + U32 * ref.abs()
    return ref, tol


def reference_experts(o, offsets, act, N):
    T = o["x"].shape[0]
    ref = torch.zeros((T, N), dtype=torch.float64, device=o["x"].device)
    tol = torch.zeros_like(ref)
    edges = offsets.tolist()
    for e, (a, b) in enumerate(zip(edges, edges[1:])):
        if b > a:
            ref[a:b], tol[a:b] = reference(o["x"][a:b], o["xs"][a:b], o["w"][e], o["ws"][e],
                                           None if o["bias"] is None else o["bias"][e],
                                           None if o["residual"] is None else o["residual"][a:b], act)
    return ref, tol


def on_gpu(o):
    return {k: None if v is None else v.cuda() for k, v in o.items()}


def call(ops, o, offsets, act, out, **kw):
    return ops.MoeLinearInt8(o["x"], o["xs"], o["w"], o["ws"], offsets, o["bias"], o["residual"], act, out, **kw)


def run_case(ops, T, N, H, act, out, bias, residual, offsets=None, seed=0):
    E = 0 if offsets is None else offsets.numel() - 1
    Z = 2 * N if act == "swiglu" else N
    o = on_gpu(operands(T, Z, H, E, out, seed, bias, residual, N))
    y = call(ops, o, None if offsets is None else offsets.cuda(), act, out)
    if E:
        ref, tol = reference_experts(o, offsets, act, N)
    else:
        ref, tol = reference(o["x"], o["xs"], o["w"], o["ws"], o["bias"], o["residual"], act)
    check(y, ref.cpu(), (tol + half_step(ref.abs() + tol, out)).cpu(), (T, N, H, act))
    return o, y


SIZES = [  # T, N, H: streams of up to 16, 32 and 64 rows, tiles of 32 to 256, split and whole, aligned or not
    (1, 1, 1), (1, 8, 16), (2, 3, 7), (5, 40, 100), (1, 130, 1008), (16, 72, 2048), (17, 2050, 144), (31, 4100, 80),
    (33, 24, 4096), (48, 1040, 528), (64, 1100, 272), (65, 128, 17), (100, 200, 1001), (130, 257, 129), (150, 96, 8192),
    (257, 300, 2064), (300, 1, 48), (515, 700, 64), (1, 2816, 7168)]


@gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T,N,H", SIZES)
def test_sizes(ops, T, N, H, act):
    out = (F16, BF16, F32)[(T + N + H) % 3]
    run_case(ops, T, N, H, act, out, bias=(T + N) % 2 == 0, residual=(N + H) % 2 == 0, seed=T + N)


@gpu
@pytest.mark.parametrize("T,N,H,act,out", [(1000, 2048, 1408, "none", F16), (4097, 515, 2048, "silu", BF16),
                                           (2049, 1056, 1040, "swiglu", F16), (8192, 2816, 2048, "swiglu", BF16),
                                           (16384, 256, 7168, "none", F32), (3000, 4096, 32, "gelu", F32),
                                           (4096, 4096, 4096, "none", BF16)])
def test_large_tiles(ops, T, N, H, act, out):
    run_case(ops, T, N, H, act, out, bias=True, residual=act == "none")


def cuts(T, E, seed, dropped=0, empty=0.2):
    """Offsets of E experts over T - dropped rows: uneven, some without rows."""
    share = torch.rand(E, generator=gen(seed), dtype=torch.float64)**3 * (torch.rand(E, generator=gen(seed + 1)) >= empty)
    share[-1] += 1e-9
    edges = torch.round(torch.cumsum(share / share.sum(), 0) * (T - dropped))
    return torch.cat([torch.zeros(1), edges]).to(torch.int32)


GROUPS = [  # T, N, H, E: rows an expert from none to hundreds, 1 to 256 experts, aligned or not
    (1, 8, 16, 1), (1, 24, 64, 256), (7, 33, 48, 3), (40, 64, 1040, 64), (300, 72, 96, 16), (300, 130, 33, 16),
    (700, 520, 144, 65), (900, 257, 1001, 6), (2000, 100, 272, 17), (2100, 136, 64, 255), (3000, 128, 128, 4),
    (4100, 300, 520, 7), (5000, 640, 80, 130), (6000, 512, 176, 2)]


@gpu
@pytest.mark.parametrize("act", ("none", "swiglu", "gelu"))
@pytest.mark.parametrize("T,N,H,E", GROUPS)
def test_experts(ops, T, N, H, E, act):
    for n, dropped in enumerate((0, T // 10)):
        out = (F16, BF16, F32)[(T + E + n) % 3]
        offsets = cuts(T, E, T + n, dropped)
        _, y = run_case(ops, T, N, H, act, out, bias=n == 0, residual=n == 1, offsets=offsets, seed=E)
        assert (y[int(offsets[-1]):] == 0).all()


@gpu
@pytest.mark.parametrize("T,N,H,act,out", [(8192, 2816, 2048, "swiglu", BF16), (8192, 2816, 2048, "swiglu", F16),
                                           (16381, 1032, 1040, "none", F16), (9001, 2056, 528, "none", BF16),
                                           (5000, 4104, 272, "swiglu", F16)])
def test_large_tiles_without_bias_and_residual(ops, T, N, H, act, out):
    """16-bit results that need scales alone, which tiles of 256 rows write by a way of their own; every value."""
    run_case(ops, T, N, H, act, out, bias=False, residual=False, seed=T)


@gpu
@pytest.mark.parametrize("act", ("none", "swiglu"))
@pytest.mark.parametrize("out", (F16, BF16))
@pytest.mark.parametrize("T,N,H,E", [(300, 264, 96, 9), (2300, 1408, 272, 64), (1300, 520, 1040, 9), (5100, 72, 64, 33),
                                     (1500, 264, 96, 9), (6000, 1032, 528, 4), (40000, 136, 80, 200)])
def test_experts_without_bias_and_residual(ops, T, N, H, E, act, out):
    """The same of experts: 33 to 159 rows each on average, where half tiles without rows are left out, and more."""
    for dropped in (0, T // 7):
        offsets = cuts(T, E, T + dropped, dropped)
        _, y = run_case(ops, T, N, H, act, out, bias=False, residual=False, offsets=offsets, seed=E)
        assert (y[int(offsets[-1]):] == 0).all()


@gpu
@pytest.mark.parametrize("T,E", [(40, 5), (400, 9), (1200, 8), (4000, 6)])
def test_experts_with_all_or_no_rows(ops, T, E):
    for filled in (0, E // 2, E - 1):
        offsets = torch.tensor([0] * (filled + 1) + [T] * (E - filled), dtype=torch.int32)
        run_case(ops, T, 72, 160, "swiglu", F16, True, False, offsets)
    _, y = run_case(ops, T, 72, 160, "none", F32, True, True, torch.zeros(E + 1, dtype=torch.int32))
    assert (y == 0).all()


@gpu
def test_sums_up_to_32_bits_are_exact(ops):
    """The longest row of the largest values, 131071 * 2^14 = 2^31 - 2^14, both signs."""
    H = 131071
    x = torch.full((2, H), -128, dtype=torch.int8)
    x[1] = 127
    w = torch.full((3, H), -128, dtype=torch.int8)
    w[1], w[2, ::2] = 127, 5
    one = torch.ones(3).cuda()
    want = (x.double() @ w.double().t()).float()
    for T in (1, 2):
        y = ops.MoeLinearInt8(x[:T].cuda(), one[:T], w.cuda(), one, outDtype=F32)
        assert torch.equal(y.cpu(), want[:T])
    H = 131056  # a multiple of 16: streamed, and split over H by tiles
    for T in (2, 100):
        xs, ws = x[1:, :H].repeat(T, 1).cuda(), w[:, :H].contiguous().cuda()
        y = ops.MoeLinearInt8(xs.contiguous(), torch.ones(T).cuda(), ws, one, outDtype=F32)
        assert torch.equal(y.cpu(), (xs.double().cpu() @ ws.double().cpu().t()).float())


@gpu
@pytest.mark.parametrize("T,N,H", [(3, 20, 48), (20, 300, 160), (100, 70, 80), (500, 300, 528)])
def test_strides_alignment_and_what_stands_beside_the_operands(ops, T, N, H):
    """Operands inside larger tensors of 127s: the same results, for each offset and pitch."""
    o = on_gpu(operands(T, N, H, 0, F16, 3, True, True, N))
    want = call(ops, o, None, "none", F16)

    def framed(t, pad, at):
        f = torch.full((t.shape[0] + 2, H + pad), 127, dtype=torch.int8, device="cuda")
        f[1:-1, at:at + H] = t
        return f[1:-1, at:at + H]

    for pad, at in ((16, 0), (32, 16), (1, 0), (7, 3), (16, 8)):
        got = call(ops, dict(o, x=framed(o["x"], pad, at), w=framed(o["w"], pad, at)), None, "none", F16)
        assert torch.equal(got, want), (pad, at)
    E = 3
    offsets = torch.tensor([0, T // 3, T // 2, T], dtype=torch.int32).cuda()
    o = on_gpu(operands(T, N, H, E, F16, 5, True, True, N))
    want = call(ops, o, offsets, "none", F16)
    for pad in (16, 5):
        big = torch.full((E, N + 1, H + pad), 127, dtype=torch.int8, device="cuda")
        big[:, :N, pad:] = o["w"]
        assert torch.equal(call(ops, dict(o, w=big[:, :N, pad:]), offsets, "none", F16), want), pad


@gpu
def test_one_expert_is_the_product_alone(ops):
    for T in (1, 30, 90, 700, 2000):
        o = on_gpu(operands(T, 136, 272, 0, F16, T, True, True, 136))
        y = call(ops, o, None, "silu", F16)
        e = dict(o, w=o["w"][None], ws=o["ws"][None], bias=o["bias"][None])
        assert torch.equal(call(ops, e, torch.tensor([0, T], dtype=torch.int32).cuda(), "silu", F16), y)


@gpu
@pytest.mark.parametrize("act", ("none", "swiglu"))
@pytest.mark.parametrize("out", (F16, BF16, F32))
def test_results_do_not_depend_on_the_launch(ops, act, out):
    """Rows of a large product without bias and residual, from tiles of 256 rows, and the same rows alone: streamed, from
    smaller tiles, split over H, and as an expert's."""
    T, N, H = 9000, 2048, 2048
    o = on_gpu(operands(T, 2 * N if act == "swiglu" else N, H, 0, out, 8, False, False, N))
    full = call(ops, o, None, act, out)
    for rows in (1, 20, 64, 100, 300, 1500):
        some = dict(o, x=o["x"][:rows], xs=o["xs"][:rows])
        assert torch.equal(call(ops, some, None, act, out), full[:rows]), rows
        for E in (1, 8):  # of 8 experts the third has all rows
            offsets = torch.tensor([0] * (1 + E // 4) + [rows] * (E - E // 4), dtype=torch.int32).cuda()
            many = dict(some, w=o["w"][None].expand(E, -1, -1).contiguous(), ws=o["ws"][None].expand(E, -1).contiguous())
            assert torch.equal(call(ops, many, offsets, act, out), full[:rows]), (rows, E)


@gpu
@pytest.mark.parametrize("T,E", [(30, 4), (200, 4), (1200, 4)])
def test_offsets_that_lie_stay_within_the_tensors(ops, T, E):
    """Offsets that fall, pass the end or are negative: guards before and after the result keep their values."""
    N, H = 40, 64
    o = on_gpu(operands(T, N, H, E, F32, 1, False, False, N))
    for values in ([0, T + 50, T + 60, 3, T], [-9, -5, 2**31 - 1, 5, 6], [5, 4, 3, 2, 1], [0, -2**31, 7, -1, 9]):
        y = torch.full((T + 2 * 64, N), 3.5, device="cuda")
        offsets = torch.tensor(values, dtype=torch.int32).cuda()
        st = lib.load().moe_linear_int8(o["x"].data_ptr(), H, o["xs"].data_ptr(), o["w"].data_ptr(), H, N * H,
                                        o["ws"].data_ptr(), offsets.data_ptr(), None, None, y[64:].data_ptr(), None, 0, T, N,
                                        H, E, 0, 0, torch.cuda.current_stream().cuda_stream)
        assert st == 0
        assert (y[:64] == 3.5).all() and (y[T + 64:] == 3.5).all()
        if values[0] == 5:  # the first expert's rows begin at 0 whatever the offset says
            ref, tol = reference(o["x"][:4], o["xs"][:4], o["w"][0], o["ws"][0], None, None, "none")
            check(y[64:68], ref.cpu(), (tol + half_step(ref.abs() + tol, F32)).cpu())


@gpu
@pytest.mark.parametrize("T,E,at", [(30, 4, 0), (50, 70, 0), (200, 9, 0), (600, 130, 0), (640, 9, 0), (200, 9, 1), (1200, 9, 1),
                                    (1500, 9, 0), (5000, 9, 0), (2000, 256, 0)])
def test_offsets_that_lie_give_every_row_one_expert(ops, T, E, at):
    """Streams and every height of tiles: an expert ends at its offset within [0, T] or where the last one did if that is
    further, and begins there, so each row is as with the offsets of which that is true. at: odd addresses."""
    N, H = 72, 64
    o = on_gpu(operands(T, N, H, E, F32, 1, True, True, N))
    frame = torch.zeros(T * H + 16, dtype=torch.int8, device="cuda")
    x = frame[at:at + T * H].view(T, H)
    x.copy_(o["x"])
    u = torch.randint(-T, 2 * T, (E + 1,), generator=gen(E))
    lies = {"there and back": [0] + [T * (e % 2 == 0) for e in range(E)], "falling": [T - e for e in range(E + 1)],
            "the last below": [0] + [T // 2] * (E - 1) + [T // 3], "far": [2**31 - 1] + [-2**31, T // 2] * E, "any": u.tolist()}
    for name, values in lies.items():
        offsets = torch.tensor(values[:E + 1], dtype=torch.int32)
        honest = offsets.long().clamp(0, T)
        honest[0] = 0
        honest = honest.cummax(0)[0].to(torch.int32)
        y = torch.full((T, N), float("nan"), device="cuda")
        off = offsets.cuda()
        st = lib.load().moe_linear_int8(x.data_ptr(), H, o["xs"].data_ptr(), o["w"].data_ptr(), H, N * H, o["ws"].data_ptr(),
                                        off.data_ptr(), o["bias"].data_ptr(), o["residual"].data_ptr(), y.data_ptr(), None, 0,
                                        T, N, H, E, 0, 0, torch.cuda.current_stream().cuda_stream)
        assert st == 0 and torch.equal(y, call(ops, dict(o, x=x), honest.cuda(), "none", F32)), name
        ref, tol = reference_experts(o, honest, "none", N)
        check(y, ref.cpu(), (tol + half_step(ref.abs() + tol, F32)).cpu(), name)


@gpu
def test_residual_that_is_the_result(ops):
    T, N, H = 70, 136, 256
    o = on_gpu(operands(T, N, H, 0, F16, 2, True, True, N))
    want, y = call(ops, o, None, "none", F16), o["residual"].clone()
    need = ops.linear_int8_workspace_bytes(T, N, H)
    ws = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    st = lib.load().moe_linear_int8(o["x"].data_ptr(), H, o["xs"].data_ptr(), o["w"].data_ptr(), H, 0, o["ws"].data_ptr(),
                                    None, o["bias"].data_ptr(), y.data_ptr(), y.data_ptr(), ws.data_ptr(), need, T, N, H, 0,
                                    0, 1, torch.cuda.current_stream().cuda_stream)
    assert st == 0 and torch.equal(y, want)


@gpu
def test_split_sums_stay_in_the_workspace(ops):
    T, N, H = 100, 72, 8192
    need = ops.linear_int8_workspace_bytes(T, N, H)
    assert need > 0
    o = on_gpu(operands(T, N, H, 0, F32, 2, True, False, N))
    ws = torch.full((need + 256,), 0x7f, dtype=torch.uint8, device="cuda")
    y = call(ops, o, None, "gelu", F32, workspace=ws)
    assert (ws[need:] == 0x7f).all() and torch.equal(y, call(ops, o, None, "gelu", F32))
    with pytest.raises(MoeError):
        call(ops, o, None, "gelu", F32, workspace=ws[:need - 16])


@gpu
def test_nan_scales_stay_in_their_rows_and_columns(ops):
    """What MoeQuantize makes of a row with an infinity: scale NaN, integers 0."""
    o = on_gpu(operands(40, 48, 64, 0, F16, 2, False, False, 48))
    o["xs"][7], o["ws"][9] = float("nan"), float("inf")
    o["x"][7] = 0
    bad = ~torch.isfinite(call(ops, o, None, "none", F16))
    assert bad[7].all() and bad[:, 9].all()
    bad[7], bad[:, 9] = False, False
    assert not bad.any()


@gpu
def test_captured_with_changed_offsets_and_on_another_stream(ops):
    T, N, H, E = 600, 200, 272, 12
    o = on_gpu(operands(T, N, H, E, F16, 4, True, False, N))
    one = on_gpu(operands(100, 72, 8192, 0, F16, 5, True, False, 72))  # split: with a workspace
    offsets = cuts(T, E, 1).cuda()

    def step(stream=None):
        return call(ops, o, offsets, "silu", F16, stream=stream), call(ops, one, None, "silu", F16, stream=stream)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(4):
        offsets.copy_(cuts(T, E, 20 + n, dropped=30 * n))
        one["x"].copy_(int8((100, 8192), 30 + n))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), n
        torch.cuda.synchronize()


@gpu
def test_weights_past_32_bits(ops):
    """Experts whose weights lie past 2^32 bytes, and rows of x and of the result past 2^31."""
    E, N, H, T = 36, 8192, 16384, 72  # 4.8 GB
    w = torch.zeros((E, N, H), dtype=torch.int8, device="cuda")
    for e in (0, 33, 35):
        w[e] = int8((N, H), e).cuda()
    xs, ws = scales((T,), 1, H).cuda(), scales((E, N), 2, H).cuda()
    x, offsets = int8((T, H), 3).cuda(), (torch.arange(E + 1) * 2).to(torch.int32).cuda()
    y = ops.MoeLinearInt8(x, xs, w, ws, offsets, outDtype=F32)
    for e in (0, 33, 35):
        ref, tol = reference(x[2 * e:2 * e + 2], xs[2 * e:2 * e + 2], w[e], ws[e], None, None, "none")
        check(y[2 * e:2 * e + 2], ref.cpu(), (tol + half_step(ref.abs() + tol, F32)).cpu(), e)
    del w, y
    T, N, H = 300000, 7200, 8192  # x 2.4e9, y 2.1e9 values
    x = torch.zeros((T, H), dtype=torch.int8, device="cuda")
    rows = torch.tensor([0, 1, T // 2, T - 2, T - 1]).cuda()
    x[rows] = int8((5, H), 1).cuda()
    w, xs, ws = int8((N, H), 2).cuda(), scales((T,), 3, H).cuda(), scales((N,), 4, H).cuda()
    for offsets in (None, torch.tensor([0, T], dtype=torch.int32).cuda()):
        y = ops.MoeLinearInt8(x, xs, w if offsets is None else w[None], ws if offsets is None else ws[None], offsets)
        ref, tol = reference(x[rows], xs[rows], w, ws, None, None, "none")
        check(y[rows], ref.cpu(), (tol + half_step(ref.abs() + tol, F16)).cpu())
        del y


# ---------------------------------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------------------------------


def c_call(T=4, N=24, H=64, E=0, act=0, out=1, x=P, xs=P, w=P, ws=P, off=P, y=P, ldx=64, ldw=64, step=1 << 16, work=None,
           wb=0):
    return lib.load().moe_linear_int8(x, ldx, xs, w, ldw, step, ws, off, None, None, y, work, wb, T, N, H, E, act, out, None)


@pytest.mark.parametrize("change,status", [
    (dict(T=-1), ARG), (dict(N=0), ARG), (dict(H=0), ARG), (dict(E=-1), ARG), (dict(E=257), UNSUPPORTED),
    (dict(H=131072, ldx=131072, ldw=131072), UNSUPPORTED), (dict(N=(1 << 20) + 1), UNSUPPORTED), (dict(act=6), ARG),
    (dict(act=-1), ARG), (dict(out=2), ARG), (dict(out=3), ARG), (dict(ldx=63), ARG), (dict(ldw=63), ARG),
    (dict(ldx=-64), ARG), (dict(E=2, step=100), ARG), (dict(E=2, step=-1), ARG), (dict(x=None), NULL), (dict(xs=None), NULL),
    (dict(w=None), NULL), (dict(ws=None), NULL), (dict(y=None), NULL), (dict(E=2, off=None), NULL),
    (dict(T=100, H=8192, ldx=8192, ldw=8192), WS), (dict(T=100, H=8192, ldx=8192, ldw=8192, work=P, wb=64), WS),
    (dict(T=100, H=8192, ldx=8192, ldw=8192, work=P + 8, wb=1 << 30), UNSUPPORTED), (dict(T=1 << 31), UNSUPPORTED),
    (dict(T=1 << 30, E=2), UNSUPPORTED)])
def test_refusals(change, status):
    assert c_call(**change) == status, lib.load().moe_last_error()
    assert lib.load().moe_last_error()


def test_nothing_to_do_and_workspace_queries():
    assert c_call(T=0, x=None, y=None) == 0
    L = lib.load()
    assert L.moe_linear_int8_workspace_bytes(100, 72, 8192, 4, 0) == 0
    assert L.moe_linear_int8_workspace_bytes(100, 72, 8192, 0, 0) > 0
    assert L.moe_linear_int8_workspace_bytes(100, 72, 8192, 0, 9) == 0
    x = torch.zeros((4, 16), dtype=torch.int8)
    with pytest.raises(MoeError, match="device tensor"):
        opsm.MoeLinearInt8(x, torch.ones(4), x, torch.ones(4))


@gpu
def test_python_refusals(ops):
    o = on_gpu(operands(6, 10, 32, 0, F16, 1, True, True, 10))
    g = on_gpu(operands(6, 10, 32, 2, F16, 1, True, True, 10))
    off = torch.tensor([0, 2, 6], dtype=torch.int32).cuda()
    for change in (dict(x=o["x"].half()), dict(w=o["w"].half()), dict(xs=o["xs"][:5]), dict(xs=None), dict(ws=None),
                   dict(ws=o["ws"].half()), dict(w=o["w"][:, :31]), dict(bias=o["bias"][:9]), dict(bias=o["bias"].float()),
                   dict(residual=o["residual"][:5]), dict(residual=o["residual"].float()), dict(w=g["w"]),
                   dict(x=int8((32, 6), 1).cuda().t()), dict(w=int8((32, 10), 1).cuda().t())):
        with pytest.raises(MoeError):
            call(ops, {**o, **change}, None, "none", F16)
    for change, offsets in ((dict(), off[:2]), (dict(), off.long()), (dict(w=o["w"]), off), (dict(ws=o["ws"]), off),
                            (dict(bias=o["bias"]), off), (dict(w=g["w"][:0]), off[:1])):
        with pytest.raises(MoeError):
            call(ops, {**g, **change}, offsets, "none", F16)
    for act, out in (("swiglu", torch.int8), ("tanh", F16)):
        with pytest.raises(MoeError):
            call(ops, o, None, act, out)
    odd = on_gpu(operands(6, 9, 32, 0, F16, 1, False, False, 9))
    with pytest.raises(MoeError):
        call(ops, odd, None, "swiglu", F16)
