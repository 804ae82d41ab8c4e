"""The operators around the routed experts at their limits: offsets past 32 bits, calls in flight on two streams, graphs
replayed on changed inputs by every kind of plan, and random sizes against 64 bits.

Where operands are whole numbers below 2^11 whose sums stay below 2^24, every product and sum is exact in fp32 in any order:
those results are compared for equality."""
from __future__ import annotations

import importlib
import random

import pytest

from conftest import PKG_NAME

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
U32 = 2.0**-24


def ones(shape, seed, dtype=F16):
    """-1, 0 or 1, on the GPU, in `dtype`."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-1, 2, shape, generator=g, device="cuda", dtype=torch.int8).to(dtype)


def test_linear_and_its_gradients_past_32_bits(ops):
    """x and grad_x hold 2.2e9 elements. Sums of up to 8192 and 16 products of -1, 0 and 1 are exact in fp32 and fp16's
    whole numbers; of 270000 below 2^24 in fp32, and their roundings to fp16 equal."""
    T, N, H = 270000, 16, 8192
    x, w, dy = ones((T, H), 1), ones((N, H), 2), ones((T, N), 3)
    y = ops.MoeLinear(x, w, outDtype=F32)
    gx, gw, gb = ops.MoeLinearGrad(dy, x, w, gradBias=True)
    sums = torch.zeros((N, H), dtype=F64, device="cuda")
    for t in range(0, T, 30000):
        at = slice(t, t + 30000)
        part = x[at].float()
        assert torch.equal(y[at], part @ w.float().t())
        assert torch.equal(gx[at].float(), dy[at].float() @ w.float())
        sums += (dy[at].float().t().contiguous() @ part).double()
    assert torch.equal(gw, sums.to(F16))
    assert torch.equal(gb, dy.double().sum(dim=0).to(F16))


def test_routing_and_its_gradient_past_32_bits(ops):
    T, E, K = (1 << 23) + 1001, 256, 4  # 2^31 logits and more
    logits = torch.empty((T, E), dtype=F16, device="cuda")
    for t in range(0, T, 1 << 20):
        logits[t:t + (1 << 20)] = torch.randn((min(1 << 20, T - t), E), device="cuda").to(F16)
    ids, w = ops.MoeRoutingGroupTopK(logits, None, K, 8, 4, 1, "sigmoid")
    gw = torch.randn((T, K), device="cuda").to(F16)
    grad = ops.MoeRoutingGroupTopKGrad(gw, logits, ids, "sigmoid")
    for t in (0, (1 << 22) - 500, T - 2003):  # a part by itself: the same rows, small offsets
        at = slice(t, t + 2003)
        part = logits[at].clone()
        pids, pw = ops.MoeRoutingGroupTopK(part, None, K, 8, 4, 1, "sigmoid")
        assert torch.equal(ids[at], pids) and torch.equal(w[at], pw)
        assert torch.equal(grad[at], ops.MoeRoutingGroupTopKGrad(gw[at].clone(), part, pids, "sigmoid"))


@pytest.mark.parametrize("E,G,TG,GT", [(65, 13, 5, 2), (100, 1, 1, 1), (256, 8, 4, 2), (256, 128, 9, 2)])
@pytest.mark.parametrize("scoring,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_routing_of_many_rows_is_that_of_few(ops, E, G, TG, GT, scoring, renorm):
    """A row's choice and weights do not depend on how many rows the call has, which decides how many lanes a row gets."""
    T = 2500
    g = torch.Generator(device="cuda").manual_seed(E + G)
    logits = torch.randn((T, E), generator=g, device="cuda")
    logits[torch.rand((T, E), generator=g, device="cuda") < 0.2] = float("-inf")
    logits[7] = float("-inf")
    logits[8] = torch.finfo(F32).min
    logits[9:40] = (logits[9:40] * 4).round() / 4  # ties
    logits[40, 1] = float("nan")
    bias = ((torch.rand((E,), generator=g, device="cuda") - 0.5) * 0.2 * 64).round() / 64
    for dtype, b in ((F32, None), (F32, bias), (F16, None), (BF16, bias)):
        x = logits.to(dtype)
        ids, w = ops.MoeRoutingGroupTopK(x, b, 8, G, TG, GT, scoring, renorm, 2.0, F32)
        for t in range(0, T, 500):
            at = slice(t, t + 500)
            pids, pw = ops.MoeRoutingGroupTopK(x[at], b, 8, G, TG, GT, scoring, renorm, 2.0, F32)
            assert torch.equal(ids[at], pids) and torch.equal(w[at], pw)


@pytest.mark.parametrize("T", [3, 2500])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_equal_scores_go_to_the_lowest_index(ops, T, scoring):
    """All 256 candidates equal, with a bias: the choice goes on to a clear gap, which is the row's end."""
    E = 256
    logits, bias = torch.full((T, E), -1.5, device="cuda"), torch.full((E,), 0.25, device="cuda")
    logits[1] = torch.finfo(F32).min
    logits[2, ::2] = float("-inf")
    want = torch.arange(8, device="cuda", dtype=torch.int32)
    for G, TG in ((1, 1), (8, 4)):
        ids, w = ops.MoeRoutingGroupTopK(logits, bias, 8, G, TG, 2, scoring, True, 1.0, F32)
        assert torch.equal(ids[0], want) and torch.equal(ids[1], want) and torch.equal(ids[2], 2 * want + 1)
        assert torch.equal(w, torch.full_like(w, 0.125))
        assert T == 3 or torch.equal(ids[3:], want.expand(T - 3, 8))


@pytest.mark.parametrize("T,N,H,act", [(1, 72, 256, 0), (64, 4096, 136, 0), (40, 64, 4096, 0), (300, 200, 1024, 5),
                                       (2304, 2304, 128, 0)])
def test_residual_may_be_the_result(ops, T, N, H, act):
    lib = ops._lib.load()
    x, w = ones((T, H), 1), ones(((2 if act else 1) * N, H), 2)
    y = ones((T, N), 3)
    want = ops.MoeLinear(x, w, residual=y, activation="swiglu" if act else "none")
    need = ops.linear_workspace_bytes(T, N, H, "swiglu" if act else "none")
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    st = lib.moe_linear(x.data_ptr(), H, w.data_ptr(), H, 0, None, y.data_ptr(), y.data_ptr(), None, ws.data_ptr(), need, T,
                        N, H, act, 1, 1, torch.cuda.current_stream().cuda_stream)
    assert st == 0, lib.moe_last_error()
    assert torch.equal(y, want)


def test_combine_gradient_past_32_bits(ops):
    T, H, K = 140001, 2048, 8  # 2.3e9 elements
    eo, dy = ones((T, K, H), 4), ones((T, H), 5)
    w = (ones((T, K), 6) * 0.5 + 1.0).to(F16)
    geo, gw = ops.MoeCombineGrad(dy, eo, w)
    for t in range(0, T, 10000):
        at = slice(t, t + 10000)
        assert torch.equal(geo[at], w[at].unsqueeze(2) * dy[at].unsqueeze(1))
        assert torch.equal(gw[at], (eo[at] * dy[at].unsqueeze(1)).float().sum(dim=2).to(F16))


def test_two_calls_in_flight(ops):
    """Two streams, each with its own inputs and workspaces, in kernels that split their sums over k."""
    T, N, H = 300, 520, 4096
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    sets = []
    for n in range(2):
        x, w = ones((T, H), 10 + n), ones((N, H), 20 + n)
        dy = ones((T, N), 30 + n)
        logits = torch.randn((T, 256), generator=torch.Generator(device="cuda").manual_seed(n), device="cuda")
        sets.append((x, w, dy, logits, torch.empty(ops.linear_workspace_bytes(T, N, H), dtype=torch.uint8, device="cuda"),
                     torch.empty(ops.linear_grad_workspace_bytes(T, N, H), dtype=torch.uint8, device="cuda")))

    def step(n, stream=None):
        x, w, dy, logits, ws, gws = sets[n]
        return (ops.MoeLinear(x, w, outDtype=F32, workspace=ws, stream=stream),
                *ops.MoeLinearGrad(dy, x, w, gradBias=True, workspace=gws, stream=stream),
                *ops.MoeRoutingGroupTopK(logits, None, 8, 8, 4, 2, "sigmoid", stream=stream))

    alone = [step(0), step(1)]
    torch.cuda.synchronize()
    both = []
    for _ in range(8):
        both.append([step(n, streams[n]) for n in range(2)])
    torch.cuda.synchronize()
    for out in both:
        for n in range(2):
            for a, b in zip(alone[n], out[n]):
                assert torch.equal(a, b)
    assert torch.equal(alone[0][0], sets[0][0].float() @ sets[0][1].float().t())


PLANS = [  # T, N, H, activation, transposed: each kind of plan of the product and of its gradients
    (1, 64, 512, "swiglu", False), (48, 2048, 256, "relu", False), (60, 96, 4096, "none", True),
    (100, 130, 2048, "gelu", False), (77, 45, 131, "silu", True), (77, 45, 131, "swiglu", True),
    (2000, 1024, 1024, "none", False), (2304, 2304, 256, "swiglu", False), (1500, 1500, 1500, "none", True)]


@pytest.mark.parametrize("T,N,H,act,transposed", PLANS)
def test_graph_replays_on_changed_inputs(ops, T, N, H, act, transposed):
    Z = 2 * N if act == "swiglu" else N
    x = torch.empty((T, H), dtype=F16, device="cuda")
    w = torch.empty((H, Z), dtype=F16, device="cuda").t() if transposed else torch.empty((Z, H), dtype=F16, device="cuda")
    dy, bias = torch.empty((T, N), dtype=F16, device="cuda"), torch.empty((Z,), dtype=F16, device="cuda")

    def fill(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (x, w, dy, bias):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda") * 0.25)

    def step():
        y = ops.MoeLinear(x, w, bias, None, act, returnPre=act != "none")
        y, pre = y if act != "none" else (y, None)
        return (y,) + ops.MoeLinearGrad(dy, x, w, pre, act, gradBias=True)

    fill(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(1, 5):
        fill(seed)
        for t in out:
            t.fill_(float("nan"))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert torch.equal(a, b)


def test_combine_gradient_and_router_replayed_on_changed_inputs(ops):
    T, H, K, E = 333, 520, 3, 96
    eo, dy = torch.empty((T, K, H), dtype=F16, device="cuda"), torch.empty((T, H), dtype=F16, device="cuda")
    logits, bias = torch.empty((T, E), device="cuda"), torch.empty((E,), device="cuda")

    def step():
        ids, w = ops.MoeRoutingGroupTopK(logits, bias, K, 6, 2, 2, "softmax")
        geo, gw = ops.MoeCombineGrad(dy, eo, w)
        return ids, w, geo, gw, ops.MoeRoutingGroupTopKGrad(gw, logits, ids, "softmax")

    graph, out = None, None
    for seed in range(5):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (eo, dy, logits, bias):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        eager = step()
        torch.cuda.synchronize()
        if graph is None:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T,N,H,act", [(1, 8190, 72, "none"), (16, 4100, 520, "none"), (17, 8184, 264, "none"),
                                       (33, 16384, 64, "none"), (64, 4100, 2040, "none"), (64, 16381, 1032, "none"),
                                       (5, 2310, 136, "swiglu"), (23, 4091, 200, "swiglu"), (64, 2816, 712, "swiglu")])
def test_weight_streaming_by_tiles_of_32_rows(ops, T, N, H, act):
    """Few rows against weights of more than one round of 16-row tiles: sums exact, so those of `pre` are equal too."""
    halves = 2 if act == "swiglu" else 1
    x, w, bias = ones((T, H), 1), ones((halves * N, H), 2), ones((halves * N,), 3)
    res = ones((T, N), 4)
    y, pre = ops.MoeLinear(x, w, bias, res, act, returnPre=True)
    z = x.float() @ w.float().t() + bias.float()
    assert torch.equal(pre, z.to(F16))
    if act == "none":
        assert torch.equal(y, (z + res.float()).to(F16))
    else:  # the sigmoid within 8 fp32 roundings, its products and the sum one each, then the result's
        g, u = z.double().chunk(2, dim=1)
        p = g / (1.0 + torch.exp(-g)) * u
        ref = p + res.double()
        tol = 16 * U32 * (p.abs() + ref.abs())
        assert ((y.double() - ref).abs() <= tol + (ref.abs() + tol) * 2.0**-11 + 2.0**-25).all()


@pytest.mark.parametrize("seed", range(24))
def test_random_sizes_without_activation(ops, seed):
    """Any size, layout, alignment and row stride: whole numbers, compared for equality, so a term lost, repeated or read
    past an operand's end shows. Everything around the operands holds NaN."""
    rng = random.Random(seed)

    def size(hi):
        return max(1, round(hi ** rng.random()))

    T, N, H = size(3000), size(1500), size(3000)
    dtype = rng.choice((F16, BF16))

    def inside(rows, cols, s):
        """`rows` x `cols` whole numbers inside a larger NaN tensor, at an odd or even place and stride."""
        pad, at, before = rng.choice((0, 1, 8, 24)), rng.choice((0, 1, 8)), rng.choice((0, 1, 3))
        wide = torch.full((rows + before + 2, cols + pad + at), float("nan"), dtype=dtype, device="cuda")
        view = wide[before:before + rows, at:at + cols]
        view.copy_(ones((rows, cols), s, dtype))
        return view

    x, dy = inside(T, H, seed), inside(T, N, seed + 100)
    w = inside(H, N, seed + 200).t() if rng.random() < 0.4 else inside(N, H, seed + 200)
    bias = ones((N,), seed + 300, dtype)
    y = ops.MoeLinear(x, w, bias, outDtype=F32)
    assert torch.equal(y, x.float() @ w.float().t() + bias.float()), (T, N, H)
    gx, gw, gb = ops.MoeLinearGrad(dy, x, w, gradBias=True)
    assert torch.equal(gx, (dy.float() @ w.float()).to(dtype)), (T, N, H)
    assert torch.equal(gw, (dy.float().t() @ x.float()).to(dtype)), (T, N, H)
    assert torch.equal(gb, dy.float().sum(dim=0).to(dtype)), (T, N, H)
