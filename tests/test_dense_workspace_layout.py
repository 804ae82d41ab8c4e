"""MoeLinear's and MoeLinearGrad's workspaces hold what the weight's layout needs, not copies that are never made."""
from __future__ import annotations

import importlib

import pytest

from conftest import PKG_NAME
from test_dense_ops import F16, U32, half_step, normal

torch = pytest.importorskip("torch")
opsm = importlib.import_module(PKG_NAME + ".ops")


def test_no_room_for_copies_that_are_not_made():
    """Rows of 8192 values are read in place, whatever the number of weight rows."""
    assert opsm.linear_workspace_bytes(1, 50257, 8192, transposed=False) < 1 << 20
    assert opsm.linear_workspace_bytes(1, 50257, 8192, transposed=True) >= 50264 * 8192 * 2
    assert opsm.linear_workspace_bytes(1, 50257, 8192) >= opsm.linear_workspace_bytes(1, 50257, 8192, transposed=True)
    few = opsm.linear_grad_workspace_bytes(64, 4100, 8192, transposed=False)
    many = opsm.linear_grad_workspace_bytes(64, 4100, 8192, transposed=True)
    assert many - few >= 8192 * 4104 * 2 and opsm.linear_grad_workspace_bytes(64, 4100, 8192) >= many
    # rows that are no multiple of 16 bytes are copied in the layout that has them
    assert opsm.linear_workspace_bytes(5, 64, 8191, transposed=False) >= (5 + 64) * 8192 * 2
    assert opsm.linear_workspace_bytes(5, 64, 8191, transposed=True) < 64 * 8192 * 2


def test_layout_calls_refuse_a_byte_less():
    lib = importlib.import_module(PKG_NAME + "._lib").load()
    for T, N, H, act in ((1, 50257, 8192, 0), (5, 64, 8191, 0), (70, 41, 65, 5), (300, 130, 2048, 4), (64, 4100, 7168, 0)):
        Z = 2 * N if act == 5 else N
        for tr in (0, 1):
            ld = Z if tr else H
            need = lib.moe_linear_layout_workspace_bytes(T, N, H, act, tr)
            if need:
                assert lib.moe_linear_layout(16, H, 16, ld, tr, None, None, 16, None, 16, need - 1, T, N, H, act, 1, 1,
                                             None) == 5
            need = lib.moe_linear_grad_layout_workspace_bytes(T, N, H, act, tr)
            assert lib.moe_linear_grad_layout(16, N, 16, H, 16, ld, tr, 16, 16, 16, 16, 16, need - 1, T, N, H, act, 1, None) == 5
    assert lib.moe_linear_layout_workspace_bytes(-1, 8, 8, 0, 0) == 0
    assert lib.moe_linear_grad_layout_workspace_bytes(4, 8, 8, 9, 0) == 0


@pytest.mark.gpu
def test_a_wide_weight_takes_no_second_copy(ops):
    """One token through 50257 rows of 2048 values: 206 MB of weights, and next to nothing besides."""
    x, w = normal((1, 2048), F16, 1).cuda(), (torch.randn((50257, 2048), device="cuda") / 45).to(F16)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = ops.MoeLinear(x, w)
    assert torch.cuda.max_memory_allocated() - before < 16 << 20
    ref = x.double() @ w.double().t()
    tol = 2049 * U32 * (x.double().abs() @ w.double().abs().t())
    assert ((y.double() - ref).abs() <= tol + half_step(ref.abs() + tol, F16)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,H,act", [(1, 4097, 2048, "none"), (70, 41, 65, "swiglu"), (70, 41, 64, "swiglu"),
                                       (300, 130, 2049, "silu"), (130, 1001, 512, "none")])
@pytest.mark.parametrize("transposed", [False, True])
def test_calls_keep_within_the_layouts_workspace(ops, T, N, H, act, transposed):
    from test_dense_ops import grad_check, linear_check

    need = ops.linear_workspace_bytes(T, N, H, act, transposed)
    ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    linear_check(ops, T, N, H, F16, act, bias=True, transposed=transposed, workspace=ws[:need])
    assert (ws[need:] == 0x5a).all()
    need = ops.linear_grad_workspace_bytes(T, N, H, act, transposed)
    ws = torch.full((need + 256,), 0x5a, dtype=torch.uint8, device="cuda")
    grad_check(ops, T, N, H, F16, act, transposed=transposed, workspace=ws[:need])
    assert (ws[need:] == 0x5a).all()
