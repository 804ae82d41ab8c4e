"""The three operators as PyTorch custom ops (torch.library), for graph capture, torch.compile and framework use.

This fills the role of the reference's (empty) framework adapter, framework/CMakeLists.txt:1-9: the operators
registered under the reference's names, with its attributes, over the same C ABI as `ops`:

    torch.ops.moe_mi355x.MoeRoutingTopK(x, w_gate, topK=2) -> (expert_ids, weights)
    torch.ops.moe_mi355x.MoeExpertFFN(x, expert_ids, weights, expert_weights, intermediateSize=0) -> expert_out
    torch.ops.moe_mi355x.MoeCombine(expert_out, expert_ids, weights, topK=2) -> y

and the operators around the routed experts, with their gradients (MoeCombine has one too; MoeRoutingTopK and
MoeExpertFFN have none):

    torch.ops.moe_mi355x.MoeRoutingGroupTopK(logits, bias, topK, ...) -> (expert_ids, weights)
    torch.ops.moe_mi355x.MoeLinear(x, weight, bias, residual, activation, outDtype, returnPre) -> (y, pre)
    torch.ops.moe_mi355x.MoeRoutingGroupTopKGrad, MoeLinearGrad, MoeCombineGrad: what their backward calls

The device implementation is registered for GPU tensors only: a CPU tensor finds no kernel (there is no CPU
fallback). The fake (meta) implementations state the InferShape / InferDataType rules of
op_host/moe_ops.cpp:181-226, 364-398, 495-525 so that tracers can propagate shapes without running anything;
argument errors that need the data (ids out of range and the like) are the device implementation's.
Importing this module registers the ops once per process.
"""
from __future__ import annotations

import torch

from . import ops

NAMESPACE = "moe_mi355x"


def _routing_shape(x, w_gate, topK):
    if x.dim() != 2 or w_gate.dim() != 2:
        raise RuntimeError("MoeRoutingTopK: x must be [T, H] and w_gate [H, E]")
    if x.shape[1] != w_gate.shape[0]:
        raise RuntimeError("MoeRoutingTopK: hiddenSize mismatch between x and w_gate")
    k = topK if topK > 0 else 2  # the attr default, op_host/moe_ops.cpp:201-204
    return (x.shape[0], k)


@torch.library.custom_op(f"{NAMESPACE}::MoeRoutingTopK", mutates_args=(), device_types="cuda")
def moe_routing_topk(x: torch.Tensor, w_gate: torch.Tensor, topK: int = 2) -> tuple[torch.Tensor, torch.Tensor]:
    ids, w = ops.MoeRoutingTopK(x, w_gate, topK)
    return ids, w


@moe_routing_topk.register_fake
def _(x, w_gate, topK=2):
    shape = _routing_shape(x, w_gate, topK)
    return x.new_empty(shape, dtype=torch.int32), x.new_empty(shape, dtype=torch.float16)


@torch.library.custom_op(f"{NAMESPACE}::MoeExpertFFN", mutates_args=(), device_types="cuda")
def moe_expert_ffn(x: torch.Tensor, expert_ids: torch.Tensor, weights: torch.Tensor, expert_weights: torch.Tensor,
                   intermediateSize: int = 0) -> torch.Tensor:
    return ops.MoeExpertFFN(x, expert_ids, weights, expert_weights, intermediateSize)


@moe_expert_ffn.register_fake
def _(x, expert_ids, weights, expert_weights, intermediateSize=0):
    if x.dim() != 2 or expert_ids.dim() != 2 or expert_weights.dim() != 3:
        raise RuntimeError("MoeExpertFFN: x [T, H], expert_ids [T, K], expert_weights [E, 3I, H] expected")
    return x.new_empty((x.shape[0], expert_ids.shape[1], x.shape[1]), dtype=torch.float16)


@torch.library.custom_op(f"{NAMESPACE}::MoeCombine", mutates_args=(), device_types="cuda")
def moe_combine(expert_out: torch.Tensor, expert_ids: torch.Tensor | None, weights: torch.Tensor,
                topK: int = 2) -> torch.Tensor:
    return ops.MoeCombine(expert_out, expert_ids, weights, topK)


@moe_combine.register_fake
def _(expert_out, expert_ids, weights, topK=2):
    if expert_out.dim() != 3:
        raise RuntimeError("MoeCombine: expert_out must be [T, K, H]")
    return expert_out.new_empty((expert_out.shape[0], expert_out.shape[2]), dtype=torch.float16)


def moe_layer(x: torch.Tensor, w_gate: torch.Tensor, expert_weights: torch.Tensor, topK: int = 2) -> torch.Tensor:
    """The reference's chain of the three operators (tests/test_moe.cpp:444-463) through the registered ops."""
    op = getattr(torch.ops, NAMESPACE)
    ids, w = op.MoeRoutingTopK(x, w_gate, topK)
    eo = op.MoeExpertFFN(x, ids, w, expert_weights, 0)
    return op.MoeCombine(eo, ids, w, topK)


# ---------------------------------------------------------------------------------------------------------------------
# operators around the routed experts
# ---------------------------------------------------------------------------------------------------------------------


@torch.library.custom_op(f"{NAMESPACE}::MoeCombineGrad", mutates_args=(), device_types="cuda")
def moe_combine_grad(grad_y: torch.Tensor, expert_out: torch.Tensor,
                     weights: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return ops.MoeCombineGrad(grad_y, expert_out, weights)


@moe_combine_grad.register_fake
def _(grad_y, expert_out, weights):
    return expert_out.new_empty(expert_out.shape), weights.new_empty(weights.shape)


def _combine_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[0], inputs[2])


def _combine_backward(ctx, grad_y):
    geo, gw = getattr(torch.ops, NAMESPACE).MoeCombineGrad(grad_y.contiguous(), *ctx.saved_tensors)
    return geo, None, gw, None


moe_combine.register_autograd(_combine_backward, setup_context=_combine_setup)


@torch.library.custom_op(f"{NAMESPACE}::MoeRoutingGroupTopK", mutates_args=(), device_types="cuda")
def moe_routing_group_topk(logits: torch.Tensor, bias: torch.Tensor | None = None, topK: int = 2, numGroups: int = 1,
                           topGroups: int = 1, groupTop: int = 1, scoring: str = "softmax", renormalize: bool = True,
                           scale: float = 1.0,
                           weightsDtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    return ops.MoeRoutingGroupTopK(logits, bias, topK, numGroups, topGroups, groupTop, scoring, renormalize, scale,
                                   weightsDtype)


@moe_routing_group_topk.register_fake
def _(logits, bias=None, topK=2, numGroups=1, topGroups=1, groupTop=1, scoring="softmax", renormalize=True, scale=1.0,
      weightsDtype=torch.float16):
    if logits.dim() != 2:
        raise RuntimeError("MoeRoutingGroupTopK: logits must be [T, E]")
    shape = (logits.shape[0], topK)
    return logits.new_empty(shape, dtype=torch.int32), logits.new_empty(shape, dtype=weightsDtype)


@torch.library.custom_op(f"{NAMESPACE}::MoeRoutingGroupTopKGrad", mutates_args=(), device_types="cuda")
def moe_routing_group_topk_grad(grad_weights: torch.Tensor, logits: torch.Tensor, expert_ids: torch.Tensor,
                                scoring: str = "softmax", renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    return ops.MoeRoutingGroupTopKGrad(grad_weights, logits, expert_ids, scoring, renormalize, scale)


@moe_routing_group_topk_grad.register_fake
def _(grad_weights, logits, expert_ids, scoring="softmax", renormalize=True, scale=1.0):
    return logits.new_empty(logits.shape)


def _route_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[0], output[0])
    ctx.attrs = inputs[6:9]
    ctx.set_materialize_grads(False)


def _route_backward(ctx, _, grad_weights):
    if grad_weights is None:
        return (None,) * 10
    logits, ids = ctx.saved_tensors
    op = getattr(torch.ops, NAMESPACE).MoeRoutingGroupTopKGrad
    return (op(grad_weights.contiguous(), logits, ids, *ctx.attrs),) + (None,) * 9


moe_routing_group_topk.register_autograd(_route_backward, setup_context=_route_setup)


@torch.library.custom_op(f"{NAMESPACE}::MoeLinear", mutates_args=(), device_types="cuda")
def moe_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               residual: torch.Tensor | None = None, activation: str = "none", outDtype: torch.dtype | None = None,
               returnPre: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (y, pre); pre is empty unless returnPre, which the gradient through an activation needs."""
    if returnPre:
        return ops.MoeLinear(x, weight, bias, residual, activation, outDtype, True)
    return ops.MoeLinear(x, weight, bias, residual, activation, outDtype), x.new_empty(0)


def _linear_shapes(x, weight, activation):
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1]:
        raise RuntimeError("MoeLinear: x must be [T, H] and weight [N, H]")
    n = weight.shape[0]
    return x.shape[0], n // 2 if activation == "swiglu" else n, n


@moe_linear.register_fake
def _(x, weight, bias=None, residual=None, activation="none", outDtype=None, returnPre=False):
    t, n, z = _linear_shapes(x, weight, activation)
    return x.new_empty((t, n), dtype=outDtype or x.dtype), x.new_empty((t, z) if returnPre else 0)


@torch.library.custom_op(f"{NAMESPACE}::MoeLinearGrad", mutates_args=(), device_types="cuda")
def moe_linear_grad(grad_y: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, pre: torch.Tensor | None = None,
                    activation: str = "none", gradX: bool = True, gradWeight: bool = True,
                    gradBias: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (grad_x, grad_weight, grad_bias), empty where not asked for."""
    got = ops.MoeLinearGrad(grad_y, x, weight, pre, activation, gradX, gradWeight, gradBias)
    return tuple(x.new_empty(0) if g is None else g for g in got)


@moe_linear_grad.register_fake
def _(grad_y, x, weight, pre=None, activation="none", gradX=True, gradWeight=True, gradBias=False):
    t, _, z = _linear_shapes(x, weight, activation)
    return (x.new_empty((t, x.shape[1]) if gradX else 0), x.new_empty((z, x.shape[1]) if gradWeight else 0),
            x.new_empty(z if gradBias else 0))


def _linear_setup(ctx, inputs, output):
    x, weight, bias, residual, activation = inputs[:5]
    ctx.activation, ctx.has = activation, (bias is not None, residual is not None)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, weight, output[1] if activation != "none" else None)


def _linear_backward(ctx, grad_y, grad_pre):
    if grad_pre is not None:
        raise RuntimeError("MoeLinear has no gradient through pre")
    x, weight, pre = ctx.saved_tensors
    if grad_y is None:
        return (None,) * 7
    need = [ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.has[0] and ctx.needs_input_grad[2]]
    got = [None, None, None]
    if any(need):
        if pre is not None and pre.numel() == 0 and x.shape[0] > 0:
            raise RuntimeError(f"MoeLinear: the gradient through {ctx.activation!r} needs returnPre=True")
        out = getattr(torch.ops, NAMESPACE).MoeLinearGrad(grad_y.contiguous(), x, weight, pre, ctx.activation, *need)
        got = [g if n else None for g, n in zip(out, need)]
    return got[0], got[1], got[2], grad_y if ctx.has[1] else None, None, None, None


moe_linear.register_autograd(_linear_backward, setup_context=_linear_setup)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, activation: str = "none",
           outDtype: torch.dtype | None = None) -> torch.Tensor:
    """y of MoeLinear; the sums before the activation are kept where a gradient will need them."""
    keep = activation != "none" and torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, weight, bias))
    return getattr(torch.ops, NAMESPACE).MoeLinear(x, weight, bias, residual, activation, outDtype, keep)[0]
