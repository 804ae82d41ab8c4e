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

and those of quantised and permuted expert layers, with the gradients of the norm and of sorting (8-bit results have
none):

    torch.ops.moe_mi355x.MoeAddRmsNorm(x, gamma, residual, eps) -> (y, v)
    torch.ops.moe_mi355x.MoeAddRmsNormQuant(x, gamma, residual, eps, returnNorm) -> (q, scale, y, v)
    torch.ops.moe_mi355x.MoeQuantize(x) -> (q, scale)
    torch.ops.moe_mi355x.MoePermute(x, expert_ids, numExperts, xScale) -> (rows, offsets, position, row_scale)
    torch.ops.moe_mi355x.MoeUnpermute(rows, position, weights) -> y
    torch.ops.moe_mi355x.MoeLinearInt8(x, xScale, weight, weightScale, offsets, bias, residual, activation,
                                    outDtype) -> y
    torch.ops.moe_mi355x.MoeAddRmsNormGrad, MoeUnpermuteGrad: what their backward calls

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


# ---------------------------------------------------------------------------------------------------------------------
# quantised and permuted expert layers; an output that a call does not have is empty
# ---------------------------------------------------------------------------------------------------------------------


def _or_empty(t: torch.Tensor | None, like: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    return like.new_empty(0, dtype=dtype) if t is None else t


def _norm_shape(x, gamma, residual):
    if x.dim() != 2 or gamma.shape != x.shape[1:] or (residual is not None and residual.shape != x.shape):
        raise RuntimeError("MoeAddRmsNorm: x and residual must be [T, H] and gamma [H]")
    return x.shape


@torch.library.custom_op(f"{NAMESPACE}::MoeAddRmsNorm", mutates_args=(), device_types="cuda")
def moe_add_rms_norm(x: torch.Tensor, gamma: torch.Tensor, residual: torch.Tensor | None = None,
                     eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (y, v = x + residual); v is empty without a residual."""
    y, v = ops.MoeAddRmsNorm(x, gamma, residual, eps)
    return y, _or_empty(v, x)


@moe_add_rms_norm.register_fake
def _(x, gamma, residual=None, eps=1e-6):
    shape = _norm_shape(x, gamma, residual)
    return x.new_empty(shape), x.new_empty(0 if residual is None else shape)


@torch.library.custom_op(f"{NAMESPACE}::MoeAddRmsNormGrad", mutates_args=(), device_types="cuda")
def moe_add_rms_norm_grad(grad_y: torch.Tensor, v: torch.Tensor, gamma: torch.Tensor,
                          grad_v: torch.Tensor | None = None, eps: float = 1e-6, gradX: bool = True,
                          gradGamma: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (grad_x, grad_gamma), empty where not asked for."""
    gx, gg = ops.MoeAddRmsNormGrad(grad_y, v, gamma, grad_v, eps, gradX, gradGamma)
    return _or_empty(gx, v), _or_empty(gg, gamma)


@moe_add_rms_norm_grad.register_fake
def _(grad_y, v, gamma, grad_v=None, eps=1e-6, gradX=True, gradGamma=True):
    return v.new_empty(v.shape if gradX else 0), gamma.new_empty(gamma.shape if gradGamma else 0)


def _norm_setup(ctx, inputs, output):
    x, gamma, residual, ctx.eps = inputs
    ctx.summed = residual is not None
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(output[1] if ctx.summed else x, gamma)


def _norm_backward(ctx, grad_y, grad_v):
    v, gamma = ctx.saved_tensors
    grad_v = grad_v if ctx.summed else None
    want = [ctx.needs_input_grad[0] or (ctx.summed and ctx.needs_input_grad[2]), ctx.needs_input_grad[1]]
    gx = gg = None
    if grad_y is None:
        gx = grad_v
    elif any(want):
        op = getattr(torch.ops, NAMESPACE).MoeAddRmsNormGrad
        got = op(grad_y.contiguous(), v, gamma, None if grad_v is None else grad_v.contiguous(), ctx.eps, *want)
        gx, gg = (g if w else None for g, w in zip(got, want))
    return gx, gg, gx if ctx.summed else None, None


moe_add_rms_norm.register_autograd(_norm_backward, setup_context=_norm_setup)


@torch.library.custom_op(f"{NAMESPACE}::MoeAddRmsNormQuant", mutates_args=(), device_types="cuda")
def moe_add_rms_norm_quant(
        x: torch.Tensor, gamma: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
        returnNorm: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    q, scale, y, v = ops.MoeAddRmsNormQuant(x, gamma, residual, eps, returnNorm)
    return q, scale, _or_empty(y, x), _or_empty(v, x)


@moe_add_rms_norm_quant.register_fake
def _(x, gamma, residual=None, eps=1e-6, returnNorm=False):
    shape = _norm_shape(x, gamma, residual)
    return (x.new_empty(shape, dtype=torch.int8), x.new_empty(shape[0], dtype=torch.float32),
            x.new_empty(shape if returnNorm else 0), x.new_empty(0 if residual is None else shape))


@torch.library.custom_op(f"{NAMESPACE}::MoeQuantize", mutates_args=(), device_types="cuda")
def moe_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return ops.MoeQuantize(x)


@moe_quantize.register_fake
def _(x):
    if x.dim() not in (2, 3):
        raise RuntimeError("MoeQuantize: x must be [R, H] or [E, N, H]")
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::MoePermute", mutates_args=(), device_types="cuda")
def moe_permute(x: torch.Tensor, expert_ids: torch.Tensor, numExperts: int, xScale: torch.Tensor | None = None
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    rows, offsets, position, row_scale = ops.MoePermute(x, expert_ids, numExperts, xScale)
    return rows, offsets, position, _or_empty(row_scale, x, torch.float32)


@moe_permute.register_fake
def _(x, expert_ids, numExperts, xScale=None):
    if x.dim() != 2 or expert_ids.dim() != 2 or expert_ids.shape[0] != x.shape[0]:
        raise RuntimeError("MoePermute: x must be [T, H] and expert_ids [T, K]")
    picks = expert_ids.shape[0] * expert_ids.shape[1]
    return (x.new_empty((picks, x.shape[1])), expert_ids.new_empty(numExperts + 1),
            expert_ids.new_empty(expert_ids.shape), x.new_empty(0 if xScale is None else picks, dtype=torch.float32))


def _permute_setup(ctx, inputs, output):
    ctx.set_materialize_grads(False)
    ctx.scaled = inputs[3] is not None
    ctx.save_for_backward(output[2])


def _permute_backward(ctx, grad_rows, grad_offsets, grad_position, grad_scale):
    back, (position,) = getattr(torch.ops, NAMESPACE).MoeUnpermute, ctx.saved_tensors
    grad_x = grad_xs = None
    if grad_rows is not None and ctx.needs_input_grad[0]:
        grad_x = back(grad_rows.contiguous(), position, None)
    if ctx.scaled and grad_scale is not None and ctx.needs_input_grad[3]:  # scales go the way of their rows
        grad_xs = back(grad_scale.contiguous()[:, None], position, None)[:, 0]
    return grad_x, None, None, grad_xs


moe_permute.register_autograd(_permute_backward, setup_context=_permute_setup)


@torch.library.custom_op(f"{NAMESPACE}::MoeUnpermute", mutates_args=(), device_types="cuda")
def moe_unpermute(rows: torch.Tensor, position: torch.Tensor, weights: torch.Tensor | None = None) -> torch.Tensor:
    """Any positions; it has a gradient where there are as many rows as picks (MoePermute's), whatever they name."""
    return ops.MoeUnpermute(rows, position, weights)


@moe_unpermute.register_fake
def _(rows, position, weights=None):
    if rows.dim() != 2 or position.dim() != 2 or (weights is not None and weights.shape != position.shape):
        raise RuntimeError("MoeUnpermute: rows must be [R, H], position and weights [T, K]")
    return rows.new_empty((position.shape[0], rows.shape[1]))


@torch.library.custom_op(f"{NAMESPACE}::MoeUnpermuteGrad", mutates_args=(), device_types="cuda")
def moe_unpermute_grad(grad_y: torch.Tensor, rows: torch.Tensor | None, position: torch.Tensor,
                       weights: torch.Tensor | None = None,
                       anyPosition: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (grad_rows, grad_weights), the latter empty without weights."""
    grad_rows, grad_w = ops.MoeUnpermuteGrad(grad_y, rows, position, weights, anyPosition=anyPosition)
    return grad_rows, _or_empty(grad_w, grad_y)


@moe_unpermute_grad.register_fake
def _(grad_y, rows, position, weights=None, anyPosition=False):
    return (grad_y.new_empty((position.shape[0] * position.shape[1], grad_y.shape[1])),
            grad_y.new_empty(0) if weights is None else weights.new_empty(weights.shape))


def _unpermute_setup(ctx, inputs, output):
    rows, position, weights = inputs
    ctx.picks = position.shape[0] * position.shape[1]
    ctx.save_for_backward(rows if weights is not None else None, position, weights)
    ctx.num_rows = rows.shape[0]


def _unpermute_backward(ctx, grad_y):
    rows, position, weights = ctx.saved_tensors
    if ctx.num_rows != ctx.picks:
        raise RuntimeError("MoeUnpermute has a gradient where rows are MoePermute's, one for each pick")
    op = getattr(torch.ops, NAMESPACE).MoeUnpermuteGrad
    grad_rows, grad_w = op(grad_y.contiguous(), rows, position, weights, True)  # the forward takes any positions
    return grad_rows, None, None if weights is None else grad_w


moe_unpermute.register_autograd(_unpermute_backward, setup_context=_unpermute_setup)


@torch.library.custom_op(f"{NAMESPACE}::MoeLinearInt8", mutates_args=(), device_types="cuda")
def moe_linear_int8(x: torch.Tensor, xScale: torch.Tensor, weight: torch.Tensor, weightScale: torch.Tensor,
                    offsets: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                    residual: torch.Tensor | None = None, activation: str = "none",
                    outDtype: torch.dtype = torch.float16) -> torch.Tensor:
    return ops.MoeLinearInt8(x, xScale, weight, weightScale, offsets, bias, residual, activation, outDtype)


@moe_linear_int8.register_fake
def _(x, xScale, weight, weightScale, offsets=None, bias=None, residual=None, activation="none",
      outDtype=torch.float16):
    dims = 2 if offsets is None else 3
    if x.dim() != 2 or weight.dim() != dims or x.shape[1] != weight.shape[-1]:
        raise RuntimeError("MoeLinearInt8: x must be [T, H] and weight [N, H], with offsets [E, N, H]")
    n = weight.shape[-2]
    return x.new_empty((x.shape[0], n // 2 if activation == "swiglu" else n), dtype=outDtype)
