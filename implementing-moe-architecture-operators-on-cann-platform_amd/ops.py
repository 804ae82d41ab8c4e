"""Python mirror of the reference's three operators over the C ABI, with torch tensors as device memory.

Reference operator interface: op_host/moe_ops.cpp:537-679 (OpDef inputs/outputs/attrs) and the kernel
entries op_kernel/moe_routing.cpp:434, op_kernel/moe_expert_ffn.cpp:613, op_kernel/moe_combine.cpp:136.
Shapes and dtypes are inferred by the library (the InferShape/InferDataType replacements), and the launch is
queued on `stream` (torch's current stream when None). Outputs and any workspace the call allocates are
allocated while that stream is current, so torch's caching allocator ties them to the stream the kernels run
on: a workspace freed on return cannot be handed to other work before those kernels have finished with it.
Errors raise MoeError with the library's message, before anything is launched.

A call's own host work is kept to a few microseconds: at decode sizes the kernels of an operator take 5-10 us, and
asking the library for every shape and entering a stream context took longer than that (T = 8, H = 64, E = 4,
I = 256, the three operators: 60 us of host time, now 25, of which the four launches take ~13). Shapes that fit are
worked out here, any other goes to the library's infer function, which words the error; the stream context is entered
only for a stream that the caller names.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import _lib
from ._lib import MoeError, check, dims

# The current stream without the Stream object that torch.cuda.current_stream() makes on each call, and the allocation
# on the current device that torch's compiled code uses (0.75 us a tensor, new_empty 1.5): private to torch, so a torch
# without them takes the public functions. The allocation passes torch's dispatch modes and its filling of new memory
# under deterministic algorithms by, so it is used where neither is on.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_device = getattr(torch._C, "_cuda_getDevice", None)
_empty_strided = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
_modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
_deterministic = getattr(torch._C, "_get_deterministic_algorithms", None)
if _modes is None or _deterministic is None:
    _empty_strided = None

_TORCH_DT = {_lib.DT_FLOAT16: torch.float16, _lib.DT_INT32: torch.int32}
_FLOAT_DT = {torch.float32: _lib.DT_FLOAT32, torch.float16: _lib.DT_FLOAT16, torch.bfloat16: _lib.DT_BFLOAT16}
_ROW_DT = {**_FLOAT_DT, torch.int8: _lib.DT_INT8, torch.int32: _lib.DT_INT32}
_SCORING = {"softmax": 0, "sigmoid": 1}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "swiglu": 5}


def _stream_ptr(stream) -> int:
    """The raw stream a call runs on: `stream`, or the current stream of the current device."""
    if stream is not None:
        return int(stream.cuda_stream)
    if _raw_stream is not None and _device is not None:
        return _raw_stream(_device())
    return int(torch.cuda.current_stream().cuda_stream)


_CURRENT = contextlib.nullcontext()


def _on(stream):
    """Allocations made within belong to the stream the kernels run on."""
    return _CURRENT if stream is None else torch.cuda.stream(stream)


def _like(t: torch.Tensor) -> torch.Tensor:
    """What outputs are allocated from: `t` without its class (new_empty of a tensor subclass gives the subclass)."""
    return t if type(t) is torch.Tensor or type(t) is torch.nn.Parameter else t.as_subclass(torch.Tensor)


def _need(t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype and t.is_contiguous():
        return
    if not isinstance(t, torch.Tensor):
        raise MoeError(1, f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise MoeError(4, f"{name} must be a device tensor (got {t.device})")
    if t.dtype != dtype:
        raise MoeError(4, f"{name} must be {dtype} (got {t.dtype})")
    raise MoeError(4, f"{name} must be contiguous (ND format)")


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def infer_routing(x_shape, w_gate_shape, topK: int = 2):
    lib = _lib.load()
    ids, w = dims([0, 0]), dims([0, 0])
    check(lib.moe_routing_topk_infer_shape(dims(x_shape), len(x_shape), dims(w_gate_shape), len(w_gate_shape),
                                           topK, ids, w))
    t_ids, t_w = C.c_int32(), C.c_int32()
    check(lib.moe_routing_topk_infer_dtype(C.byref(t_ids), C.byref(t_w)))
    return (tuple(ids), _TORCH_DT[t_ids.value]), (tuple(w), _TORCH_DT[t_w.value])


def infer_expert_ffn(x_shape, ids_shape, ew_shape, intermediateSize: int = 0):
    lib = _lib.load()
    out, inter = dims([0, 0, 0]), C.c_int64()
    check(lib.moe_expert_ffn_infer_shape(dims(x_shape), len(x_shape), dims(ids_shape), len(ids_shape),
                                         dims(ew_shape), len(ew_shape), intermediateSize, out, C.byref(inter)))
    dt = C.c_int32()
    check(lib.moe_expert_ffn_infer_dtype(C.byref(dt)))
    return tuple(out), _TORCH_DT[dt.value], inter.value


def infer_combine(eo_shape, ids_shape=None):
    lib = _lib.load()
    y = dims([0, 0])
    ids_arr = dims(ids_shape) if ids_shape is not None else None
    check(lib.moe_combine_infer_shape(dims(eo_shape), len(eo_shape), ids_arr,
                                      len(ids_shape) if ids_shape is not None else 0, y))
    dt = C.c_int32()
    check(lib.moe_combine_infer_dtype(C.byref(dt)))
    return tuple(y), _TORCH_DT[dt.value]


def workspace_bytes(T: int, H: int, E: int, K: int, I: int) -> int:
    return int(_lib.load().moe_expert_ffn_workspace_bytes(T, H, E, K, I))


def layer_workspace_bytes(T: int, H: int, E: int, K: int, I: int) -> int:
    return int(_lib.load().moe_layer_workspace_bytes(T, H, E, K, I))


def _routing_shape(x, w_gate, topK):
    """[T, K] of the routing outputs (the rules of moe_routing_topk_infer_shape)."""
    xs, gs = x.shape, w_gate.shape
    if len(xs) == 2 and len(gs) == 2 and xs[1] == gs[0] and type(topK) is int:
        k = topK if topK > 0 else 2
        if k <= gs[1]:
            return xs[0], k
    return infer_routing(tuple(xs), tuple(gs), topK)[0][0]


def _ffn_inter(x, ids_shape, expert_weights, intermediateSize) -> int:
    """The intermediate size of the expert FFN (the rules of moe_expert_ffn_infer_shape)."""
    xs, es = x.shape, expert_weights.shape
    if (len(xs) == 2 and len(ids_shape) == 2 and len(es) == 3 and ids_shape[0] == xs[0] and es[2] == xs[1]
            and es[1] % 3 == 0 and type(intermediateSize) is int):
        inter = es[1] // 3
        if intermediateSize <= 0 or intermediateSize == inter:
            return inter
    return infer_expert_ffn(tuple(xs), tuple(ids_shape), tuple(es), intermediateSize)[2]


def _bytes(workspace: torch.Tensor) -> int:
    return workspace.numel() * workspace.element_size()


def MoeRoutingTopK(x: torch.Tensor, w_gate: torch.Tensor, topK: int = 2, stream=None):
    """x[T,H] fp16, w_gate[H,E] fp16 -> (expert_ids[T,K] int32, weights[T,K] fp16)."""
    _need(x, "x", torch.float16)
    _need(w_gate, "w_gate", torch.float16)
    T, K = shape = _routing_shape(x, w_gate, topK)
    H, E = w_gate.shape
    like = _like(x)
    with _on(stream):
        ids = like.new_empty(shape, dtype=torch.int32)
        w = like.new_empty(shape)
    check(_lib.load().moe_routing_topk(x.data_ptr(), w_gate.data_ptr(), ids.data_ptr(), w.data_ptr(), T, H, E, K,
                                       _stream_ptr(stream)))
    return ids, w


def MoeExpertFFN(x: torch.Tensor, expert_ids: torch.Tensor, weights: torch.Tensor, expert_weights: torch.Tensor,
                 intermediateSize: int = 0, workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """-> expert_out[T,K,H] fp16. `workspace` (uint8, >= workspace_bytes) is allocated when not given."""
    _need(x, "x", torch.float16)
    _need(expert_ids, "expert_ids", torch.int32)
    _need(weights, "weights", torch.float16)
    _need(expert_weights, "expert_weights", torch.float16)
    inter = _ffn_inter(x, expert_ids.shape, expert_weights, intermediateSize)
    T, H = x.shape
    E, K = expert_weights.shape[0], expert_ids.shape[1]
    lib = _lib.load()
    like = _like(x)
    with _on(stream):
        if workspace is None:
            need = int(lib.moe_expert_ffn_workspace_bytes(T, H, E, K, inter))
            workspace = like.new_empty(max(need, 1), dtype=torch.uint8)
        expert_out = like.new_empty((T, K, H))
    check(lib.moe_expert_ffn(x.data_ptr(), expert_ids.data_ptr(), weights.data_ptr(), expert_weights.data_ptr(),
                             expert_out.data_ptr(), workspace.data_ptr(), _bytes(workspace), T, H, E, K, inter,
                             _stream_ptr(stream)))
    return expert_out


def MoeCombine(expert_out: torch.Tensor, expert_ids: torch.Tensor | None, weights: torch.Tensor, topK: int = 2,
               stream=None) -> torch.Tensor:
    """expert_out[T,K,H] fp16, weights[T,K] fp16 -> y[T,H] fp16. K comes from expert_out (the attr is kept
    for signature parity, as in the reference's TilingFunc, op_host/moe_ops.cpp:432)."""
    del topK
    _need(expert_out, "expert_out", torch.float16)
    _need(weights, "weights", torch.float16)
    if expert_ids is not None:
        _need(expert_ids, "expert_ids", torch.int32)
    es = expert_out.shape
    if len(es) != 3 or (expert_ids is not None and expert_ids.shape != es[:2]):
        infer_combine(tuple(es), tuple(expert_ids.shape) if expert_ids is not None else None)  # raises
    T, K, H = es
    if weights.shape != es[:2]:
        raise MoeError(3, f"weights shape {tuple(weights.shape)} != {(T, K)}")
    like = _like(expert_out)
    with _on(stream):
        y = like.new_empty((T, H))
    check(_lib.load().moe_combine(expert_out.data_ptr(), _ptr(expert_ids), weights.data_ptr(), y.data_ptr(), T, H, K,
                                  _stream_ptr(stream)))
    return y


def MoeExpertFFNCombine(x: torch.Tensor, expert_ids: torch.Tensor, weights: torch.Tensor,
                        expert_weights: torch.Tensor, intermediateSize: int = 0,
                        workspace: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """MoeExpertFFN then MoeCombine in one call (moe_expert_ffn_combine): -> (expert_out[T,K,H], y[T,H]), both
    fp16, expert_out as MoeExpertFFN returns it and y bit-identical to MoeCombine(expert_out, ...)."""
    _need(x, "x", torch.float16)
    _need(expert_ids, "expert_ids", torch.int32)
    _need(weights, "weights", torch.float16)
    _need(expert_weights, "expert_weights", torch.float16)
    inter = _ffn_inter(x, expert_ids.shape, expert_weights, intermediateSize)
    T, H = x.shape
    E, K = expert_weights.shape[0], expert_ids.shape[1]
    if weights.shape != expert_ids.shape:
        raise MoeError(3, f"weights shape {tuple(weights.shape)} != {(T, K)}")
    lib = _lib.load()
    like = _like(x)
    with _on(stream):
        if workspace is None:
            need = int(lib.moe_expert_ffn_workspace_bytes(T, H, E, K, inter))
            workspace = like.new_empty(max(need, 1), dtype=torch.uint8)
        expert_out = like.new_empty((T, K, H))
        y = like.new_empty((T, H))
    check(lib.moe_expert_ffn_combine(x.data_ptr(), expert_ids.data_ptr(), weights.data_ptr(),
                                     expert_weights.data_ptr(), expert_out.data_ptr(), y.data_ptr(),
                                     workspace.data_ptr(), _bytes(workspace), T, H, E, K, inter,
                                     _stream_ptr(stream)))
    return expert_out, y


def moe_layer(x: torch.Tensor, w_gate: torch.Tensor, expert_weights: torch.Tensor, topK: int = 2,
              workspace: torch.Tensor | None = None, stream=None):
    """The three operators chained as the reference harness chains them (tests/test_moe.cpp:444-463).
    Returns (y, expert_ids, weights, expert_out)."""
    ids, w = MoeRoutingTopK(x, w_gate, topK, stream=stream)
    eo = MoeExpertFFN(x, ids, w, expert_weights, 0, workspace, stream=stream)
    y = MoeCombine(eo, ids, w, topK, stream=stream)
    return y, ids, w, eo


def moe_layer_fused(x: torch.Tensor, w_gate: torch.Tensor, expert_weights: torch.Tensor, topK: int = 2,
                    intermediateSize: int = 0, workspace: torch.Tensor | None = None, stream=None):
    """The whole layer in one library call (moe_layer): the routing kernel also ranks the slots for the FFN's
    permute. Returns (y, expert_ids, weights, expert_out), bit-identical to moe_layer's."""
    _need(x, "x", torch.float16)
    _need(w_gate, "w_gate", torch.float16)
    _need(expert_weights, "expert_weights", torch.float16)
    T, K = shape = _routing_shape(x, w_gate, topK)
    inter = _ffn_inter(x, shape, expert_weights, intermediateSize)
    H, E = w_gate.shape
    if expert_weights.shape[0] != E:  # the library takes one E: it would read w_gate past its end or at another stride
        raise MoeError(3, f"w_gate routes to {E} experts, expert_weights holds {expert_weights.shape[0]}")
    lib = _lib.load()
    like = _like(x)
    with _on(stream):
        if workspace is None:
            need = int(lib.moe_layer_workspace_bytes(T, H, E, K, inter))
            workspace = like.new_empty(max(need, 1), dtype=torch.uint8)
        ids = like.new_empty(shape, dtype=torch.int32)
        w = like.new_empty(shape)
        expert_out = like.new_empty((T, K, H))
        y = like.new_empty((T, H))
    check(lib.moe_layer(x.data_ptr(), w_gate.data_ptr(), expert_weights.data_ptr(), ids.data_ptr(), w.data_ptr(),
                        expert_out.data_ptr(), y.data_ptr(), workspace.data_ptr(), _bytes(workspace), T, H, E, K,
                        inter, _stream_ptr(stream)))
    return y, ids, w, expert_out


# ---------------------------------------------------------------------------------------------------------------------
# operators around the routed experts (no counterpart in the reference)
# ---------------------------------------------------------------------------------------------------------------------


_F16_32 = (torch.float16, torch.float32)
_HALVES = (torch.float16, torch.bfloat16)
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_INT8 = (torch.int8,)


def _here() -> int:
    """The current device, on whose stream a call is queued: its tensors have to be there."""
    return torch.cuda.current_device() if _device is None else _device()


def _first_float(t, name: str, dtypes, dims: int) -> tuple[int, int]:
    """Checks a call's first tensor; returns its moe_dtype and the device that all the others have to be on."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.dim() == dims:
        dev = t.get_device()
        if dev == _here():
            return _ROW_DT[t.dtype], dev
        raise MoeError(4, f"{name} is on cuda:{dev}, the current device is cuda:{_here()}")
    return _need_float(t, name, dtypes, dims, -1), -1  # raises


def _need_float(t, name: str, dtypes, dims: int, dev: int) -> int:
    """Checks a floating tensor of any strides on device `dev`; returns its moe_dtype."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.dim() == dims and t.get_device() == dev:
        return _ROW_DT[t.dtype]
    if not isinstance(t, torch.Tensor):
        raise MoeError(1, f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise MoeError(4, f"{name} must be a device tensor (got {t.device})")
    if t.dtype not in dtypes:
        raise MoeError(4, f"{name} must be {' or '.join(str(d) for d in dtypes)} (got {t.dtype})")
    if t.dim() != dims:
        raise MoeError(2, f"{name} must have {dims} dimensions (got {t.dim()})")
    raise MoeError(4, f"{name} is on {t.device}, the first tensor on cuda:{dev}")


def _row_stride(t: torch.Tensor, name: str) -> int:
    """Elements between the rows of a 2-D tensor whose rows are contiguous."""
    st, one = t.stride()
    if one != 1 and t.shape[1] > 1:
        raise MoeError(4, f"{name}: the elements of a row must be contiguous (strides {t.stride()})")
    return st if t.shape[0] > 1 else max(st, t.shape[1])


def _weight_layout(t: torch.Tensor) -> tuple[int, int]:
    """(stride, transposed) of a 2-D weight that is contiguous along one of its dimensions."""
    (n, h), (sn, sh) = t.shape, t.stride()
    if sh == 1 or h == 1:
        return (sn if n > 1 else max(sn, h)), 0
    if sn == 1 or n == 1:
        return (sh if h > 1 else max(sh, n)), 1
    raise MoeError(4, f"weight must be contiguous along one dimension (strides {t.stride()})")


def _need_shape(t: torch.Tensor, name: str, shape) -> None:
    if t.shape != shape:
        raise MoeError(3, f"{name} shape {tuple(t.shape)} != {tuple(shape)}")


def _act_code(activation: str) -> int:
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise MoeError(4, f"activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    return code


def _empty(like: torch.Tensor, stream, shape: tuple, dtype: torch.dtype) -> torch.Tensor:
    """A new contiguous tensor that belongs to the stream the kernels run on."""
    if stream is None:
        if _empty_strided is None or _modes() or _deterministic():
            return like.new_empty(shape, dtype=dtype)
        dims = len(shape)
        if dims == 2:
            return _empty_strided(shape, (shape[1], 1), dtype)
        return _empty_strided(shape, (1,) if dims == 1 else (shape[1] * shape[2], shape[2], 1), dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _queue(stream, dev: int) -> int:
    """The raw stream a call on device `dev`, the current one, runs on."""
    if stream is None and _raw_stream is not None:
        return _raw_stream(dev)
    return _stream_ptr(stream)


def _scoring_code(scoring: str) -> int:
    code = _SCORING.get(scoring)
    if code is None:
        raise MoeError(4, f"scoring {scoring!r}: one of {', '.join(_SCORING)}")
    return code


def _workspace(workspace, query, args, like, dev, stream):
    """(address, bytes) of the caller's workspace or of a new one (which the caller keeps until the launch)."""
    if workspace is None:
        need = int(query(*args))
        if need == 0:
            return None, None, 0
        workspace = _empty(like, stream, (need,), torch.uint8)
        return workspace, workspace.data_ptr(), need
    if not isinstance(workspace, torch.Tensor) or workspace.get_device() != dev or not workspace.is_contiguous():
        raise MoeError(4, f"workspace must be a contiguous tensor on cuda:{dev}")
    return workspace, workspace.data_ptr(), _bytes(workspace)


def _vector(t, name: str, dtype, n: int, dev: int) -> int | None:
    """The address of an optional contiguous vector."""
    if t is None:
        return None
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == (n,) and t.is_contiguous()
            and t.get_device() == dev):
        _need_float(t, name, (dtype,), 1, dev)
        _need_shape(t, name, (n,))
        raise MoeError(4, f"{name} must be contiguous")
    return t.data_ptr()


def _matrix(t, name: str, dtype, shape, dev: int) -> int | None:
    """The address of an optional contiguous matrix."""
    if t is None:
        return None
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.is_contiguous()
            and t.get_device() == dev):
        _need_float(t, name, (dtype,), 2, dev)
        _need_shape(t, name, shape)
        raise MoeError(4, f"{name} must be contiguous (ND format)")
    return t.data_ptr()


def MoeRoutingGroupTopK(logits: torch.Tensor, bias: torch.Tensor | None = None, topK: int = 2, numGroups: int = 1,
                        topGroups: int = 1, groupTop: int = 1, scoring: str = "softmax", renormalize: bool = True,
                        scale: float = 1.0, weightsDtype: torch.dtype = torch.float16, stream=None):
    """logits[T,E] (fp32, fp16 or bf16), bias[E] fp32 -> (expert_ids[T,K] int32, weights[T,K] fp16 or fp32).

    Scores are the softmax or the sigmoid of the logits. Experts are chosen by score + bias: of numGroups groups of
    consecutive experts the topGroups best stay, a group's score being its best expert's (groupTop=1) or the sum of its
    two best (2); of the experts that stay the topK best are chosen, equal ones by lowest index. The weights are the
    chosen scores, without bias, over their sum (renormalize) and times scale. Experts whose logit is -inf or NaN
    are not available; picks a row has no expert left for are id -1, weight 0."""
    lt, dev = _first_float(logits, "logits", _FLOATS, 2)
    T, E = logits.shape
    bp = _vector(bias, "bias", torch.float32, E, dev)
    if weightsDtype not in _F16_32:
        raise MoeError(4, f"weightsDtype must be float16 or float32 (got {weightsDtype})")
    ld = _row_stride(logits, "logits")
    if type(topK) is not int or topK < 1 or topK > E:
        raise MoeError(4, f"topK={topK} must be in [1, numExperts={E}]")
    like = _like(logits)
    ids = _empty(like, stream, (T, topK), torch.int32)
    w = _empty(like, stream, (T, topK), weightsDtype)
    check(_lib.load().moe_routing_group_topk(logits.data_ptr(), ld, lt, bp, ids.data_ptr(), w.data_ptr(),
                                             _FLOAT_DT[weightsDtype], T, E, topK, numGroups, topGroups, groupTop,
                                             _scoring_code(scoring), int(renormalize), scale, _queue(stream, dev)))
    return ids, w


def MoeRoutingGroupTopKGrad(grad_weights: torch.Tensor, logits: torch.Tensor, expert_ids: torch.Tensor,
                            scoring: str = "softmax", renormalize: bool = True, scale: float = 1.0,
                            stream=None) -> torch.Tensor:
    """The gradient of MoeRoutingGroupTopK's weights -> the logits', [T,E] contiguous, of the logits' type.
    expert_ids are the forward's; the choice itself (and with it the bias) has no gradient."""
    lt, dev = _first_float(logits, "logits", _FLOATS, 2)
    T, E = logits.shape
    gt = _need_float(grad_weights, "grad_weights", _FLOATS, 2, dev)
    _need(expert_ids, "expert_ids", torch.int32)
    if expert_ids.get_device() != dev:
        raise MoeError(4, f"expert_ids is on {expert_ids.device}, logits on {logits.device}")
    ks = expert_ids.shape
    if len(ks) != 2 or ks[0] != T:
        raise MoeError(3, f"expert_ids shape {tuple(ks)} for {T} rows of logits")
    _need_shape(grad_weights, "grad_weights", ks)
    if not grad_weights.is_contiguous():
        raise MoeError(4, "grad_weights must be contiguous (ND format)")
    ld = _row_stride(logits, "logits")
    grad = _empty(_like(logits), stream, (T, E), logits.dtype)
    check(_lib.load().moe_routing_group_topk_grad(grad_weights.data_ptr(), gt, logits.data_ptr(), ld, lt,
                                                  expert_ids.data_ptr(), grad.data_ptr(), T, E, ks[1],
                                                  _scoring_code(scoring), int(renormalize), scale, _queue(stream, dev)))
    return grad


def MoeCombineGrad(grad_y: torch.Tensor, expert_out: torch.Tensor, weights: torch.Tensor, stream=None):
    """grad_y[T,H], expert_out[T,K,H], weights[T,K] fp16 -> (grad_expert_out[T,K,H], grad_weights[T,K]) fp16."""
    _need(grad_y, "grad_y", torch.float16)
    _need(expert_out, "expert_out", torch.float16)
    _need(weights, "weights", torch.float16)
    es = expert_out.shape
    if len(es) != 3:
        raise MoeError(2, f"expert_out must have 3 dimensions (got {len(es)})")
    T, K, H = es
    _need_shape(grad_y, "grad_y", (T, H))
    _need_shape(weights, "weights", (T, K))
    dev = _here()
    if expert_out.get_device() != dev or grad_y.get_device() != dev or weights.get_device() != dev:
        raise MoeError(4, f"grad_y, expert_out and weights must be on the current device cuda:{dev}")
    like = _like(expert_out)
    geo = _empty(like, stream, (T, K, H), torch.float16)
    gw = _empty(like, stream, (T, K), torch.float16)
    check(_lib.load().moe_combine_grad(grad_y.data_ptr(), expert_out.data_ptr(), weights.data_ptr(), geo.data_ptr(),
                                       gw.data_ptr(), T, H, K, _queue(stream, dev)))
    return geo, gw


def linear_workspace_bytes(T: int, N: int, H: int, activation: str = "none", transposed: bool | None = None) -> int:
    """Workspace of MoeLinear: of a weight whose rows are contiguous (transposed False), of one stored [H, N] (True), or
    of either (None)."""
    lib, act = _lib.load(), _act_code(activation)
    if transposed is None:
        return int(lib.moe_linear_workspace_bytes(T, N, H, act))
    return int(lib.moe_linear_layout_workspace_bytes(T, N, H, act, int(transposed)))


def linear_grad_workspace_bytes(T: int, N: int, H: int, activation: str = "none",
                                transposed: bool | None = None) -> int:
    """Workspace of MoeLinearGrad, as linear_workspace_bytes, for a grad_y of either type."""
    query, act = _lib.load().moe_linear_grad_f32_workspace_bytes, _act_code(activation)
    return max(int(query(T, N, H, act, int(t))) for t in ((False, True) if transposed is None else (transposed,)))


def _linear_sizes(x, weight, act: int):
    T, H = x.shape
    Z = weight.shape[0]
    if weight.shape[1] != H:
        raise MoeError(3, f"hidden size mismatch x[{H}] vs weight[{weight.shape[1]}]")
    if act == ACTIVATIONS["swiglu"] and Z % 2:
        raise MoeError(3, f"weight rows ({Z}) of a swiglu must be N gate and N up rows")
    return T, H, Z // 2 if act == ACTIVATIONS["swiglu"] else Z, Z


def MoeLinear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
              residual: torch.Tensor | None = None, activation: str = "none", outDtype: torch.dtype | None = None,
              returnPre: bool = False, workspace: torch.Tensor | None = None, stream=None):
    """act(x[T,H] @ weight[N,H]^T + bias[N]) + residual[T,N] -> y[T,N] of outDtype (x's type, or fp32).

    x and weight are fp16 or bf16; x's rows and weight along one of its dimensions must be contiguous (w_gate.t() is a
    weight). activation: none, relu, gelu, gelu_tanh, silu or swiglu, which takes weight[2N,H] (and bias[2N]), the N
    gate rows first. residual has y's type. With returnPre -> (y, pre): the sums before the activation, which
    MoeLinearGrad takes. `workspace` (uint8, >= linear_workspace_bytes) is allocated when not given."""
    act = _act_code(activation)
    dt, dev = _first_float(x, "x", _HALVES, 2)
    dtype = x.dtype
    _need_float(weight, "weight", (dtype,), 2, dev)
    T, H, N, Z = _linear_sizes(x, weight, act)
    out = dtype if outDtype is None else outDtype
    if out is not dtype and out is not torch.float32:
        raise MoeError(4, f"outDtype must be {dtype} or float32 (got {out})")
    ldx = _row_stride(x, "x")
    ldw, transposed = _weight_layout(weight)
    bp = _vector(bias, "bias", dtype, Z, dev)
    rp = _matrix(residual, "residual", out, (T, N), dev)
    lib = _lib.load()
    like = _like(x)
    workspace, wp, wb = _workspace(workspace, lib.moe_linear_layout_workspace_bytes, (T, N, H, act, transposed), like,
                                   dev, stream)
    y = _empty(like, stream, (T, N), out)
    pre = _empty(like, stream, (T, Z), dtype) if returnPre else None
    check(lib.moe_linear_layout(x.data_ptr(), ldx, weight.data_ptr(), ldw, transposed, bp, rp, y.data_ptr(), _ptr(pre),
                                wp, wb, T, N, H, act, dt, _FLOAT_DT[out], _queue(stream, dev)))
    return (y, pre) if returnPre else y


def MoeLinearGrad(grad_y: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, pre: torch.Tensor | None = None,
                  activation: str = "none", gradX: bool = True, gradWeight: bool = True, gradBias: bool = False,
                  workspace: torch.Tensor | None = None, stream=None):
    """The gradient of MoeLinear's y[T,N] (of x's type or, for an fp32 y, fp32) -> (grad_x[T,H], grad_weight[N,H],
    grad_bias[N]), contiguous, of x's type, None where not asked for. pre is MoeLinear's (needed with an activation).
    The residual's gradient is grad_y. `workspace` (uint8, >= linear_grad_workspace_bytes) is allocated when not given."""
    act = _act_code(activation)
    dt, dev = _first_float(x, "x", _HALVES, 2)
    dtype = x.dtype
    _need_float(weight, "weight", (dtype,), 2, dev)
    wide = _need_float(grad_y, "grad_y", (dtype, torch.float32), 2, dev) == _lib.DT_FLOAT32
    T, H, N, Z = _linear_sizes(x, weight, act)
    _need_shape(grad_y, "grad_y", (T, N))
    ldx, ldy = _row_stride(x, "x"), _row_stride(grad_y, "grad_y")
    ldw, transposed = _weight_layout(weight)
    if act and pre is None:
        raise MoeError(1, f"MoeLinearGrad needs pre with activation {activation!r}")
    pp = _matrix(pre, "pre", dtype, (T, Z), dev) if act else None
    lib = _lib.load()
    like = _like(x)
    query, call = ((lib.moe_linear_grad_f32_workspace_bytes, lib.moe_linear_grad_f32) if wide else
                   (lib.moe_linear_grad_layout_workspace_bytes, lib.moe_linear_grad_layout))
    workspace, wp, wb = _workspace(workspace, query, (T, N, H, act, transposed), like, dev, stream)
    gx = _empty(like, stream, (T, H), dtype) if gradX else None
    gw = _empty(like, stream, (Z, H), dtype) if gradWeight else None
    gb = _empty(like, stream, (Z,), dtype) if gradBias else None
    check(call(grad_y.data_ptr(), ldy, x.data_ptr(), ldx, weight.data_ptr(), ldw, transposed, pp, _ptr(gx), _ptr(gw),
               _ptr(gb), wp, wb, T, N, H, act, dt, _queue(stream, dev)))
    return gx, gw, gb


def moe_layer_shared(x: torch.Tensor, w_gate: torch.Tensor, expert_weights: torch.Tensor,
                     shared_gate_up: torch.Tensor | None = None, shared_down: torch.Tensor | None = None,
                     topK: int = 2, bias: torch.Tensor | None = None, numGroups: int = 1, topGroups: int = 1,
                     groupTop: int = 1, scoring: str = "softmax", renormalize: bool = True, scale: float = 1.0,
                     stream=None):
    """A layer with scored and grouped routing and a dense expert that every token passes: fp32 logits x @ w_gate[H,E]
    (MoeLinear), MoeRoutingGroupTopK, the routed experts (MoeExpertFFNCombine), and, where its weights are given, the
    dense expert's shared_gate_up[2S,H] (SwiGLU) and shared_down[H,S], whose epilogue adds the routed result.
    Returns (y, expert_ids, weights, expert_out)."""
    if (shared_gate_up is None) != (shared_down is None):
        raise MoeError(1, "shared_gate_up and shared_down are given together")
    if w_gate.dim() == 2 and expert_weights.dim() == 3 and expert_weights.shape[0] != w_gate.shape[1]:
        raise MoeError(3, f"w_gate routes to {w_gate.shape[1]} experts, expert_weights holds {expert_weights.shape[0]}")
    logits = MoeLinear(x, w_gate.t(), outDtype=torch.float32, stream=stream)
    ids, w = MoeRoutingGroupTopK(logits, bias, topK, numGroups, topGroups, groupTop, scoring, renormalize, scale,
                                 stream=stream)
    eo, y = MoeExpertFFNCombine(x, ids, w, expert_weights, stream=stream)
    if shared_gate_up is not None:
        hidden = MoeLinear(x, shared_gate_up, activation="swiglu", stream=stream)
        y = MoeLinear(hidden, shared_down, residual=y, stream=stream)
    return y, ids, w, eo


# ---------------------------------------------------------------------------------------------------------------------
# quantised and permuted expert layers (no counterpart in the reference)
# ---------------------------------------------------------------------------------------------------------------------


def _new(shape: tuple, dtype: torch.dtype) -> torch.Tensor:
    """A new contiguous tensor of one or two dimensions on the current device, where _empty may use private functions."""
    return _empty_strided(shape, (shape[1], 1) if len(shape) == 2 else (1,), dtype)


def _allocator(like: torch.Tensor, stream):
    """_empty for several results of a call, which looks at torch's modes once: (shape, dtype) -> tensor."""
    if stream is None and _empty_strided is not None and not _modes() and not _deterministic():
        return _new
    return lambda shape, dtype: _empty(like, stream, shape, dtype)


def _gamma(gamma, dtype, H: int, dev: int) -> int:
    """Checks a norm's gamma, of the rows' type or fp32; returns its moe_dtype."""
    gt = getattr(gamma, "dtype", None)
    if gt is not dtype and gt is not torch.float32:
        _need_float(gamma, "gamma", (dtype, torch.float32), 1, dev)  # raises
    _vector(gamma, "gamma", gt, H, dev)
    return _FLOAT_DT[gt]


def _rows_like(t, name: str, dtype, shape, dev: int) -> tuple[int | None, int]:
    """(address, row stride) of an optional matrix of any row stride."""
    if t is None:
        return None, 0
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == dev):
        _need_float(t, name, (dtype,), 2, dev)
        _need_shape(t, name, shape)
    return t.data_ptr(), _row_stride(t, name)


def _ids(t, name: str, T: int | None, dev: int) -> tuple[int, int]:
    """Checks contiguous int32 ids or positions [T, K]; returns their shape."""
    _need(t, name, torch.int32)
    if t.dim() != 2:
        raise MoeError(2, f"{name} must have 2 dimensions (got {t.dim()})")
    if t.get_device() != dev:
        raise MoeError(4, f"{name} is on {t.device}, the first tensor on cuda:{dev}")
    if T is not None and t.shape[0] != T:
        raise MoeError(3, f"{name} shape {tuple(t.shape)} for {T} tokens")
    return t.shape[0], t.shape[1]


def _add_rms_norm(x, gamma, residual, eps, want_y: bool, want_q: bool, stream):
    dt, dev = _first_float(x, "x", _FLOATS, 2)
    T, H = x.shape
    gt = _gamma(gamma, x.dtype, H, dev)
    rp, ldr = _rows_like(residual, "residual", x.dtype, (T, H), dev)
    ldx = _row_stride(x, "x")
    like = _like(x)
    new = _allocator(like, stream)
    q = new((T, H), torch.int8) if want_q else None
    scale = new((T,), torch.float32) if want_q else None
    y = new((T, H), x.dtype) if want_y else None
    total = None if residual is None else new((T, H), x.dtype)
    check(_lib.load().moe_add_rms_norm(x.data_ptr(), ldx, rp, ldr, gamma.data_ptr(), gt, _ptr(y), _ptr(total), _ptr(q),
                                       _ptr(scale), T, H, eps, dt, _queue(stream, dev)))
    return q, scale, y, total


def MoeAddRmsNorm(x: torch.Tensor, gamma: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
                  stream=None):
    """v = x[T,H] + residual[T,H] -> (y, v), y = v * gamma[H] / sqrt(mean(v^2) + eps), both of x's type (fp32, fp16 or
    bf16); the sum, which the next layer adds to, is None without a residual. v is summed and normalised in fp32 and
    rounded only where it is returned. gamma is of x's type or fp32; rows may be any stride apart."""
    return _add_rms_norm(x, gamma, residual, eps, True, False, stream)[2:]


def MoeAddRmsNormQuant(x: torch.Tensor, gamma: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
                       returnNorm: bool = False, stream=None):
    """MoeAddRmsNorm's y in 8 bits -> (q[T,H] int8, scale[T] fp32, y, v): q * scale is y, scale = max|y| / 127 of a row.
    y itself (for a router) with returnNorm, else None; v is None without a residual. q is rint(p * (127 / max|p|)) with
    p = v * gamma, the same bits whatever the launch; a row of zeros has scale 0, one that holds an infinity or a NaN
    has q 0 and scale NaN."""
    return _add_rms_norm(x, gamma, residual, eps, returnNorm, True, stream)


def add_rms_norm_grad_workspace_bytes(T: int, H: int) -> int:
    return int(_lib.load().moe_add_rms_norm_grad_workspace_bytes(T, H))


def MoeAddRmsNormGrad(grad_y: torch.Tensor, v: torch.Tensor, gamma: torch.Tensor, grad_v: torch.Tensor | None = None,
                      eps: float = 1e-6, gradX: bool = True, gradGamma: bool = True,
                      workspace: torch.Tensor | None = None, stream=None):
    """The gradients of MoeAddRmsNorm -> (grad_x[T,H], grad_gamma[H]), None where not asked for. v is the sum it
    returned (x itself without a residual), grad_v the gradient that reaches the sum by another way. grad_x is the
    residual's gradient too. H <= 16384. `workspace` (uint8, >= add_rms_norm_grad_workspace_bytes) is allocated when not
    given."""
    dt, dev = _first_float(v, "v", _FLOATS, 2)
    T, H = v.shape
    gt = _gamma(gamma, v.dtype, H, dev)
    yp, ldy = _rows_like(grad_y, "grad_y", v.dtype, (T, H), dev)
    if yp is None:
        raise MoeError(1, "grad_y must be a tensor")
    vp, ldv = _rows_like(grad_v, "grad_v", v.dtype, (T, H), dev)
    ld = _row_stride(v, "v")
    lib = _lib.load()
    like = _like(v)
    wp, wb = None, 0
    if gradGamma:
        workspace, wp, wb = _workspace(workspace, lib.moe_add_rms_norm_grad_workspace_bytes, (T, H), like, dev, stream)
    new = _allocator(like, stream)
    gx = new((T, H), v.dtype) if gradX else None
    gg = new((H,), gamma.dtype) if gradGamma else None
    check(lib.moe_add_rms_norm_grad(yp, ldy, v.data_ptr(), ld, gamma.data_ptr(), gt, vp, ldv, _ptr(gx), _ptr(gg), wp,
                                    wb, T, H, eps, dt, _queue(stream, dev)))
    return gx, gg


def MoeQuantize(x: torch.Tensor, stream=None):
    """Rows in 8 bits: x[R,H] (fp32, fp16 or bf16) -> (q[R,H] int8, scale[R] fp32), q * scale being x and scale = max|x|
    / 127 of a row. Contiguous experts' weights [E,N,H] -> (q[E,N,H], scale[E,N]): a weight row's scale is its output
    channel's. q is rint(x * (127 / max|x|)); rows of zeros have scale 0, rows with an infinity or a NaN q 0 and scale
    NaN."""
    if isinstance(x, torch.Tensor) and x.dim() == 3:
        if not x.is_contiguous():
            raise MoeError(4, "x must be contiguous (ND format)")
        q, scale = MoeQuantize(x.view(x.shape[0] * x.shape[1], x.shape[2]), stream)
        return q.view(x.shape), scale.view(x.shape[:2])
    dt, dev = _first_float(x, "x", _FLOATS, 2)
    R, H = x.shape
    ldx = _row_stride(x, "x")
    like = _like(x)
    new = _allocator(like, stream)
    q = new((R, H), torch.int8)
    scale = new((R,), torch.float32)
    check(_lib.load().moe_quantize(x.data_ptr(), ldx, q.data_ptr(), scale.data_ptr(), R, H, dt, _queue(stream, dev)))
    return q, scale


def permute_workspace_bytes(T: int, E: int, K: int) -> int:
    return int(_lib.load().moe_permute_workspace_bytes(T, E, K))


def MoePermute(x: torch.Tensor, expert_ids: torch.Tensor, numExperts: int, xScale: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None, stream=None):
    """x[T,H] (fp32, fp16, bf16 or int8), expert_ids[T,K] int32 -> (rows[T*K,H], offsets[E+1] int32, position[T,K]
    int32, row_scale): the rows of all picks sorted by expert, one expert's in the order of their slots. Expert e has
    rows [offsets[e], offsets[e+1]). Picks whose id is outside [0, E) come last, with rows of zeros. position is a
    pick's row, -1 - row of a pick of no expert. xScale[T] fp32 (8-bit rows' scales) is sorted alike, else row_scale is
    None. The gradient of rows is MoeUnpermute(grad_rows, position), of row_scale the same of its gradient as a column.
    `workspace` (uint8, >= permute_workspace_bytes) is allocated when not given."""
    dt, dev = _first_float(x, "x", (*_FLOATS, torch.int8), 2)
    T, H = x.shape
    _, K = _ids(expert_ids, "expert_ids", T, dev)
    sp = _vector(xScale, "xScale", torch.float32, T, dev)
    if type(numExperts) is not int or numExperts < 1:
        raise MoeError(4, f"numExperts={numExperts} must be positive")
    ldx = _row_stride(x, "x")
    lib = _lib.load()
    like = _like(x)
    workspace, wp, wb = _workspace(workspace, lib.moe_permute_workspace_bytes, (T, numExperts, K), like, dev, stream)
    new = _allocator(like, stream)
    rows = new((T * K, H), x.dtype)
    offsets = new((numExperts + 1,), torch.int32)
    position = new((T, K), torch.int32)
    row_scale = None if xScale is None else new((T * K,), torch.float32)
    check(lib.moe_permute(x.data_ptr(), ldx, sp, expert_ids.data_ptr(), rows.data_ptr(), _ptr(row_scale),
                          offsets.data_ptr(), position.data_ptr(), wp, wb, T, H, numExperts, K, dt,
                          _queue(stream, dev)))
    return rows, offsets, position, row_scale


def _row_weights(weights, shape, dev: int) -> tuple[int | None, int]:
    """(address, moe_dtype) of optional contiguous weights [T, K]."""
    if weights is None:
        return None, 0
    wt = _need_float(weights, "weights", _FLOATS, 2, dev)
    _need_shape(weights, "weights", shape)
    if not weights.is_contiguous():
        raise MoeError(4, "weights must be contiguous (ND format)")
    return weights.data_ptr(), wt


def MoeUnpermute(rows: torch.Tensor, position: torch.Tensor, weights: torch.Tensor | None = None,
                 stream=None) -> torch.Tensor:
    """rows[R,H] (fp32, fp16 or bf16), position[T,K], weights[T,K] (fp32, fp16 or bf16; None: 1) -> y[T,H] of rows'
    type, y[t] = sum over k of weights[t,k] * rows[position[t,k]] in fp32, ascending k. Positions outside [0, R) (a pick
    of no expert is negative) add nothing."""
    dt, dev = _first_float(rows, "rows", _FLOATS, 2)
    if not rows.is_contiguous():
        raise MoeError(4, "rows must be contiguous (ND format)")
    R, H = rows.shape
    T, K = _ids(position, "position", None, dev)
    wp, wt = _row_weights(weights, (T, K), dev)
    y = _empty(_like(rows), stream, (T, H), rows.dtype)
    check(_lib.load().moe_unpermute(rows.data_ptr(), R, position.data_ptr(), wp, wt, y.data_ptr(), T, H, K, dt,
                                    _queue(stream, dev)))
    return y


def unpermute_grad_any_workspace_bytes(T: int, K: int) -> int:
    return int(_lib.load().moe_unpermute_grad_any_workspace_bytes(T, K))


def MoeUnpermuteGrad(grad_y: torch.Tensor, rows: torch.Tensor | None, position: torch.Tensor,
                     weights: torch.Tensor | None = None, stream=None, anyPosition: bool = False,
                     workspace: torch.Tensor | None = None):
    """The gradients of MoeUnpermute's y[T,H] -> (grad_rows[T*K,H] of grad_y's type, grad_weights[T,K] of weights'
    type). position is MoePermute's, so every row has one pick; the rows of picks of no expert get zeros. Without
    weights rows may be None and grad_weights is None.

    With anyPosition position is whatever MoeUnpermute takes: positions outside [0, T*K) have no row and weight gradient
    0, a row that none names gets zeros and one that several name their sum (fp32, in ascending slot). `workspace`
    (uint8, >= unpermute_grad_any_workspace_bytes) is allocated when not given; otherwise it is not used."""
    dt, dev = _first_float(grad_y, "grad_y", _FLOATS, 2)
    T, H = grad_y.shape
    _, K = _ids(position, "position", T, dev)
    wp, wt = _row_weights(weights, (T, K), dev)
    rp = _matrix(rows, "rows", grad_y.dtype, (T * K, H), dev)
    if wp is not None and rows is None:
        raise MoeError(1, "MoeUnpermuteGrad needs rows with weights")
    ldy = _row_stride(grad_y, "grad_y")
    like = _like(grad_y)
    new = _allocator(like, stream)
    grad_rows = new((T * K, H), grad_y.dtype)
    grad_w = None if wp is None else new((T, K), weights.dtype)
    lib, args = _lib.load(), (grad_y.data_ptr(), ldy, rp, position.data_ptr(), wp, wt, grad_rows.data_ptr(), _ptr(grad_w))
    if anyPosition:
        workspace, ap, ab = _workspace(workspace, lib.moe_unpermute_grad_any_workspace_bytes, (T, K), like, dev, stream)
        check(lib.moe_unpermute_grad_any(*args, ap, ab, T, H, K, dt, _queue(stream, dev)))
    else:
        check(lib.moe_unpermute_grad(*args, T, H, K, dt, _queue(stream, dev)))
    return grad_rows, grad_w


def linear_int8_workspace_bytes(T: int, N: int, H: int, activation: str = "none", numExperts: int = 0) -> int:
    return int(_lib.load().moe_linear_int8_workspace_bytes(T, N, H, numExperts, _act_code(activation)))


def _contiguous(t, name: str, dtype, shape, dev: int) -> int | None:
    """The address of an optional contiguous tensor."""
    if t is None:
        return None
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.is_contiguous()
            and t.get_device() == dev):
        _need_float(t, name, (dtype,), len(shape), dev)
        _need_shape(t, name, shape)
        raise MoeError(4, f"{name} must be contiguous (ND format)")
    return t.data_ptr()


def MoeLinearInt8(x: torch.Tensor, xScale: torch.Tensor, weight: torch.Tensor, weightScale: torch.Tensor,
                  offsets: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  residual: torch.Tensor | None = None, activation: str = "none",
                  outDtype: torch.dtype = torch.float16, workspace: torch.Tensor | None = None,
                  stream=None) -> torch.Tensor:
    """act((x[T,H] @ weight[N,H]^T) * xScale[T] * weightScale[N] + bias[N]) + residual[T,N] -> y[T,N] of outDtype (fp16,
    bf16 or fp32), x and weight int8, scales fp32, bias and residual of outDtype; int32 sums, rounded once.

    With offsets[E+1] int32, weight[E,N,H], weightScale[E,N] and bias[E,N] are E experts': rows [offsets[e],
    offsets[e+1]) of x by the matrix of expert e (MoePermute's rows and offsets); rows from offsets[E] on become zeros.
    activation as MoeLinear's (swiglu: 2N weight rows, the N gate rows first). H <= 131071. Rows of x and of weight may
    be any stride apart; multiples of 16 (H too) run at full speed. `workspace` (uint8, >= linear_int8_workspace_bytes)
    is allocated when not given."""
    act = _act_code(activation)
    _, dev = _first_float(x, "x", _INT8, 2)
    _need_float(weight, "weight", _INT8, 2 if offsets is None else 3, dev)
    if outDtype not in _FLOATS:
        raise MoeError(4, f"outDtype must be float32, float16 or bfloat16 (got {outDtype})")
    T, H = x.shape
    if offsets is None:
        E, lead, step, rows = 0, (), 0, weight
    else:
        E = weight.shape[0]
        if E < 1:
            raise MoeError(3, "weight holds no experts")
        lead, step, rows = (E,), weight.stride(0), weight[0]
    Z = rows.shape[0]
    if rows.shape[1] != H:
        raise MoeError(3, f"hidden size mismatch x[{H}] vs weight[{rows.shape[1]}]")
    swiglu = act == ACTIVATIONS["swiglu"]
    if swiglu and Z % 2:
        raise MoeError(3, f"weight rows ({Z}) of a swiglu must be N gate and N up rows")
    N = Z // 2 if swiglu else Z
    sx = _contiguous(xScale, "xScale", torch.float32, (T,), dev)
    sw = _contiguous(weightScale, "weightScale", torch.float32, (*lead, Z), dev)
    if sx is None or sw is None:
        raise MoeError(1, "xScale and weightScale must be tensors")
    op = _contiguous(offsets, "offsets", torch.int32, (E + 1,), dev)
    bp = _contiguous(bias, "bias", outDtype, (*lead, Z), dev)
    rp = _contiguous(residual, "residual", outDtype, (T, N), dev)
    ldx, ldw = _row_stride(x, "x"), _row_stride(rows, "weight")
    lib = _lib.load()
    like = _like(x)
    workspace, wp, wb = _workspace(workspace, lib.moe_linear_int8_workspace_bytes, (T, N, H, E, act), like, dev, stream)
    y = _empty(like, stream, (T, N), outDtype)
    check(lib.moe_linear_int8(x.data_ptr(), ldx, sx, weight.data_ptr(), ldw, step, sw, op, bp, rp, y.data_ptr(), wp, wb,
                              T, N, H, E, act, _FLOAT_DT[outDtype], _queue(stream, dev)))
    return y


def moe_layer_int8(x: torch.Tensor, gamma: torch.Tensor, w_gate: torch.Tensor, gate_up: torch.Tensor,
                   gate_up_scale: torch.Tensor, down: torch.Tensor, down_scale: torch.Tensor,
                   residual: torch.Tensor | None = None, topK: int = 2, bias: torch.Tensor | None = None,
                   numGroups: int = 1, topGroups: int = 1, groupTop: int = 1, scoring: str = "softmax",
                   renormalize: bool = True, scale: float = 1.0, eps: float = 1e-6, stream=None):
    """A layer of 8-bit experts behind its norm, x fp16 or bf16: the norm of x + residual for the router as it is and
    for the experts in 8 bits (MoeAddRmsNormQuant), fp32 logits by w_gate[H,E] (MoeLinear), MoeRoutingGroupTopK, the
    tokens sorted by expert (MoePermute), the products by gate_up[E,2I,H] with SwiGLU and, in 8 bits again
    (MoeQuantize), by down[E,H,I] (MoeLinearInt8; MoeQuantize makes such weights and their scales [E,2I] and [E,H]), and
    the way back (MoeUnpermute). Returns (y, v, expert_ids, weights): y without the sum v = x + residual, which the next
    layer adds y to; v is None without a residual."""
    if w_gate.dim() != 2 or gate_up.dim() != 3 or gate_up.shape[0] != w_gate.shape[1]:
        raise MoeError(3, f"w_gate {tuple(w_gate.shape)} and gate_up {tuple(gate_up.shape)}: "
                          "[H, E] and [E, 2I, H] expected")
    q, q_scale, normed, v = MoeAddRmsNormQuant(x, gamma, residual, eps, returnNorm=True, stream=stream)
    logits = MoeLinear(normed, w_gate.t(), outDtype=torch.float32, stream=stream)
    ids, w = MoeRoutingGroupTopK(logits, bias, topK, numGroups, topGroups, groupTop, scoring, renormalize, scale,
                                 torch.float32, stream=stream)
    rows, offsets, position, row_scale = MoePermute(q, ids, gate_up.shape[0], q_scale, stream=stream)
    hidden = MoeLinearInt8(rows, row_scale, gate_up, gate_up_scale, offsets, activation="swiglu", outDtype=x.dtype,
                           stream=stream)
    hidden, hidden_scale = MoeQuantize(hidden, stream=stream)
    out = MoeLinearInt8(hidden, hidden_scale, down, down_scale, offsets, outDtype=x.dtype, stream=stream)
    return MoeUnpermute(out, position, w, stream=stream), v, ids, w


def synth_normal_f16_(out: torch.Tensor, seed: int, stream_id: int, sigma_a: float, sigma_b: float | None = None,
                      period: int = 0, split: int = 0, stream=None) -> torch.Tensor:
    """Fill an fp16 device tensor in place with the generator of synth.py (moe_synth_normal_f16)."""
    _need(out, "out", torch.float16)
    if sigma_b is None or period <= 0:
        sigma_b, period, split = sigma_a, 1, 1
    check(_lib.load().moe_synth_normal_f16(out.data_ptr(), out.numel(), seed, stream_id, sigma_a, sigma_b, period,
                                           split, _stream_ptr(stream)))
    return out


def copy_bytes_(dst: torch.Tensor, src: torch.Tensor, stream=None) -> None:
    n = src.numel() * src.element_size()
    check(_lib.load().moe_copy_bytes(dst.data_ptr(), src.data_ptr(), n, _stream_ptr(stream)))


def stream_read_(src: torch.Tensor, stream=None) -> None:
    """Read a device tensor (size a multiple of 16 KiB) with moe_stream_read_bytes: achievable HBM read rate."""
    n = src.numel() * src.element_size()
    check(_lib.load().moe_stream_read_bytes(src.data_ptr(), n, _stream_ptr(stream)))


@contextlib.contextmanager
def kernel_trace():
    """Record HIP events around every kernel the library launches; yields a dict filled on exit with
    {kernel_name: (launches, total_ms)}."""
    lib = _lib.load()
    result: dict[str, tuple[int, float]] = {}
    check(lib.moe_trace_enable(1))
    try:
        yield result
    finally:
        n = lib.moe_trace_collect()
        for i in range(n):
            name, launches, ms = C.c_char_p(), C.c_int64(), C.c_double()
            check(lib.moe_trace_get(i, C.byref(name), C.byref(launches), C.byref(ms)))
            result[name.value.decode()] = (launches.value, ms.value)
        check(lib.moe_trace_enable(0))
