"""Tokens sorted by expert and back, and the routing weights, each with its gradient.

``route_dispatch`` routes and dispatches in one call and is not differentiable.  The functions here are its parts for
training and for routings that come from elsewhere: ``sort_tokens`` (rows in expert order for given expert ids),
``unsort_tokens`` (the weighted way back) and ``routing_weights`` (the combine weights of chosen experts as a function
of the logits).  Where an argument requires a gradient, autograd reaches the hand-written backward kernels; the same
kernels are there as plain functions (``unsort_tokens_backward``, ``routing_weights_backward``; the gradient of the sort
is ``unsort_tokens`` without weights), which are what a CUDA graph may record.  There is no forward-mode derivative: tensors
that carry a tangent are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _cabi
from ._cabi import BIAS_MODES, ROW_DTYPE, SCORE_FN


class SortedTokens(NamedTuple):
    rows: torch.Tensor          # [R, H] the tokens' rows, experts ascending; zeros behind offsets[E]
    offsets: torch.Tensor       # [E+1] int32, offsets[E] = rows in use
    inverse_perm: torch.Tensor  # [T, K] int32 row of every pair, -1 = none
    row_token: torch.Tensor     # [R] int32 token of every row, -1 behind offsets[E]
    counts: torch.Tensor        # [E] int32 pairs per expert before dropping


class UnsortGradients(NamedTuple):
    rows: Optional[torch.Tensor]     # [R, H] gradient of the expert outputs
    weights: Optional[torch.Tensor]  # [T, K] fp32 gradient of the weights


_increment_version = torch.autograd.graph.increment_version
_VECTOR = {torch.bfloat16: 8, torch.float16: 8, torch.float32: 4}  # elements in 16 bytes


def device_index(name: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """The index of the one CUDA device of all the tensors."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name}: all tensors must be on one device, got {first.device} and {t.device}")
    if index < 0 or not first.is_cuda:
        raise RuntimeError(f"moe_rd.{name} has no CPU path: its tensors must be CUDA tensors")
    return index


def call(index: int, entry, *args) -> None:
    """Enqueue a C entry point on the current stream of CUDA device ``index``."""
    if index == torch.cuda.current_device():
        code = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            code = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    if code:
        _cabi.check(code)


def dense(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """The tensor, or a copy of it, contiguous and 16-byte aligned (a view may start anywhere), and its address."""
    t = t.resolve_neg()
    if not t.is_contiguous():
        t = t.contiguous()
    at = t.data_ptr()
    if at & 15:
        t = t.clone()
        at = t.data_ptr()
    return t, at


def packed(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """The same for what the kernels read element by element: indices, weights, logits (no alignment is needed)."""
    t = t.resolve_neg()
    if not t.is_contiguous():
        t = t.contiguous()
    return t, t.data_ptr()


def check_out(name: str, out: torch.Tensor, shape: Tuple[int, ...], dtype: torch.dtype, index: int, inputs, align: int = 1) -> int:
    """``out`` is a buffer the call may write: of this shape and type, contiguous, apart from the inputs ((address, bytes)
    each).  Returns its address."""
    if out.shape != shape or out.dtype is not dtype or out.get_device() != index or not out.is_contiguous() or out.requires_grad or out.is_neg():
        raise ValueError(f"{name}: out must be a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{index} that needs no gradient")
    lo = out.data_ptr()
    if lo % align:
        raise ValueError(f"{name}: out must be {align}-byte aligned")
    for at, nbytes in inputs:
        if lo < at + nbytes and at < lo + out.nbytes:
            raise ValueError(f"{name}: out must not share memory with an input")
    return lo


def written(*out: Optional[torch.Tensor]) -> None:
    """Tell autograd that these buffers of the caller have been overwritten: a graph that saved one of them then raises in
    its backward pass instead of computing with the new contents."""
    _increment_version([t for t in out if t is not None])


def wants_grad(*tensors: Optional[torch.Tensor]) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def refuse_tangents(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Forward mode: a tangent would be dropped without a word (an ``autograd.Function`` of the caller, whose ``jvp`` carries
    it on, calls with forward mode off)."""
    if torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and unpack_dual(t).tangent is not None:
                raise RuntimeError(f"moe_rd.{name} has no forward-mode derivative: pass tensors without a tangent")


def _not_while_capturing(name: str, instead: str) -> None:
    # A captured backward pass can end the process when an eager graph of the same leaves is alive, and nothing
    # here can see whether one is; the plain functions do not go through the autograd engine.
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"moe_rd.{name}: autograd is not recorded into a CUDA graph; capture {instead} instead")


def _check_ids(name: str, ids: torch.Tensor) -> Tuple[int, int]:
    if ids.dtype is not torch.int32:
        raise TypeError(f"{name}: row and expert indices must be int32")
    shape = ids.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{name}: row and expert indices must be [T, K]")
    return shape


def _check_rows(name: str, rows: torch.Tensor) -> int:
    if rows.dtype not in _VECTOR:
        raise TypeError(f"{name}: rows must be bfloat16, float16 or float32")
    shape = rows.shape
    if len(shape) < 2 or shape[-1] < 1 or shape[-1] % _VECTOR[rows.dtype]:
        raise ValueError(f"{name}: rows must be [..., H] with H * element size a multiple of 16 bytes")
    return shape[-1]


# --- sort ------------------------------------------------------------------------------------------------------------
def _sort(index, T, K, H, x, expert_ids, E, capacity, out):
    x, x_at = dense(x if x.dim() == 2 else x.reshape(T, H))
    ids, ids_at = packed(expert_ids)
    R = min(T * K, E * capacity) if capacity else T * K
    dtype = x.dtype
    code = ROW_DTYPE[dtype]
    if out is None:
        # parts of one buffer would share its version: a change of the counts would look like one of the places, which a
        # graph may have saved
        result = SortedTokens(torch.empty((R, H), dtype=dtype, device=x.device),
                              *(torch.empty(n, dtype=torch.int32, device=x.device) for n in ((E + 1,), (T, K), (R,), (E,))))
        at = [t.data_ptr() for t in result]
    else:
        result = out
        i32 = torch.int32
        given = ((x_at, x.nbytes), (ids_at, 4 * T * K))
        at = (check_out("sort_tokens", out.rows, (R, H), dtype, index, given, 16), check_out("sort_tokens", out.offsets, (E + 1,), i32, index, given),
              check_out("sort_tokens", out.inverse_perm, (T, K), i32, index, given), check_out("sort_tokens", out.row_token, (R,), i32, index, given),
              check_out("sort_tokens", out.counts, (E,), i32, index, given))
    ws_bytes = _cabi.sort_workspace_bytes(T, H, E, K, code)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    call(index, _cabi.lib().moe_rd_sort_tokens, T, H, E, K, code, capacity, R, x_at, ids_at, *at, ws.data_ptr() if ws_bytes else None, ws_bytes)
    if out is not None:
        _increment_version(out)
    return result


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, expert_ids, num_experts, capacity):
        out = _sort(x.get_device(), *expert_ids.shape, x.shape[-1], x, expert_ids, num_experts, capacity, None)
        ctx.save_for_backward(out.inverse_perm)
        ctx.shape = x.shape
        ctx.mark_non_differentiable(*out[1:])
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_rows, *_):
        _not_while_capturing("sort_tokens", "sort_tokens on detached tensors and unsort_tokens for its gradient")
        (inverse_perm,) = ctx.saved_tensors
        grad = _unsort(grad_rows.get_device(), *inverse_perm.shape, ctx.shape[-1], grad_rows, inverse_perm, None, None, None)
        return grad.reshape(ctx.shape), None, None, None


def sort_tokens(x: torch.Tensor, expert_ids: torch.Tensor, num_experts: int, *, capacity: int = 0,
                out: Optional[SortedTokens] = None) -> SortedTokens:
    """Rows of ``x`` in expert order: ``rows[inverse_perm[t, k]] = x[t]`` for every pair (t, k) that has a row.

    x: [..., H] bf16, fp16 or fp32 (any strides; H * element size a multiple of 16 bytes), T tokens in all.
    expert_ids: [T, K] int32; an id outside [0, num_experts) is a pair without an expert (a padded token has K of
    them), and one expert may occur twice for a token.  ``capacity`` keeps that many rows per expert, in (token, slot)
    order, as in ``route_dispatch``; 0 keeps all.  The order inside an expert is the stable (token, slot) order.
    Rows behind ``offsets[-1]`` are zero, with ``row_token`` -1.  At most 256 experts and 32 ids per token.

    Differentiable in ``x``; the gradient is ``unsort_tokens(grad_rows, inverse_perm)``.  ``out`` takes the result of
    an earlier call of the same sizes and reuses its buffers (not where ``x`` requires a gradient).
    """
    done = _cabi.fast.sort_tokens(x, expert_ids, num_experts, capacity, out)
    if done is not False:
        return out if done is True else SortedTokens(*done)
    H = _check_rows("sort_tokens", x)
    T, K = _check_ids("sort_tokens", expert_ids)
    if x.numel() != T * H:
        raise ValueError(f"sort_tokens: {x.numel() // H} tokens, but expert ids for {T}")
    if num_experts < 1 or capacity < 0:
        raise ValueError("sort_tokens: num_experts must be positive and capacity not negative")
    num_experts, capacity = int(num_experts), int(capacity)
    refuse_tangents("sort_tokens", x)
    index = device_index("sort_tokens", x, expert_ids)
    if not wants_grad(x):
        return _sort(index, T, K, H, x, expert_ids, num_experts, capacity, out)
    if out is not None:
        raise ValueError("sort_tokens: out cannot be given where x requires a gradient")
    _not_while_capturing("sort_tokens", "sort_tokens on detached tensors and unsort_tokens for its gradient")
    return SortedTokens(*_SortTokens.apply(x, expert_ids, num_experts, capacity))


# --- and back --------------------------------------------------------------------------------------------------------
def _check_unsort(name, y, inverse_perm, weights, shared):
    H = _check_rows(name, y)
    T, K = _check_ids(name, inverse_perm)
    if weights is not None:
        if weights.dtype is not torch.float32:
            raise TypeError(f"{name}: weights must be float32")
        if weights.shape != (T, K):
            raise ValueError(f"{name}: weights must be [T, K] like inverse_perm")
    if shared is not None:
        if shared.dtype is not y.dtype:
            raise TypeError(f"{name}: the [T, H] tensor must have the type of the rows")
        if shared.shape != (T, H) and (shared.dim() < 1 or shared.shape[-1] != H or shared.numel() != T * H):
            raise ValueError(f"{name}: expected a tensor of T = {T} rows of {H}")
    return T, K, H


def _unsort(index, T, K, H, y, inverse_perm, weights, shared, out):
    y, y_at = dense(y if y.dim() == 2 else y.reshape(-1, H))
    inv, inv_at = packed(inverse_perm)
    w, w_at = (None, None) if weights is None else packed(weights)
    sh, sh_at = (None, None) if shared is None else dense(shared if shared.dim() == 2 else shared.reshape(T, H))
    R = y.shape[0]
    dtype = y.dtype
    if out is None:
        result = torch.empty((T, H), dtype=dtype, device=y.device)
        at = result.data_ptr()
    else:
        result = out
        given = [(y_at, y.nbytes), (inv_at, 4 * T * K)]
        if w is not None:
            given.append((w_at, 4 * T * K))
        if sh is not None:
            given.append((sh_at, sh.nbytes))
        at = check_out("unsort_tokens", out, (T, H), dtype, index, given, 16)
    call(index, _cabi.lib().moe_rd_unsort_tokens, T, H, K, ROW_DTYPE[dtype], y_at, R, inv_at, w_at, sh_at, at)
    if out is not None:
        _increment_version(out)
    return result


class _UnsortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, inverse_perm, weights, shared, offsets):
        out = _unsort(y.get_device(), *inverse_perm.shape, y.shape[-1], y, inverse_perm, weights, shared, None)
        need_w = weights is not None and ctx.needs_input_grad[2]
        ctx.save_for_backward(y if need_w else None, inverse_perm, weights, offsets)
        ctx.y_shape = y.shape
        ctx.shared_shape = None if shared is None else shared.shape
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        _not_while_capturing("unsort_tokens", "unsort_tokens on detached tensors and unsort_tokens_backward")
        y, inverse_perm, weights, offsets = ctx.saved_tensors
        need_y, need_w = ctx.needs_input_grad[0], weights is not None and ctx.needs_input_grad[2]
        grad_y = grad_w = grad_shared = None
        if need_y or need_w:
            grad_y, grad_w = _unsort_backward(grad_out.get_device(), grad_out, y, ctx.y_shape, inverse_perm, weights, offsets, need_y, need_w, None)
        if ctx.needs_input_grad[3]:
            grad_shared = grad_out.reshape(ctx.shared_shape)
        return grad_y, None, grad_w, grad_shared, None


def unsort_tokens(y: torch.Tensor, inverse_perm: torch.Tensor, weights: Optional[torch.Tensor] = None,
                  shared: Optional[torch.Tensor] = None, *, offsets: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = shared[t] + sum_k weights[t, k] * y[inverse_perm[t, k]], rounded once from fp32.

    ``combine`` for rows of any type (bf16, fp16, fp32), with a gradient.  y: [..., H] rows in expert order;
    inverse_perm: [T, K] int32 as ``sort_tokens`` or ``route_dispatch`` return it (each row at most once; an index
    outside the rows of y is a pair that contributes nothing, whatever its weight); weights: [T, K] fp32, or None for 1;
    shared: T rows like y's, or None.

    Differentiable in ``y``, ``weights`` and ``shared``; rows of ``y`` that no pair has get a zero gradient.  With
    ``offsets`` (of the same sort: no pair has a row from ``offsets[-1]`` on) the gradient of ``y`` is written in one
    pass; without it it is cleared first.  ``out`` takes a [T, H] buffer (not where a gradient is required).
    """
    done = _cabi.fast.unsort_tokens(y, inverse_perm, weights, shared, offsets, out)
    if done is not False:
        return out if done is True else done
    T, K, H = _check_unsort("unsort_tokens", y, inverse_perm, weights, shared)
    refuse_tangents("unsort_tokens", y, weights, shared)
    index = device_index("unsort_tokens", y, inverse_perm, weights, shared, offsets)
    if offsets is not None:
        check_offsets("unsort_tokens", offsets)
    if not wants_grad(y, weights, shared):
        return _unsort(index, T, K, H, y, inverse_perm, weights, shared, out)
    if out is not None:
        raise ValueError("unsort_tokens: out cannot be given where a gradient is required")
    _not_while_capturing("unsort_tokens", "unsort_tokens on detached tensors and unsort_tokens_backward")
    return _UnsortTokens.apply(y, inverse_perm, weights, shared, offsets)


def check_offsets(name, offsets):
    if offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.numel() < 1 or not offsets.is_contiguous():
        raise TypeError(f"{name}: offsets must be a contiguous [E+1] int32 tensor")


def _unsort_backward(index, grad_out, y, y_shape, inverse_perm, weights, offsets, need_y, need_w, out):
    T, K = inverse_perm.shape
    H = y_shape[-1]
    R = 1
    for n in y_shape[:-1]:
        R *= n
    g, g_at = dense(grad_out if grad_out.dim() == 2 else grad_out.reshape(T, H))
    y, y_at = dense(y if y.dim() == 2 else y.reshape(R, H)) if need_w else (None, None)
    inv, inv_at = packed(inverse_perm)
    w, w_at = (None, None) if weights is None else packed(weights)
    dtype = g.dtype
    end_at = None if offsets is None else offsets.data_ptr() + 4 * (offsets.numel() - 1)
    rows_at = weights_at = None
    if out is None:
        result = UnsortGradients(torch.empty(y_shape, dtype=dtype, device=g.device) if need_y else None,
                                 torch.empty((T, K), dtype=torch.float32, device=g.device) if need_w else None)
        rows_at = result.rows.data_ptr() if need_y else None
        weights_at = result.weights.data_ptr() if need_w else None
    else:
        result = out
        if (out.rows is not None) != need_y or (out.weights is not None) != need_w:
            raise ValueError("unsort_tokens_backward: out must hold the gradients that are asked for")
        given = [(t_at, t.nbytes) for t, t_at in ((g, g_at), (y, y_at), (inv, inv_at), (w, w_at)) if t is not None]
        if end_at is not None:
            given.append((end_at, 4))
        if need_y:
            rows_at = check_out("unsort_tokens_backward", out.rows, y_shape, dtype, index, given, 16)
        if need_w:
            weights_at = check_out("unsort_tokens_backward", out.weights, (T, K), torch.float32, index, given)
    call(index, _cabi.lib().moe_rd_unsort_tokens_backward, T, H, K, ROW_DTYPE[dtype], g_at, y_at, R, inv_at, w_at, end_at, rows_at, weights_at)
    if out is not None:
        written(*out)
    return result


def unsort_tokens_backward(grad_out: torch.Tensor, y: torch.Tensor, inverse_perm: torch.Tensor,
                           weights: Optional[torch.Tensor] = None, *, offsets: Optional[torch.Tensor] = None,
                           need_rows: bool = True, need_weights: Optional[bool] = None,
                           out: Optional[UnsortGradients] = None) -> UnsortGradients:
    """Gradients of ``unsort_tokens`` for ``grad_out`` [T, H]: of the rows of ``y`` (the type of y) and of ``weights``
    (fp32, added in a fixed order; asked for by default where weights are given).  The gradient of ``shared`` is
    ``grad_out`` itself.  Rows of y that no pair has get a zero gradient, wherever they are.  ``offsets``: as in
    ``unsort_tokens``.  ``out`` takes the result of an earlier call of the same sizes."""
    need_weights = weights is not None if need_weights is None else need_weights
    done = _cabi.fast.unsort_tokens_backward(grad_out, y, inverse_perm, weights, offsets, need_rows, need_weights, out)
    if done is not False:
        return out if done is True else UnsortGradients(*done)
    _check_unsort("unsort_tokens_backward", y, inverse_perm, weights, grad_out)
    refuse_tangents("unsort_tokens_backward", grad_out, y, weights)
    if offsets is not None:
        check_offsets("unsort_tokens_backward", offsets)
    if not (need_rows or need_weights):
        raise ValueError("unsort_tokens_backward: no gradient is asked for")
    index = device_index("unsort_tokens_backward", grad_out, y, inverse_perm, weights, offsets)
    return _unsort_backward(index, grad_out, y, y.shape, inverse_perm, weights, offsets, need_rows, need_weights, out)


_BIAS_USE = {"none": 0, "select": 0, "logit": 1, "select_and_weight": 2}


# --- routing weights -------------------------------------------------------------------------------------------------
def _check_weights(name, logits, expert_ids, bias, bias_mode, score_fn):
    if logits.dtype is not torch.float32:
        raise TypeError(f"{name}: logits must be float32")
    T, K = _check_ids(name, expert_ids)
    shape = logits.shape
    if len(shape) != 2 or shape[0] != T or shape[1] < 1:
        raise ValueError(f"{name}: logits must be [T, E] for the T = {T} tokens of expert_ids")
    if score_fn not in SCORE_FN:
        raise ValueError(f"{name}: score_fn must be one of {tuple(SCORE_FN)}")
    if bias_mode not in BIAS_MODES:
        raise ValueError(f"{name}: bias_mode must be one of {BIAS_MODES}")
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.numel() != shape[1]:
            raise ValueError(f"{name}: bias must be a float32 tensor of E elements")
        if wants_grad(bias):
            raise ValueError(f"{name}: bias is a constant here; add a learned bias to the logits")


def _weights_call(name, entry, index, logits, expert_ids, bias, config, grad, shape, out):
    """One of the two kernels; ``shape`` is that of its result."""
    bias_mode, score_fn, renorm, routed_scale, norm_min = config
    T, E = logits.shape
    logits, logits_at = packed(logits)
    ids, ids_at = packed(expert_ids)
    given = [(logits_at, 4 * T * E), (ids_at, ids.nbytes)]
    bias_at, inputs = None, ()
    if bias is not None:
        bias, bias_at = packed(bias)
        given.append((bias_at, 4 * E))
    if grad is not None:
        grad, grad_at = packed(grad)
        given.append((grad_at, grad.nbytes))
        inputs = (grad_at,)
    if out is None:
        result = torch.empty(shape, dtype=torch.float32, device=logits.device)
        at = result.data_ptr()
    else:
        result = out
        at = check_out(name, out, shape, torch.float32, index, given)
    call(index, entry, T, E, ids.shape[1], SCORE_FN[score_fn], 1 if renorm else 0, routed_scale, norm_min, logits_at, ids_at,
         bias_at if bias_mode == "logit" else None, bias_at if bias_mode == "select_and_weight" else None, *inputs, at)
    if out is not None:
        _increment_version(out)
    return result


class _RoutingWeights(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, expert_ids, bias, config):
        ctx.save_for_backward(logits, expert_ids, bias)
        ctx.config = config
        return _weights_call("routing_weights", _cabi.lib().moe_rd_routing_weights, logits.get_device(), logits, expert_ids, bias, config, None,
                             expert_ids.shape, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _not_while_capturing("routing_weights", "routing_weights on detached logits and routing_weights_backward")
        logits, expert_ids, bias = ctx.saved_tensors
        return _weights_call("routing_weights", _cabi.lib().moe_rd_routing_weights_backward, logits.get_device(), logits, expert_ids, bias,
                             ctx.config, grad, logits.shape, None), None, None, None


def routing_weights(logits: torch.Tensor, expert_ids: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                    score_fn: str = "softmax", bias_mode: str = "select", renorm: bool = True, routed_scale: float = 1.0,
                    norm_min: float = 1e-20, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The combine weights [T, K] of the experts ``expert_ids`` as a function of the router's ``logits`` [T, E] fp32.

    The keywords are those of ``route_dispatch``, whose ``combine_weights`` these are (within rounding) for the ids that it
    chose; a bias that is for selection only ("select") has no part in them.  Slots whose id is outside [0, E) have
    weight 0 and no part in the sum.  Differentiable in ``logits`` (ids and bias are constants): with
    ``logits = x @ gate_weight`` it carries the gradient of the weights to the router.
    """
    done = _cabi.fast.routing_weights(None, logits, expert_ids, bias, _BIAS_USE.get(bias_mode), SCORE_FN.get(score_fn), renorm, routed_scale,
                                      norm_min, out)
    if done is not False:
        return out if done is True else done
    _check_weights("routing_weights", logits, expert_ids, bias, bias_mode, score_fn)
    refuse_tangents("routing_weights", logits, bias)
    index = device_index("routing_weights", logits, expert_ids, bias)
    config = (bias_mode, score_fn, renorm, routed_scale, norm_min)
    if wants_grad(logits):
        if out is not None:
            raise ValueError("routing_weights: out cannot be given where a gradient is required")
        _not_while_capturing("routing_weights", "routing_weights on detached logits and routing_weights_backward")
        return _RoutingWeights.apply(logits, expert_ids, bias, config)
    return _weights_call("routing_weights", _cabi.lib().moe_rd_routing_weights, index, logits, expert_ids, bias, config, None,
                         expert_ids.shape, out)


def routing_weights_backward(grad_weights: torch.Tensor, logits: torch.Tensor, expert_ids: torch.Tensor,
                             bias: Optional[torch.Tensor] = None, *, score_fn: str = "softmax", bias_mode: str = "select",
                             renorm: bool = True, routed_scale: float = 1.0, norm_min: float = 1e-20,
                             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient [T, E] fp32 of ``routing_weights`` with respect to the logits, for ``grad_weights`` [T, K] fp32.  Where
    the sum of the chosen scores is below ``norm_min`` it has no part in the gradient; a token without any valid id gets
    zeros."""
    if grad_weights is not None:
        done = _cabi.fast.routing_weights(grad_weights, logits, expert_ids, bias, _BIAS_USE.get(bias_mode), SCORE_FN.get(score_fn), renorm,
                                          routed_scale, norm_min, out)
        if done is not False:
            return out if done is True else done
    _check_weights("routing_weights_backward", logits, expert_ids, bias, bias_mode, score_fn)
    if grad_weights.dtype is not torch.float32 or grad_weights.shape != expert_ids.shape:
        raise ValueError("routing_weights_backward: grad_weights must be a float32 tensor like expert_ids")
    refuse_tangents("routing_weights_backward", grad_weights, logits, bias)
    index = device_index("routing_weights_backward", logits, grad_weights, expert_ids, bias)
    return _weights_call("routing_weights_backward", _cabi.lib().moe_rd_routing_weights_backward, index, logits, expert_ids, bias,
                         (bias_mode, score_fn, renorm, routed_scale, norm_min), grad_weights, logits.shape, out)
