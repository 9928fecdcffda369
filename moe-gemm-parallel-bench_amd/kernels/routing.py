"""Routing on gfx950: each token's experts, and the way to expert-sorted rows and back.

What stands before and behind the experts' products, which take expert-sorted rows and their end offsets.  A serving step
of a mixture-of-experts layer::

    weights, experts = route_topk(logits, 8)                # [T, 8] fp32 and int32
    order = sort_by_expert(experts, num_experts)            # end offsets, and where each token's slots went
    xs = gather_rows(x, order)                              # [T * 8, H], sorted by expert
    ys = grouped_mm(grouped_mm_swiglu(xs, w13, order.offs), w2, order.offs)
    out = combine_rows(ys, order, weights)                  # [T, H], weighted

In training ``gate_up_swiglu`` takes the place of ``grouped_mm_swiglu``; ``grouped_mm`` keeps no history, so the gradient of the
second product is the program's own (``grouped_mm`` of the transposed weight for the rows).  ``route_topk``, ``gather_rows`` and
``combine_rows`` are differentiable, in reverse mode only; ``route_topk_backward`` and ``combine_rows_backward`` are the
gradients for programs that run their own backward pass (without a history of their own), and the gradient of ``gather_rows`` is ``combine_rows`` of the
sorted rows' gradient.  An expert-parallel rank sorts for its own experts (``first``, ``num_experts``); slots of other ranks'
experts get no row.

Calls run on the current stream of their tensors' device, read no counts back and keep nothing, so they can be captured in
a HIP graph; repeated calls give the same bits.  ``ValueError`` for arguments the kernels cannot take, ``RuntimeError``
without library or GPU.  The reference routes uniformly on the host (README.md:55-57): this has no counterpart there.
"""

from __future__ import annotations

from typing import NamedTuple

from . import _native

MAX_EXPERTS = 1024
MAX_TOP_K = 64
SCORES = ("softmax", "sigmoid")


class ExpertOrder(NamedTuple):
    """Slots (token t's j-th expert is slot ``t * k + j``) sorted by expert, equal ones in slot order; all int32.

    ``offs`` [experts]: each expert's end row, as the products take it.  ``slots`` [T * k]: the slot of each sorted row,
    -1 at and past ``offs[-1]``.  ``places`` [T, k]: the sorted row of each slot, -1 where its expert is not among
    the sorted ones.
    """

    offs: object
    slots: object
    places: object


def _score_flag(score: str) -> int:
    if score not in SCORES:
        raise ValueError(f"score must be one of {SCORES}, got {score!r}")
    return SCORES.index(score)


def _check_logits(logits, k) -> tuple[int, int]:
    if logits.ndim != 2:
        raise ValueError("logits must be a 2-D [tokens, experts] tensor")
    tokens, experts = logits.shape
    if not logits.is_cuda:
        raise ValueError("logits must be on a GPU device")
    if tokens > _native.INT32_MAX or not 0 < experts <= MAX_EXPERTS:
        raise ValueError(f"route_topk takes under 2**31 tokens and 1 to {MAX_EXPERTS} experts (got {tuple(logits.shape)})")
    if not 0 < k <= min(experts, MAX_TOP_K):
        raise ValueError(f"k must be 1 to min(experts, {MAX_TOP_K}) (got {k})")
    if logits.stride(1) != 1 and experts > 1:
        raise ValueError("logits need a unit stride along the experts")
    return tokens, experts


def _row_stride(t) -> int:
    """Stride between rows; of a single row, or none, one that covers it."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def route_topk(logits, k: int, *, score: str = "softmax", bias=None, groups: int = 1, top_groups: int | None = None,
               group_best: int = 1, normalize: bool = True, scale: float = 1.0):
    """Each token's ``k`` experts by score: ``(weights [T, k] fp32, experts [T, k] int32)``, best first.

    ``s = softmax(logits)`` or ``sigmoid(logits)`` over the experts; ``c = s + bias`` (fp32 [E], or none) chooses.  With
    ``groups`` equal runs of experts, only the ``top_groups`` (default: all) runs with the largest sums of their
    ``group_best`` (1 or 2) best ``c`` are eligible.  The ``k`` largest ``c`` win; ties go to the lowest index, of groups
    too, and 0.0 and -0.0 are one number.  ``weights = s`` of the chosen, divided by their sum if ``normalize``, times ``scale``
    (held in fp32).  Divided, a softmax's are the softmax of the chosen logits alone, also where every chosen score
    underflows; they are 0 where the chosen logits are all -inf, and a sigmoid's where their 64-bit sum is 0.

    logits: fp16, bf16 or fp32 [T, E] with unit stride along E, E at most 1024 and k at most 64.  Choices are made on 64-bit
    scores, so they do not hang on the rounding of an exponential; without a bias, and with ``group_best`` 1, the logits rank,
    which is the scores' order and tells apart what is equal in 64 bits (sigmoids past 37; softmax scores that underflow).  A
    logit of -inf has score 0; a NaN ranks below every other score, and makes all softmax weights of its token NaN.
    Differentiable in logits (through ``s``; the choice is taken as given, and no gradient goes to ``bias``).
    """
    import torch

    _native.refuse_tangents("route_topk", logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _functions()[0].apply(logits, k, score, bias, groups, top_groups, group_best, normalize, scale)
    return _route(logits, k, score, bias, groups, top_groups, group_best, normalize, scale)


def _route(logits, k, score, bias, groups, top_groups, group_best, normalize, scale):
    import torch

    sigmoid = _score_flag(score)
    tokens, experts = _check_logits(logits, k)
    code = _native.dtype_code(logits.dtype)
    top_groups = groups if top_groups is None else top_groups
    if groups <= 0 or experts % groups or not 0 < top_groups <= groups or group_best not in (1, 2):
        raise ValueError(f"groups must divide the {experts} experts, top_groups be 1 to groups, group_best 1 or 2 "
                         f"(got {groups}, {top_groups}, {group_best})")
    if k > top_groups * (experts // groups):
        raise ValueError(f"k={k} experts do not fit {top_groups} groups of {experts // groups}")
    if bias is not None and (bias.shape != (experts,) or bias.dtype is not torch.float32 or bias.device != logits.device
                             or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous float32 [{experts}] tensor on logits' device")
    weights = logits.new_empty((tokens, k), dtype=torch.float32)
    chosen = logits.new_empty((tokens, k), dtype=torch.int32)
    if tokens:
        _native.launch(logits.device, _native.library().moegemm_route_topk, logits.data_ptr(),
                       None if bias is None else bias.data_ptr(), weights.data_ptr(), chosen.data_ptr(), tokens, experts, k,
                       _row_stride(logits), code, sigmoid, groups, top_groups, group_best, int(bool(normalize)), float(scale))
    return weights, chosen


def route_topk_backward(dweights, logits, experts, *, score: str = "softmax", normalize: bool = True, scale: float = 1.0):
    """Gradient [T, E] of ``route_topk``'s logits, in their dtype, for the gradient of its weights (fp32 [T, k]).

    ``experts``: what ``route_topk`` chose (an index outside 0 to E - 1 counts for nothing; a token's are distinct).
    """
    import torch

    sigmoid = _score_flag(score)
    if experts.ndim != 2:
        raise ValueError("experts must be a 2-D [tokens, k] tensor")
    k = experts.shape[1]
    tokens, count = _check_logits(logits, k)
    code = _native.dtype_code(logits.dtype)
    device = logits.device
    for name, t, dtype in (("experts", experts, torch.int32), ("dweights", dweights, torch.float32)):
        if t.shape != (tokens, k) or t.dtype is not dtype or t.device != device or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dtype} [{tokens}, {k}] tensor on logits' device")
    dlogits = logits.new_empty((tokens, count))
    if tokens:
        _native.launch(device, _native.library().moegemm_route_topk_backward, dweights.data_ptr(), logits.data_ptr(),
                       experts.data_ptr(), dlogits.data_ptr(), tokens, count, k, _row_stride(logits), code, sigmoid,
                       int(bool(normalize)), float(scale))
    return dlogits


def sort_by_expert(experts, num_experts: int, *, first: int = 0) -> ExpertOrder:
    """Slots of ``experts`` [T, k] (int32, contiguous) sorted by expert, stably, for experts ``first`` to ``first +
    num_experts - 1`` (at most 1024); others, negative ones among them, get no row."""
    import torch

    if experts.ndim != 2 or experts.dtype is not torch.int32 or not experts.is_contiguous():
        raise ValueError("experts must be a contiguous int32 [tokens, k] tensor")
    if not experts.is_cuda:
        raise ValueError("experts must be on a GPU device")
    if not 0 < num_experts <= MAX_EXPERTS or not 0 <= first <= _native.INT32_MAX:
        raise ValueError(f"num_experts must be 1 to {MAX_EXPERTS} and first 0 to 2**31 - 1 (got {num_experts}, {first})")
    entries, lib = experts.numel(), _native.library()
    if entries > _native.INT32_MAX or experts.shape[1] == 0:
        raise ValueError(f"sort_by_expert takes 1 or more experts a token and under 2**31 in all (got {tuple(experts.shape)})")
    nbytes = lib.moegemm_sort_workspace_bytes(entries, num_experts)
    workspace = experts.new_empty((nbytes // 4,)) if nbytes else None
    offs, slots, places = experts.new_empty((num_experts,)), experts.new_empty((entries,)), torch.empty_like(experts)
    _native.launch(experts.device, lib.moegemm_sort_by_expert, experts.data_ptr(), offs.data_ptr(), slots.data_ptr(),
                   places.data_ptr(), entries, first, num_experts,
                   workspace.data_ptr() if nbytes else None, nbytes)
    return ExpertOrder(offs, slots, places)


def _check_order(order: ExpertOrder, device) -> tuple[int, int]:
    """(tokens, k) of an order on ``device``."""
    import torch

    offs, places, int32 = order.offs, order.places, torch.int32
    shape = places.shape
    if (len(shape) != 2 or places.dtype is not int32 or places.device != device or not places.is_contiguous()
            or shape[1] == 0):
        raise ValueError("order.places must be a contiguous int32 [tokens, k] tensor on the rows' device")
    if (offs.ndim != 1 or offs.dtype is not int32 or offs.device != device or not offs.is_contiguous()
            or len(offs) == 0):
        raise ValueError("order.offs must be a contiguous int32 vector on the rows' device")
    return shape


def _end_of(order: ExpertOrder) -> int:
    """Address of the last offset."""
    return order.offs.data_ptr() + 4 * (len(order.offs) - 1)


def _check_rows(name: str, t, rows: int | None, width: int | None) -> tuple[int, int]:
    """(rows, width) of a matrix whose rows the kernels can walk."""
    shape = t.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (width is not None and shape[1] != width):
        expected = ", ".join("any" if n is None else str(n) for n in (rows, width))
        raise ValueError(f"{name} must be a 2-D [{expected}] tensor (got {tuple(shape)})")
    count, columns = shape
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU device")
    if columns > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} needs a unit stride along its rows")
    if columns == 0 or (count | columns) > _native.INT32_MAX or columns * t.element_size() > _native.INT32_MAX:
        raise ValueError(f"{name} must have between 1 and 2**31 - 1 bytes a row and under 2**31 rows (got {tuple(shape)})")
    return count, columns


def gather_rows(x, order: ExpertOrder, *, rows: int | None = None):
    """Expert-sorted rows [rows, H] of the tokens ``x`` [T, H]: row ``places[t, j]`` is token t's.

    ``rows``: how many there is room for (default T * k, which holds any routing); sorted rows past it are dropped, and
    rows at or past ``offs[-1]`` are zeros.  x has any dtype of 1, 2 or 4 bytes (e4m3 rows of ``quantize_fp8`` among them)
    and unit stride along H.  Differentiable for fp16, bf16 and fp32: the gradient is ``combine_rows`` of the rows'.
    """
    import torch

    _native.refuse_tangents("gather_rows", x)
    if torch.is_grad_enabled() and x.requires_grad:
        return _functions()[1].apply(x, order, rows)
    return _gather(x, order, rows)


def _gather(x, order, rows):
    tokens, k = _check_order(order, x.device)
    _, width = _check_rows("x", x, tokens, None)
    size = x.element_size()
    if size > 4:
        raise ValueError(f"x must have elements of 1, 2 or 4 bytes (got {x.dtype})")
    rows = tokens * k if rows is None else rows
    if not 0 <= rows <= _native.INT32_MAX:
        raise ValueError(f"rows must be 0 to 2**31 - 1 (got {rows})")
    out = x.new_empty((rows, width))
    if rows:
        width *= size
        _native.launch(x.device, _native.library().moegemm_gather_rows, x.data_ptr(), out.data_ptr(), order.places.data_ptr(),
                       _end_of(order), tokens, k, rows, width, x.stride(0) * size if tokens > 1 else width, width)
    return out


def _check_weights(weights, tokens: int, k: int, device) -> None:
    import torch

    if (weights.shape != (tokens, k) or weights.dtype is not torch.float32 or weights.device != device
            or not weights.is_contiguous()):
        raise ValueError(f"weights must be a contiguous float32 [{tokens}, {k}] tensor on the rows' device")


def combine_rows(y, order: ExpertOrder, weights=None):
    """Tokens [T, H] of the expert-sorted rows ``y`` [rows, H]: ``out[t] = sum_j weights[t, j] * y[places[t, j]]``.

    Summed in fp32 in the order of j and rounded once; slots without a row (or whose row is past y's) count for nothing.
    ``weights``: contiguous fp32 [T, k], or None for ones.  y is fp16, bf16 or fp32 with unit stride along H.
    Differentiable in y and weights.
    """
    import torch

    _native.refuse_tangents("combine_rows", y, weights)
    if torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
        return _functions()[2].apply(y, weights, order)
    return _combine(y, order, weights)


def _combine(y, order, weights):
    device = y.device
    tokens, k = _check_order(order, device)
    rows, width = _check_rows("y", y, None, None)
    code = _native.dtype_code(y.dtype)
    if weights is not None:
        _check_weights(weights, tokens, k, device)
    out = y.new_empty((tokens, width))
    if tokens:
        _native.launch(device, _native.library().moegemm_combine_rows, y.data_ptr(),
                       None if weights is None else weights.data_ptr(), out.data_ptr(), order.places.data_ptr(), tokens, k,
                       rows, width, y.stride(0) if rows > 1 else width, width, code)
    return out


def combine_rows_backward(dout, y, order: ExpertOrder, weights=None, *, need_dy: bool = True, need_dweights: bool = True):
    """``(dy, dweights)`` of ``combine_rows`` for the gradient ``dout`` [T, H] of its output; None for one not needed.

    ``dy[places[t, j]] = weights[t, j] * dout[t]`` in y's dtype and shape, zeros at and past ``offs[-1]``;
    ``dweights[t, j] = <dout[t], y[places[t, j]]>`` in fp32, 0 for a slot without a row.
    """
    tokens, k = _check_order(order, y.device)
    _check_rows("y", y, None, None)
    return _combine_gradients(dout, y, order, weights, y.shape[0], need_dy, need_dweights)


def _combine_gradients(dout, y, order, weights, rows: int, need_dy: bool, need_dweights: bool):
    """The gradients; y is read for dweights only (else it may be None)."""
    import torch

    tokens, k = order.places.shape
    code = _native.dtype_code(dout.dtype)
    _check_rows("dout", dout, tokens, None if y is None else y.shape[1])
    if y is not None and (y.dtype != dout.dtype or y.device != dout.device):
        raise ValueError(f"dout must have y's dtype and device ({y.dtype}, {y.device})")
    if weights is not None:
        _check_weights(weights, tokens, k, dout.device)
    width = dout.shape[1]
    dy = dout.new_empty((rows, width)) if need_dy else None
    dweights = dout.new_empty((tokens, k), dtype=torch.float32) if need_dweights else None
    if (need_dy and rows) or (need_dweights and tokens):
        _native.launch(dout.device, _native.library().moegemm_combine_rows_backward, dout.data_ptr(),
                       y.data_ptr() if need_dweights else None, None if weights is None else weights.data_ptr(),
                       dy.data_ptr() if need_dy and rows else None, dweights.data_ptr() if need_dweights else None,
                       order.places.data_ptr(), _end_of(order), tokens, k, rows, width, _row_stride(dout),
                       _row_stride(y) if need_dweights else 0, code)
    return dy, dweights


_FUNCTIONS: list = []


def _functions():
    """The autograd functions of route_topk, gather_rows and combine_rows, made on first use (this package imports torch
    lazily)."""
    if _FUNCTIONS:
        return _FUNCTIONS
    import torch

    def dense(gradient):
        """Autograd hands out expanded and transposed gradients too."""
        return gradient if gradient.stride(-1) == 1 and (gradient.shape[0] < 2 or gradient.stride(0) >= gradient.shape[1]) \
            else gradient.clone(memory_format=torch.contiguous_format)

    class RouteTopk(torch.autograd.Function):
        @staticmethod
        def forward(ctx, logits, k, score, bias, groups, top_groups, group_best, normalize, scale):
            weights, experts = _route(logits, k, score, bias, groups, top_groups, group_best, normalize, scale)
            ctx.mark_non_differentiable(experts)
            ctx.save_for_backward(logits, experts)
            ctx.how = dict(score=score, normalize=normalize, scale=scale)
            return weights, experts

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dweights, _):
            logits, experts = ctx.saved_tensors
            return route_topk_backward(dweights.contiguous(), logits, experts, **ctx.how), *[None] * 8

    class GatherRows(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, order, rows):
            _native.dtype_code(x.dtype)  # what the gradient is summed in
            out = _gather(x, order, rows)
            ctx.save_for_backward(*order)
            return out

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, gradient):
            return _combine(dense(gradient), ExpertOrder(*ctx.saved_tensors), None), None, None

    class CombineRows(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y, weights, order):
            out = _combine(y, order, weights)
            # y is read for the weights' gradient only: where that is not needed it may change before the backward pass.
            ctx.save_for_backward(y if ctx.needs_input_grad[1] else None, weights, *order)
            ctx.rows = y.shape[0]
            return out

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dout):
            y, weights, *order = ctx.saved_tensors
            need_dy, need_dweights = ctx.needs_input_grad[:2]
            dy, dweights = _combine_gradients(dense(dout), y, ExpertOrder(*order), weights, ctx.rows, need_dy, need_dweights)
            return dy, dweights, None

    _FUNCTIONS.extend((RouteTopk, GatherRows, CombineRows))
    return _FUNCTIONS
