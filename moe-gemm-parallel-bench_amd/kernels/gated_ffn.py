"""Training form of the packed Gate+Up block over expert-sorted rows on gfx950: forward and backward.

``h = silu(x W_gate) * (x W_up)`` per expert, with W [G, H, 2F] = [gate | up] as ``grouped_mm_swiglu`` takes it.
The forward pass is one launch that also keeps the projections [g | u] in fp32; the backward pass is three: the
elementwise gradient of [g | u], then ``dx`` and ``dW`` (each product launches again for every further 768 groups or 192
rounds of tiles).  The reference times the forward GEMMs only (README.md:55-57).

``gate_up_swiglu`` is the differentiable call; ``gate_up_swiglu_forward`` and ``gate_up_swiglu_backward`` are
its two halves for programs that run their own backward pass.  Offsets are read on the device at run time, calls run
on the current stream, and repeated calls give the same bits.  ``ValueError`` for operands the kernels cannot take,
``RuntimeError`` without library or GPU.
"""

from __future__ import annotations

from . import _native
from .fp8 import _cu_count

_PITCH_LIMIT = 1 << 22  # elements between rows: 256 rows of a tile span under 2 GiB


def _rows_ok(tensor) -> bool:
    """Unit inner stride and rows at multiples of 16 bytes."""
    strides, shape = tensor.stride(), tensor.shape
    return (strides[-1] == 1 and not tensor.data_ptr() & 15 and not (strides[-2] & 7 and shape[-2] > 1)
            and not (len(shape) == 3 and strides[0] & 7 and shape[0] > 1))


def _validate(x, weight, offs):
    """(rows, H, F, groups) of the block's operands."""
    import torch

    grouped = offs is not None
    shape = weight.shape
    if x.ndim != 2 or len(shape) != (3 if grouped else 2):
        raise ValueError("expected a 2-D x [rows, H] and " + ("a 3-D weight [G, H, 2F]" if grouped else
                                                               "a 2-D weight [H, 2F]"))
    rows, h = x.shape
    groups = shape[0] if grouped else 1
    if shape[-2] != h:
        raise ValueError(f"contraction mismatch: x H={h}, weight H={shape[-2]}")
    dtype, device = x.dtype, x.device
    if (dtype is not torch.float16 and dtype is not torch.bfloat16) or weight.dtype is not dtype:
        raise ValueError("x and weight must both be fp16 or bf16")
    if groups <= 0 or h <= 0 or h % 8 or shape[-1] <= 0 or shape[-1] % 16:
        raise ValueError(f"H and F must be positive multiples of 8 (H={h}, packed width {shape[-1]})")
    if rows | h | shape[-1] | groups > _native.INT32_MAX:
        raise ValueError(f"extents must be under 2**31 (rows={rows} H={h} packed width {shape[-1]} groups={groups})")
    if not x.is_cuda or weight.device != device or (grouped and offs.device != device):
        raise ValueError("x, weight and offs must be on the same GPU device")
    if grouped:
        if offs.ndim != 1 or offs.dtype is not torch.int32 or offs.shape[0] != groups:
            raise ValueError(f"offs must be an int32 vector with one entry per group ({groups})")
        if not offs.is_contiguous():
            raise ValueError("offs must be contiguous (pass offs.contiguous())")
    for name, t in (("x", x), ("weight", weight)):
        if not _rows_ok(t):
            raise ValueError(f"{name} needs a unit inner stride and rows at multiples of 16 bytes")
    return rows, h, shape[-1] // 2, groups


def _pitch(tensor) -> int:
    """Row stride (of a single row, any that covers it)."""
    return tensor.stride(-2) if tensor.shape[-2] > 1 else tensor.shape[-1]


def _group_stride(weight) -> int:
    return weight.stride(0) if weight.ndim == 3 and weight.shape[0] > 1 else 0


def gate_up_swiglu_forward(x, weight, offs=None, *, variant: int | None = None):
    """``(h, saved)``: h [rows, F] = silu(x @ W[:, :F]) * (x @ W[:, F:]) and the fp32 projections saved [rows, 2F].

    x is expert-sorted [rows, H]; weight [G, H, 2F] with int32 end rows ``offs`` [G] on the device, or [H, 2F] without.
    fp16 or bf16, H and F multiples of 8, rows at multiples of 16 bytes, less than 2**23 bytes apart; a group's weight
    spans less than 2 GiB.  Rows at or past offs[-1] get h = 0; their
    saved values are unspecified.
    """
    return _forward(x, weight, offs, variant, True)


def _forward(x, weight, offs, variant, keep: bool):
    """``gate_up_swiglu_forward``; without ``keep`` nothing but h is written (and None returned for the projections)."""
    import torch

    rows, h, f, groups = _validate(x, weight, offs)
    lib, device = _native.library(), x.device
    out = x.new_empty((rows, f))
    saved = x.new_empty((rows, 2 * f), dtype=torch.float32) if keep else None
    if rows:
        _native.check(lib.moegemm_gate_up_forward(
            x.data_ptr(), weight.data_ptr(), out.data_ptr(), saved.data_ptr() if keep else None,
            None if offs is None else offs.data_ptr(), groups, rows, h, f, _pitch(x), _group_stride(weight),
            _pitch(weight), f, _native.dtype_code(x.dtype), -1 if variant is None else variant, _cu_count(device),
            _native.current_stream_handle(device)))
    return out, saved


def gate_up_swiglu_backward(dh, x, weight, offs, saved, *, need_dx: bool = True, need_dw: bool = True,
                            variants: tuple[int, int] | None = None):
    """``(dx, dw)`` of ``gate_up_swiglu_forward`` for the gradient dh [rows, F] of its h; None for one not needed.

    The gradient of [g | u] is rounded once to the operand type before the two products.  dx [rows, H] is zero past
    offs[-1], dw [G, H, 2F] (or [H, 2F]) is zero for an expert without rows.
    """
    import torch

    rows, h, f, groups = _validate(x, weight, offs)
    if dh.shape != (rows, f) or dh.dtype is not x.dtype or dh.device != x.device:
        raise ValueError(f"dh must be a [{rows}, {f}] {x.dtype} matrix on x's device")
    if (saved.shape != (rows, 2 * f) or saved.dtype is not torch.float32 or saved.device != x.device
            or not saved.is_contiguous()):
        raise ValueError(f"saved must be the contiguous [{rows}, {2 * f}] float32 tensor of the forward pass")
    return _gradients(dh, x, weight, offs, saved, rows, h, f, groups, weight.shape, variants, need_dx, need_dw)


def _gradients(dh, x, weight, offs, saved, rows: int, h: int, f: int, groups: int, weight_shape, variants, need_dx: bool,
               need_dw: bool):
    """(dx, dw) of checked operands; x is read for dw only, weight for dx only (else they may be None)."""
    device = dh.device
    pitch, inner = dh.stride()
    if inner != 1 or dh.data_ptr() & 15 or (rows > 1 and (pitch & 7 or not f <= pitch < _PITCH_LIMIT)):
        # Autograd hands out expanded and transposed gradients, slices of wide ones, and dense views at any offset, which
        # contiguous() returns.
        import torch

        dh = dh.clone(memory_format=torch.contiguous_format)
        pitch = f
    lib = _native.library()
    dx_variant, dw_variant = variants or (-1, -1)
    dp = dh.new_empty((rows, 2 * f))
    dx = dh.new_empty((rows, h)) if need_dx else None
    dw = dh.new_empty(weight_shape) if need_dw else None
    _native.check(lib.moegemm_gate_up_backward(
        dh.data_ptr(), x.data_ptr() if need_dw else None, weight.data_ptr() if need_dx else None, saved.data_ptr(),
        dp.data_ptr(), dx.data_ptr() if need_dx else None, dw.data_ptr() if need_dw else None,
        None if offs is None else offs.data_ptr(), groups, rows, h, f, pitch if rows > 1 else f,
        _pitch(x) if need_dw else 0, _group_stride(weight) if need_dx else 0, _pitch(weight) if need_dx else 0,
        _native.dtype_code(dh.dtype), dx_variant, dw_variant, _cu_count(device), _native.current_stream_handle(device)))
    return dx, dw


def gate_up_swiglu(x, weight, offs=None):
    """Differentiable h [rows, F] = silu(x @ W_gate) * (x @ W_up) per expert (``gate_up_swiglu_forward``'s operands).

    The projections are kept only where a gradient is to come: grad mode is on and x or weight requires one.
    """
    import torch

    if not (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)):
        return _forward(x, weight, offs, None, False)[0]
    return _function().apply(x, weight, offs)


_FUNCTION: list = []


def _function():
    """The autograd function, made on first use (this package imports torch lazily)."""
    if _FUNCTION:
        return _FUNCTION[0]
    import torch

    class GateUpSwiglu(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, offs):
            h, saved = gate_up_swiglu_forward(x, weight, offs)
            need_dx, need_dw = ctx.needs_input_grad[:2]
            # x is read for dW and the weight for dx: what is not kept may change before the backward pass.
            ctx.save_for_backward(saved, x if need_dw else None, weight if need_dx else None, offs)
            ctx.sizes = (*x.shape, h.shape[1], 1 if offs is None else weight.shape[0], weight.shape)
            return h

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dh):
            saved, x, weight, offs = ctx.saved_tensors
            return (*_gradients(dh, x, weight, offs, saved, *ctx.sizes, None, *ctx.needs_input_grad[:2]), None)

    _FUNCTION.append(GateUpSwiglu)
    return GateUpSwiglu
