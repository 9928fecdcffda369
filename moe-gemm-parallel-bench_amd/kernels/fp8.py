"""Block-scaled fp8 (e4m3) products on gfx950: quantisation, single and expert-sorted GEMMs, fused Gate+Up.

The format is the one ``model_configs/deepseek-v3.json`` names: activations carry one fp32 scale for each 1 x 128
run of a row, weights one for each 128 x 128 block, and a value stands for ``q * scale``.  Weights are stored
``[N, K]`` (``[G, N, K]`` for experts), as linear layers and checkpoints store them.  The reference has no 8-bit
path; this is the expert GEMM of its kernels/torch_grouped_gemm.py:121-174 on those operands.

A serving step of one expert layer::

    q, s = quantize_fp8(x)                                          # [rows, H] expert-sorted activations
    h, hs = grouped_mm_fp8_swiglu(q, s, w13, w13_scale, offs)       # silu(gate) * up, quantised again
    y = grouped_mm_fp8(h, hs, w2, w2_scale, offs)                   # [rows, H] bf16

Each call runs on the current stream, reads ``offs`` on the device and keeps nothing, so it can be captured in a HIP
graph.  It is one kernel launch, and another for every further 2**24 workgroups of a quantisation, 768 groups or 192
rounds of tiles of a product.  ``ValueError`` for operands a kernel cannot take, ``RuntimeError`` without library or GPU.
"""

from __future__ import annotations

from functools import lru_cache

from . import _native
from .matmul import _device_signature

SCALE_BLOCK = 128


def _blocks(extent: int) -> int:
    return -(-extent // SCALE_BLOCK)


@lru_cache(maxsize=None)
def _cu_count(device) -> int:
    return _device_signature(device) % 1000


def quantize_fp8(x, *, block_rows: int = 1, out=None, scale=None):
    """e4m3 values and fp32 scales of ``x`` [..., K]; returns ``(q, scale)``.

    ``block_rows=1`` (activations): x [rows, K], scale [rows, ceil(K / 128)], one scale for each run of 128 columns;
    ``block_rows=128`` (weights): x [N, K] or [G, N, K], scale [..., ceil(N / 128), ceil(K / 128)].  For each block
    ``amax = max(max|x|, 2**-96)``, ``scale = amax / 448`` and ``q = e4m3(x * (448 / amax))``, rounded to nearest even;
    a block that holds a NaN or an infinity becomes NaN.  x is fp16, bf16 or fp32 with unit stride along K.
    q's rows are padded to multiples of 16 bytes, as the products need them, and activation scales have unit
    stride along the rows, which is what they read fastest.
    """
    import torch

    if block_rows not in (1, SCALE_BLOCK):
        raise ValueError(f"block_rows must be 1 or {SCALE_BLOCK}, got {block_rows!r}")
    shape = x.shape
    if len(shape) not in (2, 3):
        raise ValueError("quantize_fp8 expects a 2-D [rows, K] or a 3-D [G, rows, K] tensor")
    *head, rows, k = shape
    batch = head[0] if head else 1
    if rows | k | batch > _native.INT32_MAX:
        raise ValueError(f"x's extents must be under 2**31 (got {tuple(shape)})")
    if x.device.type != "cuda":
        raise ValueError("x must be on a GPU device")
    code = _native.dtype_code(x.dtype)
    if k <= 0:
        raise ValueError("quantize_fp8 needs a positive K")
    if x.stride(-1) != 1 and k > 1:
        raise ValueError("x needs a unit stride along its last dimension")
    scale_shape = (*head, -(-rows // block_rows), _blocks(k))
    if out is None:
        pitch = -(-k // 16) * 16
        buffer = torch.empty((*head, rows, pitch), dtype=torch.float8_e4m3fn, device=x.device)
        out = buffer if pitch == k else buffer[..., :k]
    elif (out.shape != shape or out.dtype != torch.float8_e4m3fn or out.device != x.device
          or (out.stride(-1) != 1 and k > 1) or out.data_ptr() % 8
          or (rows > 1 and (out.stride(-2) % 8 or out.stride(-2) < k)) or (batch > 1 and out.stride(0) % 8)):
        raise ValueError(f"out must be a {tuple(shape)} float8_e4m3fn tensor on x's device whose rows start at "
                         "multiples of 8 bytes")
    if scale is None:
        if block_rows == 1:
            blocks = scale_shape[-1]
            strides = (blocks * rows, 1, rows) if head else (1, rows)
            scale = torch.empty_strided(scale_shape, strides, dtype=torch.float32, device=x.device)
        else:
            scale = torch.empty(scale_shape, dtype=torch.float32, device=x.device)
    elif tuple(scale.shape) != scale_shape or scale.dtype != torch.float32 or scale.device != x.device:
        raise ValueError(f"scale must be a {scale_shape} float32 tensor on x's device")
    xs, qs, ss = x.stride(), out.stride(), scale.stride()
    three = batch > 1  # a stride that is not walked may be anything
    status = _native.library().moegemm_quantize_fp8(
        x.data_ptr(), out.data_ptr(), scale.data_ptr(), batch, rows, k, xs[0] if three else 0, xs[-2],
        qs[0] if three else 0, qs[-2] if rows > 1 else -(-k // 8) * 8, ss[0] if three else 0, ss[-2], ss[-1], code,
        block_rows, _native.current_stream_handle(x.device))
    _native.check(status)
    return out, scale


def _validate(a, scale_a, weight, scale_w, offs):
    """Checks shared by the products; returns (rows, n, k, groups)."""
    import torch

    grouped = offs is not None
    if a.ndim != 2 or weight.ndim != (3 if grouped else 2):
        raise ValueError("expected a 2-D a [rows, K] and " + ("a 3-D weight [G, N, K]" if grouped else
                                                               "a 2-D weight [N, K]"))
    rows, k = a.shape
    *head, n, width = weight.shape
    groups = head[0] if grouped else 1
    if width != k:
        raise ValueError(f"contraction mismatch: a K={k}, weight K={width}")
    if a.dtype != torch.float8_e4m3fn or weight.dtype != torch.float8_e4m3fn:
        raise ValueError("a and weight must be float8_e4m3fn")
    if groups <= 0 or n <= 0 or k <= 0:
        raise ValueError("fp8 products need at least one group and positive K and N")
    if rows | n | k | groups > _native.INT32_MAX:
        raise ValueError(f"extents must be under 2**31 (rows={rows} N={n} K={k} groups={groups})")
    if scale_a.shape != (rows, _blocks(k)) or scale_a.dtype is not torch.float32:
        raise ValueError(f"scale_a must be a float32 [{rows}, {_blocks(k)}] tensor")
    expected = (groups, _blocks(n), _blocks(k)) if grouped else (_blocks(n), _blocks(k))
    if scale_w.shape != expected or scale_w.dtype is not torch.float32:
        raise ValueError(f"scale_w must be a float32 {list(expected)} tensor")
    device = a.device
    if (not a.is_cuda or weight.device != device or scale_a.device != device or scale_w.device != device
            or (grouped and offs.device != device)):
        raise ValueError("operands, scales and offs must be on the same GPU device")
    if grouped:
        if offs.ndim != 1 or offs.dtype != torch.int32 or offs.shape[0] != groups:
            raise ValueError(f"offs must be an int32 vector with one entry per group ({groups})")
        if not offs.is_contiguous():
            raise ValueError("offs must be contiguous (pass offs.contiguous())")
    for name, t in (("a", a), ("weight", weight)):
        strides, shape = t.stride(), t.shape
        if strides[-1] != 1 and k > 1:
            raise ValueError(f"{name} needs a unit stride along K")
        if (t.data_ptr() & 15 or (strides[-2] & 15 and shape[-2] > 1)
                or (len(shape) == 3 and strides[0] & 15 and shape[0] > 1)):
            raise ValueError(f"{name} rows must start at multiples of 16 bytes (quantize_fp8 pads them so)")
    return rows, n, k, groups


def _pitch(tensor, width: int) -> int:
    """Row stride of a matrix (any one that covers a row, where there is a single row)."""
    return tensor.stride(-2) if tensor.shape[-2] > 1 else -(-width // 16) * 16


def _operand_args(a, scale_a, weight, scale_w, k: int):
    grouped = weight.ndim == 3
    sa, sw = scale_a.stride(), scale_w.stride()
    return (a.shape[0], weight.shape[-2], k, _pitch(a, k), sa[0], sa[1],
            weight.stride(0) if grouped and weight.shape[0] > 1 else 0, _pitch(weight, k), sw[0] if grouped else 0,
            sw[-2], sw[-1])


def _product(a, scale_a, weight, scale_w, offs, out, out_dtype, fast_accum, variant):
    import torch

    rows, n, k, groups = _validate(a, scale_a, weight, scale_w, offs)
    if out is not None:
        if out_dtype is not None and out_dtype != out.dtype:
            raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
        out_dtype = out.dtype
    out_dtype = out_dtype or torch.bfloat16
    code = _native.dtype_code(out_dtype)
    if out is None:
        out = torch.empty((rows, n), dtype=out_dtype, device=a.device)
    elif tuple(out.shape) != (rows, n) or out.device != a.device or (out.stride(1) != 1 and n > 1):
        raise ValueError(f"out must be a [{rows}, {n}] matrix with unit column stride on the operands' device")
    if rows == 0:
        return out
    status = _native.library().moegemm_grouped_mm_fp8(
        a.data_ptr(), scale_a.data_ptr(), weight.data_ptr(), scale_w.data_ptr(), out.data_ptr(),
        offs.data_ptr() if offs is not None else None, groups, *_operand_args(a, scale_a, weight, scale_w, k),
        out.stride(0) if rows > 1 else n, code, int(bool(fast_accum)), -1 if variant is None else variant,
        _cu_count(a.device), _native.current_stream_handle(a.device))
    _native.check(status)
    return out


def matmul_fp8(a, scale_a, weight, scale_w, *, out=None, out_dtype=None, fast_accum: bool = False,
               variant: int | None = None):
    """``(a * scale_a) @ (weight * scale_w).T`` of block-quantised operands; returns ``out`` (allocated if None).

    a [M, K] and scale_a [M, ceil(K / 128)], weight [N, K] and scale_w [ceil(N / 128), ceil(K / 128)]; fp32 sums,
    output in ``out_dtype`` (bf16 by default; fp16 and fp32 too).  M, N and K are arbitrary; rows of a and weight
    start at multiples of 16 bytes, less than 2**23 bytes apart.  By default every sum is fp32.  ``fast_accum=True`` lets
    the 8-bit matrix instructions sum inside a block of 128, at twice the rate, with sums of eight products that keep
    about 14 bits below the largest.  It takes effect above 32 rows of one weight and above a mean of 20 rows a group;
    calls with fewer rows are bound by reading the weights and keep fp32 sums.  ``variant`` names a compiled kernel,
    None lets the library choose.
    """
    return _product(a, scale_a, weight, scale_w, None, out, out_dtype, fast_accum, variant)


def grouped_mm_fp8(a, scale_a, weight, scale_w, offs, *, out=None, out_dtype=None, fast_accum: bool = False,
                   variant: int | None = None):
    """``matmul_fp8`` of each group of expert-sorted rows with its own weight [G, N, K]; returns ``out`` [rows, N].

    Group e owns rows offs[e-1]:offs[e] (int32 end rows on the device), as in ``grouped_mm``: rows at or past
    offs[-1] are not written and offsets beyond ``rows`` are clamped.
    """
    if offs is None:
        raise ValueError("grouped_mm_fp8 needs offs (matmul_fp8 takes one weight)")
    return _product(a, scale_a, weight, scale_w, offs, out, out_dtype, fast_accum, variant)


def grouped_mm_fp8_swiglu(a, scale_a, weight, scale_w, offs=None, *, fast_accum: bool = False,
                          variant: int | None = None):
    """Packed Gate+Up in fp8 with silu(gate) * up quantised in the epilogue; returns ``(q, scale)``.

    ``weight`` [G, 2F, K] holds each group's [gate | up] rows (without ``offs``: [2F, K], one group); F is a multiple
    of 8.  q [rows, F] and scale [rows, ceil(F / 128)] are what ``quantize_fp8`` makes of the fp32 activations, laid
    out as it does, so they go straight into the down projection.  Offsets as in ``grouped_mm_fp8``.
    """
    import torch

    rows, n, k, groups = _validate(a, scale_a, weight, scale_w, offs)
    if n % 16:
        raise ValueError(f"packed Gate+Up width must be 2F with F a multiple of 8 (got {n} rows)")
    f = n // 2
    pitch = -(-f // 16) * 16
    buffer = torch.empty((rows, pitch), dtype=torch.float8_e4m3fn, device=a.device)
    out = buffer if pitch == f else buffer[:, :f]
    scale = torch.empty((_blocks(f), rows), dtype=torch.float32, device=a.device).t()
    if rows == 0:
        return out, scale
    status = _native.library().moegemm_grouped_mm_fp8_swiglu(
        a.data_ptr(), scale_a.data_ptr(), weight.data_ptr(), scale_w.data_ptr(), out.data_ptr(), scale.data_ptr(),
        offs.data_ptr() if offs is not None else None, groups, *_operand_args(a, scale_a, weight, scale_w, k),
        pitch, scale.stride(0), scale.stride(1), int(bool(fast_accum)), -1 if variant is None else variant,
        _cu_count(a.device), _native.current_stream_handle(a.device))
    _native.check(status)
    return out, scale
