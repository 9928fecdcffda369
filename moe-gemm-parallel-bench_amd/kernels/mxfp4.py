"""4-bit (MXFP4) expert weights on gfx950: conversions, single and expert-sorted products with 16-bit rows, Gate+Up.

The format is the one ``model_configs/gpt-oss-120b.json`` names (mxfp4), the OCP microscaling one: e2m1 values, two a byte
with the even k in the low half, and an e8m0 byte ``s`` for each 32 along K; a value stands for ``v * 2**(s - 127)``.  Weights
are stored ``[N, K / 2]`` (``[G, N, K / 2]`` for experts) with scales ``[..., N, K / 32]``, as checkpoints store them.  Rows
stay 16-bit (fp32 ones are taken too).  The reference has no 4-bit path; this is the expert GEMM of its
kernels/torch_grouped_gemm.py:121-174 on such weights.

A serving step of one expert layer::

    q, s = quantize_mxfp4(w)                                        # once
    h = grouped_mm_mxfp4_swiglu(x, w13, s13, offs)                  # silu(gate) * up, [rows, F]
    y = grouped_mm_mxfp4(h, w2, s2, offs)                           # [rows, H]

h is rounded to x's 16 bits between the two; ``out_dtype=torch.float32`` in the first and x's in the second leaves one
rounding, at the end (256 rows over 32 experts of [7168, 2048]: 66 us for the second, of bf16 rows 53).

The products are made for decode, where an expert has few rows and reading its weights is the bound; they take any
number of rows, but past 128 an expert a bf16 copy (``dequantize_mxfp4``) and ``grouped_mm`` are faster. Gate+Up is
``silu(gate) * up`` of [gate | up] rows without a bias: an expert with biases, interleaved rows, a clamp or another
activation (gpt-oss among them) takes ``grouped_mm_mxfp4`` and its own epilogue. Each call runs on the current stream,
reads ``offs`` on the device and keeps nothing, so it can be captured in a HIP graph; repeated calls give the same bits.
Serving only: the products have no gradient, and rows that ask for one are refused. ``ValueError`` for operands a kernel
cannot take, ``RuntimeError`` without library or GPU.
"""

from __future__ import annotations

from . import _native
from .fp8 import _cu_count

MX_GROUP = 32


def _are_bytes(codes, scales) -> bool:
    """Both uint8, or torch's own types of such bytes."""
    import torch

    uint8 = torch.uint8
    return ((codes.dtype is uint8 or codes.dtype is getattr(torch, "float4_e2m1fn_x2", None))
            and (scales.dtype is uint8 or scales.dtype is getattr(torch, "float8_e8m0fnu", None)))


def _matrices(t) -> list:
    """The matrices of a 2-D or 3-D tensor: one where its rows lie evenly, else one per leading index."""
    if t.ndim == 2:
        return [t]
    if t.shape[1] == 1:
        return [t.select(1, 0)]
    if t.shape[0] == 1 or t.stride(0) == t.shape[1] * t.stride(1):
        return [t.as_strided((t.shape[0] * t.shape[1], t.shape[2]), (t.stride(1), t.stride(2)))]
    return list(t.unbind(0))


def _row_stride(t) -> int:
    """Stride between rows; of a single row, one that covers it."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def quantize_mxfp4(x):
    """``(q, scale)`` of ``x`` [..., K]: uint8 [..., K / 2] of e2m1 pairs and uint8 e8m0 [..., K / 32].

    x is [N, K] or [G, N, K], fp16, bf16 or fp32 with unit stride along K, K a multiple of 32.  For each 32 values
    ``scale = 2**(floor(log2 max|x|) - 2)``, at least 2**-127, and ``q = e2m1(x / scale)``, rounded to nearest even and at most 6; a
    group that holds a NaN or an infinity gets the scale 255, which makes all of it NaN.
    """
    import torch

    if x.ndim not in (2, 3):
        raise ValueError("quantize_mxfp4 expects a 2-D [N, K] or a 3-D [G, N, K] tensor")
    if not x.is_cuda:
        raise ValueError("x must be on a GPU device")
    code = _native.dtype_code(x.dtype)
    *head, k = x.shape
    if k <= 0 or k % MX_GROUP or k > _native.INT32_MAX:
        raise ValueError(f"K must be a positive multiple of {MX_GROUP} under 2**31 (got {k})")
    if x.stride(-1) != 1:
        raise ValueError("x needs a unit stride along its last dimension")
    q = x.new_empty((*head, k // 2), dtype=torch.uint8)
    scale = x.new_empty((*head, k // MX_GROUP), dtype=torch.uint8)
    if x.numel():
        parts = _matrices(x)
        rows = parts[0].shape[0]
        for i, part in enumerate(parts):
            _native.launch(x.device, _native.library().moegemm_quantize_mxfp4, part.data_ptr(), q.data_ptr() + i * rows * k // 2,
                           scale.data_ptr() + i * rows * k // MX_GROUP, rows, k, _row_stride(part), k // 2, k // MX_GROUP, code)
    return q, scale


def dequantize_mxfp4(q, scale, *, dtype=None):
    """The values [..., K] that ``q`` [..., K / 2] and ``scale`` [..., K / 32] stand for, in ``dtype`` (bf16 by default, exact there
    and in fp32; fp16 rounds and overflows)."""
    import torch

    dtype = torch.bfloat16 if dtype is None else dtype
    code = _native.dtype_code(dtype)
    if q.ndim not in (2, 3) or scale.ndim != q.ndim:
        raise ValueError("dequantize_mxfp4 expects q [N, K / 2] with scale [N, K / 32], or both with a leading dimension")
    *head, half = q.shape
    k = 2 * half
    _check_weight(q, scale, k)
    if not q.is_cuda or scale.device != q.device:
        raise ValueError("q and scale must be on the same GPU device")
    out = q.new_empty((*head, k), dtype=dtype)
    if q.numel():
        even = q.ndim == 2 or len(_matrices(q)) == len(_matrices(scale)) == 1
        pairs = [(_matrices(q)[0], _matrices(scale)[0])] if even else list(zip(q.unbind(0), scale.unbind(0)))
        rows = pairs[0][0].shape[0]
        for i, (part, s) in enumerate(pairs):
            _native.launch(q.device, _native.library().moegemm_dequantize_mxfp4, part.data_ptr(), s.data_ptr(),
                           out.data_ptr() + i * rows * k * out.element_size(), rows, k, _row_stride(part), _row_stride(s), code)
    return out


def _check_weight(weight, scale, k: int) -> None:
    """Shapes, types and layout of packed weights [..., K / 2] and their scales."""
    shape, strides = weight.shape, weight.stride()
    if not _are_bytes(weight, scale):
        raise ValueError("4-bit weights and their scales must be uint8 (or float4_e2m1fn_x2 and float8_e8m0fnu)")
    if k <= 0 or k % MX_GROUP or k > _native.INT32_MAX:
        raise ValueError(f"K must be a positive multiple of {MX_GROUP} under 2**31 (got {k})")
    if shape[-1] * 2 != k:
        raise ValueError(f"contraction mismatch: K={k}, weight rows hold {2 * shape[-1]}")
    expected = (*shape[:-1], k // MX_GROUP)
    if scale.shape != expected:
        raise ValueError(f"scale must be {list(expected)} (got {list(scale.shape)})")
    if strides[-1] != 1 or (k > MX_GROUP and scale.stride(-1) != 1):
        raise ValueError("weight and scale need a unit stride along K")
    if (weight.data_ptr() & 15 or (strides[-2] & 15 and shape[-2] > 1)
            or (len(shape) == 3 and strides[0] & 15 and shape[0] > 1)):
        raise ValueError("weight rows must start at multiples of 16 bytes")


def _product(entry: str, a, weight, scale, offs, out, out_dtype, variant, gated: bool):
    import torch

    if a.requires_grad and torch.is_grad_enabled():
        raise ValueError("4-bit products have no gradient: pass a.detach(), or call them under torch.no_grad()")
    _native.refuse_tangents("a 4-bit product", a)
    grouped = offs is not None
    shape = weight.shape
    if a.ndim != 2 or len(shape) != (3 if grouped else 2):
        raise ValueError("expected a 2-D a [rows, K] and " + ("a 3-D weight [G, N, K / 2]" if grouped else
                                                               "a 2-D weight [N, K / 2]"))
    rows, k = a.shape
    n, groups = shape[-2], shape[0] if grouped else 1
    _check_weight(weight, scale, k)
    a_code = _native.dtype_code(a.dtype)
    if groups <= 0 or n <= 0:
        raise ValueError("4-bit products need at least one group and a positive N")
    if rows | n | groups > _native.INT32_MAX:
        raise ValueError(f"extents must be under 2**31 (rows={rows} N={n} groups={groups})")
    if gated and n % 2:
        raise ValueError(f"packed Gate+Up width must be 2F (got {n} rows)")
    device = a.device
    if not a.is_cuda or weight.device != device or scale.device != device or (grouped and offs.device != device):
        raise ValueError("a, weight, scale and offs must be on the same GPU device")
    if grouped:
        if offs.ndim != 1 or offs.dtype is not torch.int32 or offs.shape[0] != groups:
            raise ValueError(f"offs must be an int32 vector with one entry per group ({groups})")
        if not offs.is_contiguous():
            raise ValueError("offs must be contiguous (pass offs.contiguous())")
    pitch, inner = a.stride()
    if inner != 1 or a.data_ptr() & 15 or (rows > 1 and pitch & (3 if a_code == _native.DTYPE_F32 else 7)):
        raise ValueError("a needs a unit stride along K and rows at multiples of 16 bytes")
    cols = n // 2 if gated else n
    if out is not None:
        if out_dtype is not None and out_dtype != out.dtype:
            raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
        if (out.shape != (rows, cols) or out.device != device or (out.stride(1) != 1 and cols > 1)
                or (rows > 1 and out.stride(0) < cols)):
            raise ValueError(f"out must be a [{rows}, {cols}] matrix with unit column stride on the operands' device")
        out_dtype = out.dtype
    out_dtype = out_dtype or a.dtype
    code = _native.dtype_code(out_dtype)
    if out is None:
        out = a.new_empty((rows, cols), dtype=out_dtype)
    if rows:
        _native.launch(device, getattr(_native.library(), entry), a.data_ptr(), weight.data_ptr(), scale.data_ptr(),
                       out.data_ptr(), offs.data_ptr() if grouped else None, groups, rows, n, k, pitch if rows > 1 else k,
                       weight.stride(0) if grouped and groups > 1 else 0, weight.stride(-2) if n > 1 else k // 2,
                       scale.stride(0) if grouped and groups > 1 else 0, scale.stride(-2) if n > 1 else k // MX_GROUP,
                       out.stride(0) if rows > 1 else cols, a_code, code,
                       -1 if variant is None else variant, _cu_count(device))
    return out


def matmul_mxfp4(a, weight, scale, *, out=None, out_dtype=None, variant: int | None = None):
    """``a @ dequantized(weight, scale).T``; returns ``out`` (allocated if None).

    a [M, K] is fp16, bf16 or fp32 (taken whole, below 2**-110 to within 2**-134), weight [N, K / 2] and scale [N, K / 32] uint8 as ``quantize_mxfp4`` returns them (or torch's
    float4_e2m1fn_x2 and float8_e8m0fnu).  fp32 sums; output in ``out_dtype`` (fp16, bf16 or fp32; a's by default).  M and N
    are arbitrary (under 2**30), K is a multiple of 32; rows of a and weight start at multiples of 16 bytes, less than 2**23
    bytes apart.  ``variant`` names a compiled kernel, None lets the library choose.
    """
    return _product("moegemm_grouped_mm_mxfp4", a, weight, scale, None, out, out_dtype, variant, False)


def grouped_mm_mxfp4(a, weight, scale, offs, *, out=None, out_dtype=None, variant: int | None = None):
    """``matmul_mxfp4`` of each group of expert-sorted rows with its own weight [G, N, K / 2]; returns ``out`` [rows, N].

    Group e owns rows offs[e-1]:offs[e] (int32 end rows on the device), as in ``grouped_mm``: rows at or past
    offs[-1] are not written and offsets beyond ``rows`` are clamped.
    """
    if offs is None:
        raise ValueError("grouped_mm_mxfp4 needs offs (matmul_mxfp4 takes one weight)")
    return _product("moegemm_grouped_mm_mxfp4", a, weight, scale, offs, out, out_dtype, variant, False)


def grouped_mm_mxfp4_swiglu(a, weight, scale, offs=None, *, out=None, out_dtype=None, variant: int | None = None):
    """Packed Gate+Up with silu(gate) * up in fp32 in the epilogue; returns ``out`` [rows, F].

    ``weight`` [G, 2F, K / 2] holds each group's [gate | up] rows (without ``offs``: [2F, K / 2], one group).  Operands, offsets
    and output as in ``grouped_mm_mxfp4``.
    """
    return _product("moegemm_grouped_mm_mxfp4_swiglu", a, weight, scale, offs, out, out_dtype, variant, True)
