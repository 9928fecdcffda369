"""CPU tests of the 4-bit operators' argument checks, in Python and at the C boundary."""

from __future__ import annotations

import pytest
import torch

from kernels import (
    _native,
    dequantize_mxfp4,
    grouped_mm_mxfp4,
    grouped_mm_mxfp4_swiglu,
    matmul_mxfp4,
    quantize_mxfp4,
)

U8, BF16 = torch.uint8, torch.bfloat16


@pytest.mark.parametrize("x,match", [(torch.zeros(4, 64), "GPU"), (torch.zeros(64), "2-D")])
def test_quantize_refuses_what_it_cannot_take(x, match):
    with pytest.raises(ValueError, match=match):
        quantize_mxfp4(x)


@pytest.mark.parametrize("q,scale,match", [
    (torch.zeros(4, 32, dtype=U8), torch.zeros(4, 2, dtype=U8), "GPU"), (torch.zeros(4, 32), torch.zeros(4, 2, dtype=U8), "uint8"),
    (torch.zeros(4, 32, dtype=U8), torch.zeros(4, 2), "uint8"), (torch.zeros(4, 32, dtype=U8), torch.zeros(4, 3, dtype=U8), "scale"),
    (torch.zeros(4, 24, dtype=U8), torch.zeros(4, 1, dtype=U8), "multiple of 32"),
    (torch.zeros(32, dtype=U8), torch.zeros(2, dtype=U8), "expects"),
    (torch.zeros(4, 32, dtype=U8), torch.zeros(1, 4, 2, dtype=U8), "expects"),
    (torch.zeros(32, 4, dtype=U8).t(), torch.zeros(4, 2, dtype=U8), "unit stride"),
])
def test_dequantize_refuses_what_it_cannot_take(q, scale, match):
    with pytest.raises(ValueError, match=match):
        dequantize_mxfp4(q, scale)


def test_dequantize_refuses_other_types():
    with pytest.raises(ValueError, match="dtype"):
        dequantize_mxfp4(torch.zeros(4, 32, dtype=U8), torch.zeros(4, 2, dtype=U8), dtype=torch.float64)


@pytest.mark.parametrize("change,match", [
    (dict(), "GPU"), (dict(a=torch.zeros(3, 64, dtype=torch.float64)), "dtype"), (dict(a=torch.zeros(3, 96, dtype=BF16)), "contraction"),
    (dict(a=torch.zeros(64, dtype=BF16)), "2-D"), (dict(w=torch.zeros(2, 8, 32)), "uint8"),
    (dict(w=torch.zeros(8, 32, dtype=U8)), "3-D"), (dict(s=torch.zeros(2, 8, 3, dtype=U8)), "scale"),
    (dict(a=torch.zeros(3, 48, dtype=BF16), w=torch.zeros(2, 8, 24, dtype=U8)), "multiple of 32"),
    (dict(w=torch.zeros(0, 8, 32, dtype=U8), s=torch.zeros(0, 8, 2, dtype=U8)), "group"),
    (dict(w=torch.zeros(2, 0, 32, dtype=U8), s=torch.zeros(2, 0, 2, dtype=U8)), "group"),
    (dict(w=torch.zeros(2, 8, 40, dtype=U8)[:, :, 8:]), "16 bytes"), (dict(w=torch.zeros(2, 8, 41, dtype=U8)[:, :, :32]), "16 bytes"),
    (dict(s=torch.zeros(2, 2, 8, dtype=U8).transpose(1, 2)), "unit stride"),
])
def test_products_refuse_what_they_cannot_take(change, match):
    args = dict(a=torch.zeros(3, 64, dtype=BF16), w=torch.zeros(2, 8, 32, dtype=U8), s=torch.zeros(2, 8, 2, dtype=U8)) | change
    for product in (grouped_mm_mxfp4, grouped_mm_mxfp4_swiglu):
        with pytest.raises(ValueError, match=match):
            product(args["a"], args["w"], args["s"], torch.zeros(2, dtype=torch.int32))


def test_missing_offsets_and_odd_gate_up_widths():
    a, s = torch.zeros(3, 64, dtype=BF16), torch.zeros(2, 9, 2, dtype=U8)
    w = torch.zeros(2, 9, 32, dtype=U8)
    with pytest.raises(ValueError, match="needs offs"):
        grouped_mm_mxfp4(a, w, s, None)
    with pytest.raises(ValueError, match="2F"):
        grouped_mm_mxfp4_swiglu(a, w, s, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        matmul_mxfp4(a, w[0], s[0])


def _product(gated=False, **changes):
    v = dict(a=4096, w=4096, s=4096, out=4096, offs=4096, groups=2, rows=4, n=16, k=64, lda=64, swg=512, ldw=32, ssg=32, ssn=2, ldo=16,
             dtype=_native.DTYPE_BF16, out_dtype=_native.DTYPE_BF16, variant=-1) | changes
    lib = _native.library()
    entry = lib.moegemm_grouped_mm_mxfp4_swiglu if gated else lib.moegemm_grouped_mm_mxfp4
    return entry(v["a"], v["w"], v["s"], v["out"], v["offs"], v["groups"], v["rows"], v["n"], v["k"], v["lda"], v["swg"], v["ldw"],
                 v["ssg"], v["ssn"], v["ldo"], v["dtype"], v["out_dtype"], v["variant"], 256, None)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("changes", [
    dict(dtype=7), dict(out_dtype=4), dict(lda=1 << 22), dict(dtype=_native.DTYPE_F32, lda=66), dict(groups=0), dict(offs=None), dict(rows=-1), dict(n=0), dict(k=0), dict(k=48),
    dict(a=None), dict(w=None), dict(s=None), dict(out=None), dict(a=4104), dict(w=4104), dict(lda=68), dict(lda=-8), dict(ldw=24),
    dict(ldw=40), dict(swg=520), dict(ssn=1), dict(ldo=7), dict(out=4097), dict(groups=1 << 20, n=1 << 20, rows=1 << 21, ldo=1 << 20)])
def test_product_entries_refuse(gated, changes):
    assert _product(gated, **changes) == _native.ERR_INVALID
    assert _native.last_error()


def test_variants_and_empty_calls():
    count = _native.library().moegemm_mxfp4_variant_count()
    assert count >= 2
    for gated in (False, True):
        assert _product(gated, variant=count) == _native.ERR_NO_KERNEL
        assert _product(gated, variant=-2) == _native.ERR_NO_KERNEL
        assert _product(gated, rows=0) == _native.OK
    assert _product(True, n=15) == _native.ERR_INVALID


def test_conversion_entries_refuse():
    lib = _native.library()
    bad = [
        lib.moegemm_quantize_mxfp4(4096, 4096, 4096, 4, 48, 48, 24, 2, 2, None), lib.moegemm_quantize_mxfp4(4096, 4096, 4096, 4, 0, 0, 0, 0, 2, None),
        lib.moegemm_quantize_mxfp4(4096, 4096, 4096, -1, 64, 64, 32, 2, 2, None), lib.moegemm_quantize_mxfp4(4096, 4096, 4096, 4, 64, 64, 32, 2, 9, None),
        lib.moegemm_quantize_mxfp4(None, 4096, 4096, 4, 64, 64, 32, 2, 2, None), lib.moegemm_quantize_mxfp4(4096, 4098, 4096, 4, 64, 64, 32, 2, 2, None),
        lib.moegemm_quantize_mxfp4(4098, 4096, 4096, 4, 64, 64, 32, 2, 2, None), lib.moegemm_quantize_mxfp4(4096, 4096, 4096, 4, 64, 64, 34, 2, 2, None),
        lib.moegemm_dequantize_mxfp4(4096, None, 4096, 4, 64, 32, 2, 2, None), lib.moegemm_dequantize_mxfp4(4096, 4096, 4104, 4, 64, 32, 2, 2, None),
        lib.moegemm_dequantize_mxfp4(4096, 4096, 4096, 4, 80, 40, 2, 2, None),
    ]
    assert bad == [_native.ERR_INVALID] * len(bad)
    assert lib.moegemm_quantize_mxfp4(None, None, None, 0, 64, 64, 32, 2, 2, None) == _native.OK
    assert lib.moegemm_dequantize_mxfp4(None, None, None, 0, 64, 32, 2, 2, None) == _native.OK
