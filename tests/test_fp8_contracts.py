"""CPU tests of the fp8 operators' argument checks, in Python and at the C boundary."""

from __future__ import annotations

import pytest
import torch

from kernels import _native, grouped_mm_fp8, grouped_mm_fp8_swiglu, matmul_fp8, quantize_fp8

E4M3 = torch.float8_e4m3fn


def _fp8(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(E4M3)


def test_quantize_refuses_what_it_cannot_take():
    with pytest.raises(ValueError, match="block_rows"):
        quantize_fp8(torch.zeros(4, 128), block_rows=64)
    with pytest.raises(ValueError, match="2-D"):
        quantize_fp8(torch.zeros(128))
    with pytest.raises(ValueError, match="GPU"):
        quantize_fp8(torch.zeros(4, 128))


@pytest.mark.parametrize("change,match", [
    (dict(a=_fp8(4, 64)), "contraction"), (dict(a=torch.zeros(4, 128)), "float8"), (dict(a=_fp8(4, 2, 128)), "2-D"),
    (dict(sa=torch.ones(4, 2)), "scale_a"), (dict(sa=torch.ones(4, 1).double()), "scale_a"),
    (dict(sw=torch.ones(2, 1)), "scale_w"), (dict(w=_fp8(2, 32, 128)), "weight"), (dict(), "GPU"),
])
def test_matmul_refuses_what_it_cannot_take(change, match):
    args = dict(a=_fp8(4, 128), sa=torch.ones(4, 1), w=_fp8(32, 128), sw=torch.ones(1, 1)) | change
    with pytest.raises(ValueError, match=match):
        matmul_fp8(args["a"], args["sa"], args["w"], args["sw"])


def test_grouped_refuses_missing_offsets():
    with pytest.raises(ValueError, match="offs"):
        grouped_mm_fp8(_fp8(4, 128), torch.ones(4, 1), _fp8(2, 32, 128), torch.ones(2, 1, 1), None)
    with pytest.raises(ValueError, match="GPU"):
        grouped_mm_fp8_swiglu(_fp8(4, 128), torch.ones(4, 1), _fp8(2, 24, 128), torch.ones(2, 1, 1),
                              torch.zeros(2, dtype=torch.int32))


def _product(gated=False, **changes):
    args = dict(a=4096, sa=4096, w=4096, sw=4096, out=4096, scale=4096, offs=4096, groups=2, rows=4, n=64, k=128,
                lda=128, sam=1, sak=4, swg=8192, ldw=128, ssg=1, ssn=1, ssk=1, ldo=64, osm=1, osk=4,
                dtype=_native.DTYPE_BF16, variant=-1, fast=0)
    args.update(changes)
    v = args
    lib = _native.library()
    head = (v["a"], v["sa"], v["w"], v["sw"], v["out"])
    tail = (v["offs"], v["groups"], v["rows"], v["n"], v["k"], v["lda"], v["sam"], v["sak"], v["swg"], v["ldw"],
            v["ssg"], v["ssn"], v["ssk"], v["ldo"])
    if gated:
        return lib.moegemm_grouped_mm_fp8_swiglu(*head, v["scale"], *tail, v["osm"], v["osk"], v["fast"], v["variant"], 256, None)
    return lib.moegemm_grouped_mm_fp8(*head, *tail, v["dtype"], v["fast"], v["variant"], 256, None)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("changes,match", [
    (dict(groups=0), "group_count"), (dict(offs=None), "one group"), (dict(rows=-1), "shape"), (dict(n=0), "shape"),
    (dict(k=0), "shape"), (dict(a=None), "non-null"), (dict(sw=None), "non-null"), (dict(a=4100), "16 bytes"),
    (dict(lda=136), "16 bytes"), (dict(swg=8200), "16 bytes"), (dict(lda=112), "cover"), (dict(ldo=8), "cover"),
    (dict(ldw=1 << 23), "under"), (dict(sam=-1), "scale strides"), (dict(sam=1 << 22), "scale strides"),
    (dict(fast=2), "fast_accum"),
])
def test_c_entries_refuse_before_any_launch(gated, changes, match):
    assert _product(gated, **changes) == _native.ERR_INVALID
    assert match in _native.last_error()


def test_c_entries_refuse_unknown_variants_and_types():
    assert _product(dtype=9) == _native.ERR_INVALID and "dtype" in _native.last_error()
    for gated in (False, True):
        count = _native.library().moegemm_fp8_variant_count(1 if gated else 0)
        assert count > 0
        assert _product(gated, variant=count) == _native.ERR_NO_KERNEL and "variant" in _native.last_error()
        assert _product(gated, rows=0) == _native.OK
    assert _product(True, n=72, ldo=72) == _native.ERR_INVALID and "multiple of 16" in _native.last_error()
    assert _product(True, scale=None) == _native.ERR_INVALID


@pytest.mark.parametrize("changes,match", [
    (dict(dtype=7), "dtype"), (dict(block_rows=2), "block_rows"), (dict(k=0), "shape"), (dict(x=None), "non-null"),
    (dict(q=4097), "8 bytes"), (dict(ldq=100), "8 bytes"), (dict(batch=70000), "batch"), (dict(x=4097), "aligned"),
])
def test_quantize_entry_refuses_before_any_launch(changes, match):
    v = dict(x=4096, q=4096, scale=4096, batch=1, rows=4, k=128, ldq=128, dtype=_native.DTYPE_BF16, block_rows=1)
    v.update(changes)
    status = _native.library().moegemm_quantize_fp8(v["x"], v["q"], v["scale"], v["batch"], v["rows"], v["k"], 0, 128,
                                                    0, v["ldq"], 0, 1, 4, v["dtype"], v["block_rows"], None)
    assert status == _native.ERR_INVALID and match in _native.last_error()


def test_quantize_entry_refuses_columns_past_one_launch():
    status = _native.library().moegemm_quantize_fp8(4096, 4096, 4096, 1, 1, 2 ** 31 - 1, 0, 2 ** 31, 0, 2 ** 31, 0, 1, 1,
                                                    _native.DTYPE_BF16, 128, None)
    assert status == _native.ERR_INVALID and "2^31 - 128" in _native.last_error()


def _meta(shape, dtype=E4M3):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("shape", [(2 ** 32 + 5, 16), (2 ** 31, 16), (4, 2 ** 32 + 16), (2 ** 32 + 1, 4, 16)])
def test_quantize_refuses_extents_past_32_bits(shape):
    """The library takes 32-bit extents: 2^32 + 5 rows would arrive as 5, and the others stay unwritten."""
    with pytest.raises(ValueError, match="2\\*\\*31"):
        quantize_fp8(_meta(shape, torch.bfloat16))


@pytest.mark.parametrize("rows,n,k,groups", [(2 ** 32 + 5, 32, 16, 1), (2 ** 31, 32, 16, 1), (4, 2 ** 32 + 16, 16, 1),
                                             (4, 32, 2 ** 32 + 16, 1), (4, 32, 16, 2 ** 32 + 1)])
def test_products_refuse_extents_past_32_bits(rows, n, k, groups):
    blocks, fp32 = -(-k // 128), torch.float32
    a, sa = _meta((rows, k)), _meta((rows, blocks), fp32)
    w, sw = _meta((groups, n, k)), _meta((groups, -(-n // 128), blocks), fp32)
    offs = _meta((groups,), torch.int32)
    for call in (grouped_mm_fp8, grouped_mm_fp8_swiglu):
        with pytest.raises(ValueError, match="2\\*\\*31"):
            call(a, sa, w, sw, offs)
