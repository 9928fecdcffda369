"""CPU tests of the Gate+Up training form's argument checks, in Python and at the C boundary."""

from __future__ import annotations

import pytest
import torch

from kernels import _native, gate_up_swiglu_backward, gate_up_swiglu_forward

BF16 = torch.bfloat16


@pytest.mark.parametrize("change,match", [
    (dict(x=torch.zeros(4, 32, dtype=BF16)), "contraction"), (dict(x=torch.zeros(4, 16)), "fp16 or bf16"),
    (dict(w=torch.zeros(2, 16, 24, dtype=BF16)), "multiples of 8"), (dict(w=torch.zeros(16, 32, dtype=BF16)), "3-D"),
    (dict(w=torch.zeros(2, 16, 32, dtype=torch.float16)), "fp16 or bf16"), (dict(), "GPU"),
])
def test_forward_refuses_what_it_cannot_take(change, match):
    args = dict(x=torch.zeros(4, 16, dtype=BF16), w=torch.zeros(2, 16, 32, dtype=BF16)) | change
    with pytest.raises(ValueError, match=match):
        gate_up_swiglu_forward(args["x"], args["w"], torch.zeros(2, dtype=torch.int32))


def test_backward_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="GPU"):
        gate_up_swiglu_backward(torch.zeros(4, 16, dtype=BF16), torch.zeros(4, 16, dtype=BF16),
                                torch.zeros(16, 32, dtype=BF16), None, torch.zeros(4, 32))


def _call(entry, **changes):
    v = dict(x=4096, w=4096, out=4096, saved=4096, dp=4096, dh=4096, offs=4096, groups=2, rows=4, h=16, f=16, sx=16,
             swg=512, swh=32, so=32, sog=512, sdh=16, dtype=_native.DTYPE_BF16, variant=-1)
    v.update(changes)
    lib = _native.library()
    if entry == "forward":
        return lib.moegemm_gate_up_forward(v["x"], v["w"], v["out"], v["saved"], v["offs"], v["groups"], v["rows"], v["h"],
                                           v["f"], v["sx"], v["swg"], v["swh"], v["so"], v["dtype"], v["variant"], 256,
                                           None)
    dx, dw = (v["out"] if entry in (name, "backward") else None for name in ("dx", "dw"))
    return lib.moegemm_gate_up_backward(v["dh"], v["x"], v["w"], v["saved"], v["dp"], dx, dw, v["offs"], v["groups"], v["rows"],
                                        v["h"], v["f"], v["sdh"], v["sx"], v["swg"], v["swh"], v["dtype"], v["variant"],
                                        v["variant"], 256, None)


ENTRIES = ("forward", "backward", "dx", "dw")


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("changes,match", [(dict(dtype=_native.DTYPE_F32), "fp16 or bf16"), (dict(groups=0), "group_count"),
                                           (dict(offs=None), "one group"), (dict(rows=-1), "shape"),
                                           (dict(f=12), "multiples of 8"), (dict(rows=1 << 30), "shape")])
def test_c_entries_refuse_bad_shapes(entry, changes, match):
    assert _call(entry, **changes) == _native.ERR_INVALID
    assert match in _native.last_error()


@pytest.mark.parametrize("entry,changes", [
    ("forward", dict(x=None)), ("forward", dict(x=4104)), ("forward", dict(sx=20)), ("forward", dict(sx=8)),
    ("forward", dict(swh=24)), ("forward", dict(so=8)), ("forward", dict(saved=4100)), ("forward", dict(swg=516)),
    ("forward", dict(sx=1 << 22)), ("backward", dict(dh=None)), ("backward", dict(sdh=12)), ("backward", dict(dp=4104)),
    ("backward", dict(saved=None)), ("dx", dict(w=None)), ("dx", dict(out=4104)), ("dx", dict(swg=4)),
    ("dx", dict(swh=24)), ("dw", dict(out=4104)), ("dw", dict(x=None)), ("dw", dict(sx=12)),
])
def test_c_entries_refuse_bad_operands(entry, changes):
    assert _call(entry, **changes) == _native.ERR_INVALID
    assert _native.last_error()


def test_unknown_variants_and_empty_calls():
    for product, entry in enumerate(("forward", "dx", "dw")):
        count = _native.library().moegemm_gate_up_variant_count(product)
        assert count >= 3
        assert _call(entry, variant=count) == _native.ERR_NO_KERNEL
    assert _native.library().moegemm_gate_up_variant_count(3) == _native.ERR_INVALID
    for entry in ("forward", "dx"):
        assert _call(entry, rows=0) == _native.OK


@pytest.mark.parametrize("rows,h,width,groups", [(2 ** 32 + 8, 16, 32, 1), (2 ** 31, 16, 32, 1), (4, 2 ** 32 + 16, 32, 1),
                                                 (4, 16, 2 ** 32 + 32, 1), (4, 16, 32, 2 ** 32 + 1)])
def test_extents_past_32_bits_are_refused(rows, h, width, groups):
    """The library takes 32-bit extents: 2^32 + 8 rows would arrive as 8, and the others stay unwritten."""
    x, w = (torch.empty(shape, dtype=BF16, device="meta") for shape in ((rows, h), (groups, h, width)))
    with pytest.raises(ValueError, match="2\\*\\*31"):
        gate_up_swiglu_forward(x, w, torch.empty(groups, dtype=torch.int32, device="meta"))


def test_forward_refuses_a_weight_that_spans_two_gib():
    assert _call("forward", swh=1 << 21) == _native.ERR_INVALID
    assert "2 GiB" in _native.last_error()
