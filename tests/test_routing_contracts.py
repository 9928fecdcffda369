"""CPU tests of the routing operators' argument checks, in Python and at the C boundary."""

from __future__ import annotations

import pytest
import torch

from kernels import (
    ExpertOrder,
    _native,
    combine_rows,
    combine_rows_backward,
    gather_rows,
    route_topk,
    route_topk_backward,
    sort_by_expert,
)


class _Gpu:
    """A CPU tensor that says it is on a GPU, for the checks behind that one."""

    def __init__(self, tensor):
        self._tensor = tensor
        self.is_cuda = True

    def __getattr__(self, name):
        return getattr(self._tensor, name)


def on_gpu(*shape, dtype=torch.float32):
    return _Gpu(torch.zeros(shape, dtype=dtype))


@pytest.mark.parametrize("change,match", [
    (dict(logits=torch.zeros(4, 8)), "GPU"), (dict(logits=on_gpu(8)), "2-D"), (dict(k=0), "k must"), (dict(k=9), "k must"),
    (dict(logits=on_gpu(4, 1025)), "1024"), (dict(logits=on_gpu(4, 100), k=65), "k must"), (dict(score="relu"), "score"),
    (dict(logits=_Gpu(torch.zeros(8, 4).t())), "unit stride"), (dict(logits=on_gpu(4, 8, dtype=torch.float64)), "dtype"),
    (dict(groups=3), "groups"), (dict(groups=4, top_groups=5), "groups"), (dict(groups=4, top_groups=0), "groups"),
    (dict(groups=4, group_best=3), "groups"), (dict(groups=8, top_groups=1, k=2), "do not fit"), (dict(groups=0), "groups"),
    (dict(bias=torch.zeros(7)), "bias"), (dict(bias=torch.zeros(8, dtype=torch.float64)), "bias"),
    (dict(bias=torch.zeros(16)[::2]), "bias"),
])
def test_route_refuses_what_it_cannot_take(change, match):
    args = dict(logits=on_gpu(4, 8), k=2) | change
    with pytest.raises(ValueError, match=match):
        route_topk(args.pop("logits"), args.pop("k"), **args)


@pytest.mark.parametrize("change,match", [
    (dict(experts=torch.zeros(4, dtype=torch.int32)), "2-D"), (dict(experts=torch.zeros(4, 2)), "experts must"),
    (dict(experts=torch.zeros(5, 2, dtype=torch.int32)), "experts must"), (dict(dweights=torch.zeros(4, 3)), "dweights must"),
    (dict(dweights=torch.zeros(4, 2, dtype=torch.bfloat16)), "dweights must"),
    (dict(dweights=torch.zeros(2, 4).t()), "dweights must"), (dict(score="max"), "score"),
    (dict(experts=torch.zeros(4, 0, dtype=torch.int32)), "k must"),
])
def test_route_backward_refuses_what_it_cannot_take(change, match):
    args = dict(dweights=torch.zeros(4, 2), logits=on_gpu(4, 8), experts=torch.zeros(4, 2, dtype=torch.int32)) | change
    with pytest.raises(ValueError, match=match):
        route_topk_backward(args.pop("dweights"), args.pop("logits"), args.pop("experts"), **args)


@pytest.mark.parametrize("experts,count,first,match", [
    (torch.zeros(4, 2, dtype=torch.int32), 4, 0, "GPU"), (on_gpu(4, 2, dtype=torch.int64), 4, 0, "int32"),
    (on_gpu(8, dtype=torch.int32), 4, 0, "tokens, k"), (on_gpu(4, 2, dtype=torch.int32), 0, 0, "num_experts"),
    (on_gpu(4, 2, dtype=torch.int32), 1025, 0, "1024"), (on_gpu(4, 2, dtype=torch.int32), 4, -1, "first"),
    (on_gpu(4, 0, dtype=torch.int32), 4, 0, "1 or more"), (_Gpu(torch.zeros(2, 4, dtype=torch.int32).t()), 4, 0, "contiguous"),
    (on_gpu(4, 2, dtype=torch.int32), 4, 2 ** 31, "first"),
])
def test_sort_refuses_what_it_cannot_take(experts, count, first, match):
    with pytest.raises(ValueError, match=match):
        sort_by_expert(experts, count, first=first)


def an_order(tokens=4, k=2, **change):
    parts = dict(offs=torch.zeros(3, dtype=torch.int32), slots=torch.zeros(tokens * k, dtype=torch.int32),
                 places=torch.zeros(tokens, k, dtype=torch.int32)) | change
    return ExpertOrder(**parts)


@pytest.mark.parametrize("x,order,rows,match", [
    (torch.zeros(4, 8), an_order(), None, "GPU"), (on_gpu(5, 8), an_order(), None, "x must"), (on_gpu(4), an_order(), None, "x must"),
    (on_gpu(4, 0), an_order(), None, "bytes a row"), (on_gpu(4, 8), an_order(), -1, "rows must"),
    (on_gpu(4, 8, dtype=torch.float64), an_order(), None, "1, 2 or 4"), (_Gpu(torch.zeros(8, 4).t()), an_order(), None, "unit stride"),
    (on_gpu(4, 8), an_order(places=torch.zeros(4, 2)), None, "places"),
    (on_gpu(4, 8), an_order(places=torch.zeros(2, 4, dtype=torch.int32).t()), None, "places"),
    (on_gpu(4, 8), an_order(places=torch.zeros(4, 0, dtype=torch.int32)), None, "places"),
    (on_gpu(4, 8), an_order(offs=torch.zeros(0, dtype=torch.int32)), None, "offs"),
    (on_gpu(4, 8), an_order(offs=torch.zeros(3)), None, "offs"), (on_gpu(4, 8), an_order(), 2 ** 31, "rows must"),
])
def test_gather_refuses_what_it_cannot_take(x, order, rows, match):
    with pytest.raises(ValueError, match=match):
        gather_rows(x, order, rows=rows)


@pytest.mark.parametrize("y,weights,match", [
    (torch.zeros(8, 8), None, "GPU"), (on_gpu(8, 8, dtype=torch.int32), None, "dtype"),
    (on_gpu(8, 8), torch.zeros(4, 3), "weights"), (on_gpu(8, 8), torch.zeros(4, 2, dtype=torch.bfloat16), "weights"),
    (on_gpu(8, 8), torch.zeros(2, 4).t(), "weights"), (on_gpu(8), None, "y must"),
])
def test_combine_refuses_what_it_cannot_take(y, weights, match):
    with pytest.raises(ValueError, match=match):
        combine_rows(y, an_order(), weights)


@pytest.mark.parametrize("dout,y,match", [
    (torch.zeros(4, 8), on_gpu(8, 8), "GPU"), (on_gpu(5, 8), on_gpu(8, 8), "dout must"), (on_gpu(4, 9), on_gpu(8, 8), "dout must"),
    (on_gpu(4, 8, dtype=torch.float16), on_gpu(8, 8), "y's dtype"), (_Gpu(torch.zeros(8, 4).t()), on_gpu(8, 8), "unit stride"),
])
def test_combine_backward_refuses_what_it_cannot_take(dout, y, match):
    with pytest.raises(ValueError, match=match):
        combine_rows_backward(dout, y, an_order())


def _route(**changes):
    v = dict(logits=4096, bias=4096, weights=4096, experts=4096, tokens=4, count=8, k=2, stride=8, dtype=_native.DTYPE_F32,
             sigmoid=0, groups=1, top=1, best=1, normalize=1) | changes
    return _native.library().moegemm_route_topk(v["logits"], v["bias"], v["weights"], v["experts"], v["tokens"], v["count"], v["k"],
                                                v["stride"], v["dtype"], v["sigmoid"], v["groups"], v["top"], v["best"],
                                                v["normalize"], 1.0, None)


@pytest.mark.parametrize("changes", [
    dict(dtype=5), dict(tokens=-1), dict(count=0), dict(count=1025), dict(k=0), dict(k=9), dict(count=200, k=65), dict(sigmoid=2),
    dict(normalize=3), dict(logits=None), dict(logits=4098), dict(groups=0), dict(groups=3), dict(top=2), dict(top=0), dict(best=3),
    dict(groups=8, top=1), dict(weights=None), dict(experts=None)])
def test_route_entry_refuses(changes):
    assert _route(**changes) == _native.ERR_INVALID
    assert _native.last_error()


def test_empty_calls_are_no_ops():
    lib = _native.library()
    assert _route(tokens=0) == _native.OK
    assert lib.moegemm_route_topk_backward(None, None, None, None, 0, 8, 2, 8, 2, 0, 1, 1.0, None) == _native.OK
    assert lib.moegemm_gather_rows(None, None, None, 4096, 0, 2, 0, 16, 16, 16, None) == _native.OK
    assert lib.moegemm_combine_rows(None, None, None, None, 0, 2, 0, 8, 8, 8, 2, None) == _native.OK
    assert lib.moegemm_combine_rows_backward(None, None, None, None, None, 4096, 4096, 4, 2, 8, 8, 8, 8, 2, None) == _native.OK


def test_other_entries_refuse():
    lib = _native.library()
    bad = [
        lib.moegemm_route_topk_backward(None, 4096, 4096, 4096, 4, 8, 2, 8, 2, 0, 1, 1.0, None),
        lib.moegemm_route_topk_backward(4096, 4096, 4096, 4098, 4, 8, 2, 8, 2, 0, 1, 1.0, None),
        lib.moegemm_sort_by_expert(4096, 4096, 4096, 4096, 8, -1, 4, 4096, 4096, None),
        lib.moegemm_sort_by_expert(4096, 4096, 4096, 4096, 8, 0, 0, 4096, 4096, None),
        lib.moegemm_sort_by_expert(4096, 4096, 4096, 4096, 8, 0, 1025, 4096, 4096, None),
        lib.moegemm_sort_by_expert(4096, 4096, 4096, 4096, 10 ** 6, 0, 4, 4096, 15, None),
        lib.moegemm_sort_by_expert(None, 4096, 4096, 4096, 8, 0, 4, 4096, 4096, None),
        lib.moegemm_sort_by_expert(4096, 4096, 4096, 4096, -1, 0, 4, 4096, 4096, None),
        lib.moegemm_gather_rows(4096, 4096, 4096, None, 4, 2, 8, 16, 16, 16, None),
        lib.moegemm_gather_rows(4096, None, 4096, 4096, 4, 2, 8, 16, 16, 16, None),
        lib.moegemm_gather_rows(4096, 4096, 4096, 4096, 4, 0, 8, 16, 16, 16, None),
        lib.moegemm_gather_rows(4096, 4096, 4096, 4096, 4, 2, 8, 0, 16, 16, None),
        lib.moegemm_combine_rows(4096, None, 4096, 4096, 4, 2, 8, 8, 8, 8, 7, None),
        lib.moegemm_combine_rows(4097, None, 4096, 4096, 4, 2, 8, 8, 8, 8, 1, None),
        lib.moegemm_combine_rows(4096, None, 4096, None, 4, 2, 8, 8, 8, 8, 1, None),
        lib.moegemm_combine_rows_backward(None, 4096, None, 4096, None, 4096, 4096, 4, 2, 8, 8, 8, 8, 2, None),
        lib.moegemm_combine_rows_backward(4096, None, None, 4096, 4096, 4096, 4096, 4, 2, 8, 8, 8, 8, 2, None),
    ]
    assert bad == [_native.ERR_INVALID] * len(bad)
    assert lib.moegemm_sort_workspace_bytes(2 ** 31, 4) == _native.ERR_INVALID
    assert lib.moegemm_sort_workspace_bytes(100, 4) == 0 and lib.moegemm_sort_workspace_bytes(10 ** 6, 4) > 15
