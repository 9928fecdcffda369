"""The expert-layer driver: its arguments and routing on the CPU, one small run of all its parts on a GPU."""

from __future__ import annotations

import json

import pytest
import torch

from harness.expert_layer import build_parser, layer_sizes, main, uneven_ends


def test_sizes_are_one_ranks_of_the_model():
    sizes = layer_sizes(build_parser().parse_args([]))
    assert (sizes.experts, sizes.hidden, sizes.ffn) == (32, 7168, 2048)
    assert (sizes.rows, sizes.decode_rows) == (32 * 128, 32 * 4)
    sizes = layer_sizes(build_parser().parse_args(["--num-experts", "6", "--parallel-size", "2", "--hidden-size", "64",
                                                   "--ffn-size", "32", "--rows", "5", "--decode-rows", "1"]))
    assert (sizes.experts, sizes.hidden, sizes.ffn, sizes.rows, sizes.decode_rows) == (3, 64, 32, 15, 3)


@pytest.mark.parametrize("flags,match", [(["--rows", "0"], "--rows"), (["--parallel-size", "7"], "divisible"),
                                         (["--hidden-size", "24"], "multiples of 16"), (["--steps", "-1"], "--steps"),
                                         (["--learning-rate", "0"], "--learning-rate"),
                                         (["--model-config", "no/such/config.json"], "config.json")])
def test_bad_arguments_end_with_status_2(flags, match, capsys):
    assert main(flags) == 2
    assert match in capsys.readouterr().out


@pytest.mark.parametrize("rows,experts", [(4096, 32), (7, 3), (1, 4), (5, 1)])
def test_ends_cover_the_rows(rows, experts):
    ends = uneven_ends(rows, experts)
    assert ends.dtype == torch.int32 and len(ends) == experts and int(ends[-1]) == rows
    assert (ends.diff() >= 0).all() and int(ends[0]) >= 0


@pytest.mark.gpu
@pytest.mark.parametrize("fast", [False, True])
def test_all_parts_run_together(fast, capsys):
    """The loss falls at every step (a step far below the curvature's limit).  fp8 is within 0.25 of the bf16 layer:
    four operands are each rounded by at most 2^-4 of an element's size."""
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")
    flags = ["--num-experts", "4", "--parallel-size", "1", "--hidden-size", "256", "--ffn-size", "144", "--rows", "40",
             "--decode-rows", "2", "--steps", "3", "--repeat", "0"]
    assert main(flags + ["--fast-accum"] * fast) == 0
    lines = [json.loads(line) for line in capsys.readouterr().out.splitlines() if line.startswith("{")]
    losses = [line["loss"] for line in lines if line["part"] == "train"]
    assert len(losses) == 3 and losses[0] > losses[1] > losses[2] > 0
    distances = {line["part"]: line["distance"] for line in lines if "distance" in line}
    assert set(distances) == {"prefill", "decode"} and all(0 < d < 0.25 for d in distances.values())


@pytest.mark.parametrize("device", ["cpu", "cuda:x", "gpu"])
def test_a_bad_device_ends_with_status_2(device, capsys):
    assert main(["--device", device]) == 2
    assert "--device" in capsys.readouterr().out
