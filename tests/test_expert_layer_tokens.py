"""harness.expert_layer's part that routes tokens: its arguments on the CPU, one small run on a GPU."""

from __future__ import annotations

import json

import pytest
import torch

from harness.expert_layer import build_parser, layer_sizes, main

SMALL = ["--num-experts", "6", "--parallel-size", "1", "--hidden-size", "256", "--ffn-size", "160", "--rows", "40",
         "--decode-rows", "2", "--steps", "1", "--repeat", "0"]


def test_the_part_is_left_out_by_default():
    assert layer_sizes(build_parser().parse_args(SMALL)).top_k == 0
    assert layer_sizes(build_parser().parse_args(SMALL + ["--top-k", "3"])).top_k == 3


@pytest.mark.parametrize("flags,match", [(["--top-k", "-1"], "--top-k"), (["--top-k", "7"], "--top-k"),
                                         (["--top-k", "2", "--ffn-size", "144"], "multiples of 32")])
def test_bad_arguments_end_with_status_2(flags, match, capsys):
    assert main(SMALL + flags) == 2
    assert match in capsys.readouterr().out


@pytest.mark.gpu
def test_tokens_run_through_routed_experts(capsys):
    """4-bit values are off by at most a quarter of their size, twice along gate * up and once down: within 0.95 of the
    bf16 experts' (1.25^3 - 1)."""
    if not torch.cuda.is_available():
        pytest.skip("ROCm GPU unavailable")
    assert main(SMALL + ["--top-k", "2"]) == 0
    lines = [json.loads(line) for line in capsys.readouterr().out.splitlines() if line.startswith("{")]
    parts = {line["part"]: line for line in lines}
    assert parts["tokens_prefill"]["tokens"] == 120 and parts["tokens_decode"]["tokens"] == 6
    assert all(0 < parts[name]["distance"] < 0.95 for name in ("tokens_prefill", "tokens_decode"))
