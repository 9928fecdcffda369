"""``python -m harness.expert_layer``: one rank's expert layer, trained in bf16 and served in fp8.

The experts are those of one expert-parallel rank of ``--model-config`` (``num_experts / --parallel-size`` of them), with
expert-sorted rows routed unevenly.  Three parts run on the same weights:

* training: ``--steps`` steps of gradient descent of the packed Gate+Up weights towards a target (the down projection
  stays as it is): ``gate_up_swiglu_forward``, ``grouped_mm``, and back through ``grouped_mm`` and
  ``gate_up_swiglu_backward``.  Weights are updated in fp32 and used in bf16; the loss is printed per step;
* quantisation: the trained weights as e4m3 with a scale for each 128 x 128 block (``quantize_fp8``), once;
* serving: ``quantize_fp8`` of the rows, ``grouped_mm_fp8_swiglu`` and ``grouped_mm_fp8``, for the training's rows and for
  ``--decode-rows`` rows an expert; its normwise distance from the bf16 layer and both times are printed.

Each line is one JSON object.  Exit status 2 for bad arguments.  The reference times the forward GEMMs only
(README.md:55-57): this driver has no counterpart there.
"""

from __future__ import annotations

import argparse
import json
from dataclasses import dataclass
from pathlib import Path

from utils.config import load_model_defaults

from .cli import DEFAULT_MODEL_CONFIG, _model_path


def build_parser() -> argparse.ArgumentParser:
    p = argparse.ArgumentParser(prog="python -m harness.expert_layer",
                                description="One rank's expert layer: bf16 training steps, then fp8 serving")
    add = p.add_argument
    add("--model-config", type=Path, default=DEFAULT_MODEL_CONFIG)
    add("--parallel-size", type=int, default=8)
    add("--num-experts", type=int)
    add("--hidden-size", type=int)
    add("--ffn-size", type=int)
    add("--rows", type=int, default=128, help="mean rows per expert of a training step and of prefill")
    add("--decode-rows", type=int, default=4, help="mean rows per expert of a decode step")
    add("--steps", type=int, default=4)
    add("--learning-rate", type=float, default=0.01, help="step against the squared distance's gradient over (rows + H)")
    add("--fast-accum", action="store_true", help="8-bit matrix instructions in the fp8 products")
    add("--repeat", type=int, default=50, help="timed calls per measurement; 0 skips the timing")
    add("--device", default="cuda")
    add("--seed", type=int, default=1234)
    return p


@dataclass(frozen=True)
class LayerSizes:
    experts: int
    hidden: int
    ffn: int
    rows: int
    decode_rows: int


def layer_sizes(args: argparse.Namespace) -> LayerSizes:
    """One rank's sizes; ValueError for what cannot be run."""
    model = load_model_defaults(_model_path(args.model_config))
    experts = model.num_experts if args.num_experts is None else args.num_experts
    hidden = model.hidden_size if args.hidden_size is None else args.hidden_size
    ffn = model.ffn_size if args.ffn_size is None else args.ffn_size
    for flag, value in (("--parallel-size", args.parallel_size), ("--num-experts", experts), ("--hidden-size", hidden),
                        ("--ffn-size", ffn), ("--rows", args.rows), ("--decode-rows", args.decode_rows)):
        if value <= 0:
            raise ValueError(f"{flag} must be positive")
    if args.steps < 0 or args.repeat < 0 or not args.learning_rate > 0:
        raise ValueError("--steps and --repeat must not be negative, --learning-rate must be positive")
    if experts % args.parallel_size:
        raise ValueError("num_experts must be divisible by parallel_size")
    if hidden % 16 or ffn % 16:
        raise ValueError("hidden and ffn sizes must be multiples of 16 (e4m3 rows of 16 bytes)")
    local = experts // args.parallel_size
    return LayerSizes(local, hidden, ffn, local * args.rows, local * args.decode_rows)


def uneven_ends(rows: int, experts: int):
    """int32 end rows on the host: shares from 0.4 to 1.6 of the mean, the remainder on the last experts."""
    import torch

    shares = torch.linspace(0.4, 1.6, experts, dtype=torch.float64)
    return (shares.cumsum(0) / shares.sum() * rows).round().to(torch.int32)


class ExpertLayer:
    """y = (silu(x Wg) * (x Wu)) W2 per expert, bf16, with a gradient step of [Wg | Wu]."""

    def __init__(self, sizes: LayerSizes, device, seed: int):
        import torch

        generator = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape):
            return torch.randn(shape, device=device, generator=generator)

        self.master = normal(sizes.experts, sizes.hidden, 2 * sizes.ffn) / sizes.hidden ** 0.5
        self.w13 = self.master.bfloat16()
        self.w2 = (normal(sizes.experts, sizes.ffn, sizes.hidden) / sizes.ffn ** 0.5).bfloat16()
        self.w2t = self.w2.transpose(1, 2).contiguous()  # [E, H, F]: the backward product's and fp8's layout

    def forward(self, x, offs):
        """Serving: the activation is fused into the Gate+Up launch and nothing is kept for a gradient."""
        from kernels import grouped_mm, grouped_mm_swiglu

        return grouped_mm(grouped_mm_swiglu(x, self.w13, offs), self.w2, offs)

    def step(self, x, target, offs, learning_rate: float):
        """One step on the squared distance from ``target``; returns its mean (a device scalar).

        The gradient is taken over (an expert's mean rows + H), which bounds the rows' part of the curvature (twice that
        for normal x), so that one learning rate holds at every size.
        """
        from kernels import gate_up_swiglu_backward, gate_up_swiglu_forward, grouped_mm

        h, saved = gate_up_swiglu_forward(x, self.w13, offs)
        error = grouped_mm(h, self.w2, offs).float() - target
        dh = grouped_mm((error / (x.shape[0] / len(offs) + x.shape[1])).bfloat16(), self.w2t, offs)
        _, dw = gate_up_swiglu_backward(dh, x, self.w13, offs, saved, need_dx=False)
        self.master.add_(dw, alpha=-learning_rate)
        self.w13.copy_(self.master)
        return error.square().mean()


class Fp8ExpertLayer:
    """The layer with e4m3 weights in 128 x 128 blocks; rows are quantised per call."""

    def __init__(self, layer: ExpertLayer, fast_accum: bool = False):
        from kernels import quantize_fp8

        self.w13, self.s13 = quantize_fp8(layer.w13.transpose(1, 2).contiguous(), block_rows=128)
        self.w2, self.s2 = quantize_fp8(layer.w2t, block_rows=128)
        self.fast_accum = fast_accum

    def forward(self, x, offs):
        from kernels import grouped_mm_fp8, grouped_mm_fp8_swiglu, quantize_fp8

        q, scale = quantize_fp8(x)
        h, scale = grouped_mm_fp8_swiglu(q, scale, self.w13, self.s13, offs, fast_accum=self.fast_accum)
        return grouped_mm_fp8(h, scale, self.w2, self.s2, offs, fast_accum=self.fast_accum)


def run(args: argparse.Namespace, emit) -> None:
    """The three parts; ``emit`` takes a dict per line."""
    import torch

    from utils.benchmark import normwise_relative_error, select_cuda_device, time_cuda

    sizes = layer_sizes(args)
    device = torch.device(select_cuda_device(args.device))
    layer = ExpertLayer(sizes, device, args.seed)
    generator = torch.Generator(device=device).manual_seed(args.seed + 1)
    emit({"part": "layer", "experts": sizes.experts, "hidden": sizes.hidden, "ffn": sizes.ffn, "rows": sizes.rows,
          "decode_rows": sizes.decode_rows, "fast_accum": args.fast_accum})

    def rows_of(count):
        x = torch.randn(count, sizes.hidden, device=device, generator=generator).bfloat16()
        return x, uneven_ends(count, sizes.experts).to(device)

    x, offs = rows_of(sizes.rows)
    target = torch.randn(sizes.rows, sizes.hidden, device=device, generator=generator) * 0.1
    for index in range(args.steps):
        emit({"part": "train", "step": index, "loss": layer.step(x, target, offs, args.learning_rate).item()})
    served = Fp8ExpertLayer(layer, args.fast_accum)
    for name, count in (("prefill", sizes.rows), ("decode", sizes.decode_rows)):
        x, offs = rows_of(count)
        line = {"part": name, "rows": count,
                "distance": normwise_relative_error(served.forward(x, offs), layer.forward(x, offs))}
        if args.repeat:
            for kind, run_one in (("fp8", served), ("bf16", layer)):
                timing = time_cuda(lambda _: run_one.forward(x, offs), 10, args.repeat)
                line[f"{kind}_us"] = round(timing.median_ms * 1e3, 2)
        emit(line)


def main(argv: list[str] | None = None) -> int:
    from utils.benchmark import select_cuda_device

    args = build_parser().parse_args(argv)
    try:
        layer_sizes(args)
        select_cuda_device(args.device)
    except (OSError, ValueError) as exc:
        print(f"expert_layer: {exc}")
        return 2
    run(args, lambda line: print(json.dumps(line), flush=True))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
