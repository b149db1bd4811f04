#!/usr/bin/env python3
"""The feed-forward half of a decoder layer in fp8 with a scale for each block of 128 values.

    h = x + residual          y = silu(norm(h) @ gate^T) * (norm(h) @ up^T) @ down^T

Inference keeps fp8 between the kernels: the norm writes the codes and scales that the gate and up projection (one weight)
reads, the gated activation those of the down projection, so four launches and no 16-bit activations but the projections'
outputs. Training runs the same layer on 16-bit activations and quantizes what each product needs.

    python feather-ops_amd/examples/block_scaled_mlp.py --tokens 1 --width 4096 --hidden 14336
"""

import argparse
import pathlib
import sys

import torch
from torch import nn

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

import feather_ops as fo  # noqa: E402


class BlockScaledMLP(nn.Module):
    def __init__(self, width: int, hidden: int, eps: float = 1e-6, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        super().__init__()
        self.eps = eps
        self.norm = nn.Parameter(torch.ones(width, dtype=dtype, device=device))
        self.gate_up = nn.Linear(width, 2 * hidden, bias=False, dtype=dtype, device=device)
        self.down = nn.Linear(hidden, width, bias=False, dtype=dtype, device=device)
        fo.to_block_scaled_linear(self)

    def freeze_(self) -> "BlockScaledMLP":
        """For inference: the weights take no gradients and are quantized once. (Inputs may still ask for theirs.)"""
        self.requires_grad_(False)
        self.gate_up.quantize_weight_()
        self.down.quantize_weight_()
        return self

    def forward(self, x: torch.Tensor, residual: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(the layer's output, the residual stream h) for x and residual `[tokens, width]`."""
        wide, narrow = self.gate_up.quantized_weight(), self.down.quantized_weight()
        differentiable = torch.is_grad_enabled() and any(t.requires_grad for t in (x, residual, *self.parameters()))
        if differentiable or wide is None or narrow is None:
            y, h = fo.rms_norm(x, self.norm, residual, self.eps)
            return self.down(fo.silu_mul(self.gate_up(y))), h
        codes, scale, h = fo.rms_norm_quantized(x, self.norm, residual, self.eps)
        codes, scale = fo.silu_mul_quantized(fo.block_scaled_mm(codes, scale, *wide, None, x.dtype))
        return fo.block_scaled_mm(codes, scale, *narrow, None, x.dtype), h


def reference(mlp: BlockScaledMLP, x: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
    """The layer's output without quantization, in 32 bits."""
    h = (x + residual).float()
    y = h * (h.square().mean(-1, keepdim=True) + mlp.eps).rsqrt() * mlp.norm.float()
    gate, up = (y @ mlp.gate_up.weight.float().t()).chunk(2, -1)
    return (nn.functional.silu(gate) * up) @ mlp.down.weight.float().t()


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--tokens", type=int, default=16)
    parser.add_argument("--width", type=int, default=4096)
    parser.add_argument("--hidden", type=int, default=14336)
    args = parser.parse_args()
    torch.manual_seed(0)
    mlp = BlockScaledMLP(args.width, args.hidden)
    x, residual = (torch.randn(args.tokens, args.width, device="cuda").bfloat16() for _ in range(2))

    y, h = mlp(x.requires_grad_(), residual)
    (y.float().square().mean() + h.float().mean()).backward()
    print("training:  gradients of", ", ".join(f"{name} {tuple(p.grad.shape)}" for name, p in mlp.named_parameters()))

    with torch.no_grad():
        mlp.freeze_()
        y, _ = mlp(x, residual)
        want = reference(mlp, x, residual)
        off = ((y.float() - want).norm() / want.norm()).item()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            mlp(x, residual)
        times = []
        for _ in range(20):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            graph.replay()
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
    print(f"inference: {off:.3f} off the 32-bit layer, {sorted(times)[10] * 1e3:.1f} us for {args.tokens} tokens")


if __name__ == "__main__":
    main()
