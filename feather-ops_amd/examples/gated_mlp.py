#!/usr/bin/env python3
"""The feed-forward half of a decoder layer in 16 bits, trained, and with 4-bit weights, decoding or under an adapter.

    h = x + residual          y = (act(norm(h) @ gate^T) * (norm(h) @ up^T)) @ down^T

The gate's and up's projections, the activation and the product are one operator, of 16-bit or of 4-bit weights. With 4-bit
weights, which are frozen, gradients still reach the layer's input and the norm.

    python feather-ops_amd/examples/gated_mlp.py --tokens 1 --width 4096 --hidden 14336
"""

import argparse
import pathlib
import sys

import torch
from torch import nn

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

import feather_ops as fo  # noqa: E402


class GatedMLP(nn.Module):
    def __init__(self, width: int, hidden: int, activation: str = "silu", eps: float = 1e-6, dtype: torch.dtype = torch.bfloat16,
                 device="cuda"):
        super().__init__()
        self.activation, self.eps, self.int4 = activation, eps, False
        self.norm = nn.Parameter(torch.ones(width, dtype=dtype, device=device))
        self.gate_up = nn.Linear(width, 2 * hidden, bias=False, dtype=dtype, device=device)
        self.down = nn.Linear(hidden, width, bias=False, dtype=dtype, device=device)

    def quantize_(self, group: int = 128, zeros: bool = True) -> "GatedMLP":
        """The projections' weights to 4 bits, in the layers' buffers."""
        fo.to_int4_linear(self, group, zeros)
        self.int4 = True
        return self

    def forward(self, x: torch.Tensor, residual: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(the layer's output, the residual stream h) for x and residual `[tokens, width]`."""
        y, h = fo.rms_norm(x, self.norm, residual, self.eps)
        if self.int4:
            y = fo.int4_gated_linear(y, *self.gate_up.quantized_weight(), activation=self.activation)
        else:
            y = fo.gated_linear(y, self.gate_up.weight, activation=self.activation)
        return self.down(y), h


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--tokens", type=int, default=16)
    parser.add_argument("--width", type=int, default=4096)
    parser.add_argument("--hidden", type=int, default=14336)
    args = parser.parse_args()
    torch.manual_seed(0)
    mlp = GatedMLP(args.width, args.hidden)
    x, residual = (torch.randn(args.tokens, args.width, device="cuda").bfloat16() for _ in range(2))

    y, h = mlp(x.requires_grad_(), residual)
    (y.float().square().mean() + h.float().mean()).backward()
    print("training:  gradients of", ", ".join(f"{name} {tuple(p.grad.shape)}" for name, p in mlp.named_parameters()))

    with torch.no_grad():
        want = mlp(x, residual)[0].float()
        y = mlp.quantize_()(x, residual)[0].float()
        off = ((y - want).norm() / want.norm()).item()
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
    print(f"inference: 4-bit weights {off:.3f} off the 16-bit layer, {sorted(times)[10] * 1e3:.1f} us for {args.tokens} tokens")


if __name__ == "__main__":
    main()
