"""A gated MLP block of a W8A8 language model on the 8-bit operators.

Per block and token the work is
    x1     = x + scale * gate * N_post(attention)        residual_norm_quantized
    q, s   = int8 rows of N_pre(x1)                          (the same launch)
    hidden = silu(q W_gate^T) * (q W_up^T)               gemm_scaled, gated: int8 rows again
    y      = hidden W_down^T                             linear
    x2, h  = x1 + scale * gate2 * N_post(y), N_pre(x2)   residual_norm
Weights are quantised once with quantize_rows, one scale per output channel.

    python examples/w8a8_block.py [--tokens T] [--dim D] [--hidden F] [--steps K]

prints how far the int8 block is from the same block in 32-bit floats, and the
time of a step. It also shows the training side: one residual_norm backward
through autograd.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from rns8_b200 import quant  # noqa: E402


class W8A8Block:
    """Norms, gates and int8 weights of one block."""

    def __init__(self, dim: int, hidden: int, dtype=torch.bfloat16, seed: int = 0, device: str = "cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def randn(*shape):
            return torch.randn(*shape, generator=g, device=device)

        self.float_weights = [(randn(2 * hidden, dim) / dim**0.5).to(dtype), (randn(dim, hidden) / hidden**0.5).to(dtype)]
        self.gate_up, self.down = (quant.quantize_rows(w) for w in self.float_weights)
        self.norms = [(1 + 0.1 * randn(dim)).to(dtype) for _ in range(4)]
        self.gates = [(0.5 + 0.1 * randn(1, dim)).to(dtype) for _ in range(2)]
        self.scale = 0.7

    def forward(self, x: torch.Tensor, attention: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        post1, pre1, post2, pre2 = self.norms
        x1, q, s = quant.residual_norm_quantized(x, attention, post_weight=post1, pre_weight=pre1, gate=self.gates[0],
                                                 scale=self.scale)
        hidden = quant.gemm_scaled(q, s, *self.gate_up, gated=True, out_dtype=x.dtype, quantize=True)
        y = quant.linear(hidden, *self.down)
        return quant.residual_norm(x1, y, post_weight=post2, pre_weight=pre2, gate=self.gates[1], scale=self.scale)

    def reference(self, x: torch.Tensor, attention: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The same block from the unquantised weights, in 32-bit floats."""

        def norm(v, w):
            return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w.float()

        post1, pre1, post2, pre2 = self.norms
        gate_up, down = (w.float() for w in self.float_weights)
        x1 = x.float() + self.scale * self.gates[0].float() * norm(attention.float(), post1)
        g, u = (norm(x1, pre1) @ gate_up.t()).chunk(2, dim=-1)
        y = (torch.nn.functional.silu(g) * u) @ down.t()
        x2 = x1 + self.scale * self.gates[1].float() * norm(y, post2)
        return x2, norm(x2, pre2)


def relative_error(got: torch.Tensor, want: torch.Tensor) -> float:
    return float((got.float() - want).norm() / want.norm())


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--dim", type=int, default=4096)
    ap.add_argument("--hidden", type=int, default=8192)
    ap.add_argument("--steps", type=int, default=50)
    args = ap.parse_args(argv)
    if not torch.cuda.is_available():
        print("a CUDA device is needed")
        return 1
    block = W8A8Block(args.dim, args.hidden)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, attention = (torch.randn(args.tokens, args.dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    got, want = block.forward(x, attention), block.reference(x, attention)
    print("relative error: residual %.4f, normed %.4f" % tuple(relative_error(a, b) for a, b in zip(got, want)))

    # A decode loop replays its launches from a graph.
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.forward(x, attention)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    graph.replay()
    begin.record()
    for _ in range(args.steps):
        graph.replay()
    end.record()
    quant.check_status()
    print("%d tokens: %.1f us a block" % (args.tokens, 1e3 * begin.elapsed_time(end) / args.steps))

    weight = block.norms[0].clone().requires_grad_()
    x_out, h = quant.residual_norm(x, attention, post_weight=weight, pre_weight=block.norms[1], gate=block.gates[0])
    (x_out.float().square().mean() + h.float().square().mean()).backward()
    print("gradient of the first norm's weight: norm %.4g" % float(weight.grad.float().norm()))
    return 0


if __name__ == "__main__":
    sys.exit(main())
