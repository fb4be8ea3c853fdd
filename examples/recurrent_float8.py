#!/usr/bin/env python3
"""Two layers whose dense products run in 8-bit floating point -- one around a gated recurrence, one around linear attention -- trained for a few
steps on a residual stream that their norms add up, then a prompt and single tokens with the weights laid out for serving.

    python examples/recurrent_float8.py [--width 1280] [--length 2048] [--steps 5]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from savanna_amd.operators.block import MixerBlockFloat8  # noqa: E402
from savanna_amd.operators.gated_recurrence import GatedRecurrence  # noqa: E402
from savanna_amd.operators.linear_attention import LinearAttention  # noqa: E402
from savanna_amd.operators.norm import RMSNorm  # noqa: E402


class Model(torch.nn.Module):
    def __init__(self, width, device="cuda"):
        super().__init__()
        mixers = GatedRecurrence(width, device=device), LinearAttention(width, width // 64, device=device)
        self.layers = torch.nn.ModuleList(MixerBlockFloat8(width, m, device=device) for m in mixers)
        self.norm = RMSNorm(width, dtype=torch.bfloat16, device=device)

    def forward(self, x):
        residual = None
        for layer in self.layers:
            x, residual = layer(x, residual)
        return self.norm(x, residual)[0]

    @torch.no_grad()
    def prefill(self, x, lengths=None):
        residual, states = None, []
        for layer in self.layers:
            x, residual, state = layer.prefill(x, residual, lengths=lengths)
            states.append(state)
        return self.norm(x, residual)[0], states

    @torch.no_grad()
    def step(self, x, states):
        residual = None
        for layer, state in zip(self.layers, states):
            x, residual = layer.step(x, state, residual)
        return self.norm(x, residual)[0]


def main(args=None):
    parser = argparse.ArgumentParser()
    parser.add_argument("--width", type=int, default=1280)
    parser.add_argument("--length", type=int, default=2048)
    parser.add_argument("--steps", type=int, default=5)
    args = parser.parse_args(args)

    torch.manual_seed(0)
    x = torch.randn(2, args.length, args.width, device="cuda").to(torch.bfloat16)
    target = torch.roll(x, 1, 1).float()
    model = Model(args.width)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    for step in range(args.steps):
        loss = torch.nn.functional.mse_loss(model(x).float(), target)
        loss.backward()
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
        print(f"step {step}: loss {loss.item():.4f}")

    model.eval()
    for layer in model.layers:
        layer.lay_out()
    lengths = torch.tensor([args.length, args.length // 3], dtype=torch.int32, device="cuda")
    y, states = model.prefill(x, lengths)
    token = y[:, 0]
    for _ in range(8):
        token = model.step(token, states)
    finite = bool(torch.isfinite(token).all())
    print(f"prompts of {lengths.tolist()} rows, then 8 tokens: states {[tuple(s.shape) for s in states]}, finite {finite}")
    return finite


if __name__ == "__main__":
    main()
