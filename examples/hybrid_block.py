#!/usr/bin/env python3
"""Two layers of a hybrid -- one Hyena-MR, one with linear attention -- trained for a few steps with their activations kept in 8
bits, then a prompt and single tokens through the layer that carries a state.

    python examples/hybrid_block.py [--width 1280] [--length 2048] [--steps 5]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from savanna_amd.operators.block import MixerBlock  # noqa: E402
from savanna_amd.operators.hyena import CgcgConfig, HyenaMixer, HyenaMROperator  # noqa: E402
from savanna_amd.operators.linear_attention import LinearAttention  # noqa: E402


def layers(width, save_8bit, dtype=torch.bfloat16, device="cuda"):
    """Groups of 16 channels and a filter of 128 taps; heads of 64 channels."""
    hyena = HyenaMixer(HyenaMROperator(width, width // 16, 128, CgcgConfig(cgcg_dtype="bfloat16"), small_init=False, device=device),
                       dtype=dtype, device=device)
    return [MixerBlock(width, mixer, save_8bit=save_8bit, dtype=dtype, device=device)
            for mixer in (hyena, LinearAttention(width, width // 64, device=device))]


def main():
    parser = argparse.ArgumentParser()
    parser.add_argument("--width", type=int, default=1280)
    parser.add_argument("--length", type=int, default=2048)
    parser.add_argument("--steps", type=int, default=5)
    args = parser.parse_args()

    x = torch.randn(2, args.length, args.width, device="cuda").to(torch.bfloat16)
    target = torch.roll(x, 1, 1)
    for save_8bit in (False, True):
        torch.manual_seed(0)
        model = torch.nn.Sequential(*layers(args.width, save_8bit))
        optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
        for step in range(args.steps):
            before = torch.cuda.memory_allocated()
            loss = torch.nn.functional.mse_loss(model(x).float(), target.float())
            kept = torch.cuda.memory_allocated() - before
            first = loss.item() if step == 0 else first
            loss.backward()
            optimizer.step()
            optimizer.zero_grad(set_to_none=True)
        print(f"activations in {'8' if save_8bit else '16'} bits: loss {first:.4f}, after {args.steps} steps {loss.item():.4f}; "
              f"{kept / 2 ** 20:.1f} MiB kept from forward to backward")

    layer = model[1]
    lengths = torch.tensor([args.length, args.length // 3], dtype=torch.int32, device="cuda")
    y, state = layer.prefill(x, lengths=lengths)
    token = x[:, 0]
    for _ in range(8):
        token = layer.step(token, state)
    print(f"prompts of {lengths.tolist()} rows, then 8 tokens: state {tuple(state.shape)}, output {tuple(token.shape)}, "
          f"finite {bool(torch.isfinite(token).all())}")


if __name__ == "__main__":
    main()
