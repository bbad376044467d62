"""The MLP half of a block on int8 weights and int8 rows, as a server and as a LoRA trainer run it.

    python mac-kernels-public_amd/examples/mlp_block.py

serve(): tokens of a prompt, then single ones.  A step is
    add_rms_norm_int8     the residual's addition and the norm, the result rotated and held in 8 bits
    w8a8_int8_linear      the fused gate and up projection
    gated_act_int8        silu(gate) * up, rotated and held in 8 bits
    w8a8_int8_linear      the down projection, with the residual
train(): the same in 16 bits between the products, through frozen weights; the gradients reach the inputs and the norm's weight.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import qlin  # noqa: E402
from qlin.quantize import quantize_int8_convrot_weight  # noqa: E402

DEV = "cuda"
WIDTH, HIDDEN, GROUP = 512, 1536, 128


def _int8(n, k, seed):
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) * k ** -0.5
    return [torch.from_numpy(a).to(DEV) for a in quantize_int8_convrot_weight(w.numpy(), GROUP)]


class Block:
    """The packed weights of one MLP half, rotated in groups of GROUP values, and its norm."""

    def __init__(self, dtype=torch.bfloat16):
        self.gate_up, self.gate_up_scale = _int8(2 * HIDDEN, WIDTH, 1)
        self.down, self.down_scale = _int8(WIDTH, HIDDEN, 2)
        self.norm = (1 + 0.1 * torch.randn(WIDTH, generator=torch.Generator().manual_seed(3))).to(DEV, dtype)

    def step(self, x, residual):
        """x: the attention half's output, residual: what it is added to -> the block's output, the next block's residual."""
        codes, scale, h = qlin.add_rms_norm_int8(x, residual, self.norm, convrot_groupsize=GROUP)
        both = qlin.w8a8_int8_linear(codes, scale, self.gate_up, self.gate_up_scale, None, x.dtype)
        codes, scale = qlin.gated_act_int8(*both.chunk(2, -1), convrot_groupsize=GROUP)
        return qlin.w8a8_int8_linear(codes, scale, self.down, self.down_scale, residual=h)

    def trained(self, x, residual, norm):
        y, h = qlin.add_rms_norm_trainable(x, residual, norm)
        both = qlin.w8a8_linear_trainable(y, self.gate_up, self.gate_up_scale, None, True, GROUP)
        a = qlin.gated_act_trainable(both, packed=True)
        return qlin.w8a8_linear_trainable(a, self.down, self.down_scale, None, True, GROUP) + h


def rows(tokens, seed, dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(tokens, WIDTH, generator=gen).to(DEV, dtype) for _ in range(2)]


def serve(prompt=77, answers=3):
    """(block, inputs, outputs) of a prompt and `answers` single tokens."""
    block = Block()
    inputs = [rows(n, seed) for seed, n in enumerate([prompt] + [1] * answers)]
    return block, inputs, [block.step(*pair) for pair in inputs]


def train(tokens=144):
    """One step: (block, inputs and norm, gradients of all three)."""
    block = Block()
    leaves = [t.requires_grad_(True) for t in (*rows(tokens, 9), block.norm.clone())]
    loss = block.trained(*leaves).float().square().mean()
    return block, leaves, torch.autograd.grad(loss, leaves)


def main():
    _, _, outputs = serve()
    print("served", [tuple(o.shape) for o in outputs], "finite:", all(bool(o.isfinite().all()) for o in outputs))
    _, _, grads = train()
    print("trained, gradients", [tuple(g.shape) for g in grads], "finite:", all(bool(g.isfinite().all()) for g in grads))


if __name__ == "__main__":
    main()
