"""The attention half of a block on packed weights, as a server and as a LoRA trainer run it.

    python mac-kernels-public_amd/examples/attention_block.py

serve(): three requests with prompts of different lengths, then a few tokens each.  A step is
    paged_plan            pages and slots for the step's new tokens, from the lengths on the GPU
    gguf_linear           the fused QKV projection (Q4_K)
    qk_norm_rope_store    q normalized and rotated, k and v normalized, rotated and put into the cache
    paged_attention       every new token against its request's cache (a prompt's tokens are rows of their own)
    gguf_linear           the output projection, with the residual
train(): image tokens with positions on three axes through a frozen INT8 projection, the trainable norms and rotation and
torch's attention; the gradients reach the input and the norms' weights.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import qlin  # noqa: E402
from qlin.quantize import quantize_gguf, quantize_int8_convrot_weight  # noqa: E402

DEV = "cuda"
HEADS, KV_HEADS, DIM, PAGE = 8, 2, 64, 16
WIDTH = HEADS * DIM


def _q4(n, k, seed):
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) * k ** -0.5
    return torch.from_numpy(quantize_gguf(w.numpy(), "Q4_K")).to(DEV)


class Block:
    """The packed weights and norms of one attention half, and its cache."""

    def __init__(self, blocks=64, dtype=torch.float16):
        self.qkv = _q4((HEADS + 2 * KV_HEADS) * DIM, WIDTH, 1)
        self.out = _q4(WIDTH, WIDTH, 2)
        self.q_norm = (1 + 0.1 * torch.randn(DIM, generator=torch.Generator().manual_seed(3))).to(DEV, dtype)
        self.k_norm = (1 + 0.1 * torch.randn(DIM, generator=torch.Generator().manual_seed(4))).to(DEV, dtype)
        self.inv_freq, _ = qlin.rope_frequencies(DIM, 1e6, device=DEV)
        # a head's page in one piece: [blocks, kv heads, page, D], seen as [blocks, page, kv heads, D]
        self.k_cache, self.v_cache = (torch.empty(blocks, KV_HEADS, PAGE, DIM, dtype=dtype, device=DEV).transpose(1, 2)
                                      for _ in range(2))

    def step(self, x, plan, table):
        """x [tokens, WIDTH] of one step, its plan and the requests' block table -> the block's output."""
        qkv = qlin.gguf_linear(x, self.qkv, "Q4_K", ((HEADS + 2 * KV_HEADS) * DIM, WIDTH))
        q, k, v = qkv.view(-1, HEADS + 2 * KV_HEADS, DIM).split((HEADS, KV_HEADS, KV_HEADS), 1)
        q = qlin.qk_norm_rope_store(q, k, v, self.q_norm, self.k_norm, plan.positions, self.inv_freq, plan.slots,
                                    self.k_cache, self.v_cache)
        # a token is a row: its request's pages, as far as itself
        y = qlin.paged_attention(q, self.k_cache, self.v_cache, table[plan.rows.long()], plan.positions + 1)
        return qlin.gguf_linear(y.view(-1, WIDTH), self.out, "Q4_K", (WIDTH, WIDTH), residual=x)


def serve(prompts=(5, 40, 17), answers=4, seed=0):
    """Runs the prompts and `answers` single tokens a request; returns (inputs, outputs) a request, in order."""
    gen = torch.Generator().manual_seed(seed)
    block, n = Block(), len(prompts)
    table = torch.full((n, 8), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(64, generator=gen).to(torch.int32).to(DEV)
    context = torch.zeros(n, dtype=torch.int32, device=DEV)
    inputs, outputs = [[] for _ in prompts], [[] for _ in prompts]
    for added in [list(prompts)] + [[1] * n] * answers:
        x = torch.randn(sum(added), WIDTH, generator=gen).half().to(DEV)
        plan = qlin.paged_plan(context, torch.tensor(added, dtype=torch.int32, device=DEV), table, free, PAGE, sum(added))
        y = block.step(x, plan, table)
        used = int(plan.used)  # a server keeps its own count; this also says whether the list was long enough
        assert used <= free.numel()
        free, context = free[used:], plan.lengths
        for i, (a, b) in enumerate(zip(x.split(added), y.split(added))):
            inputs[i].append(a)
            outputs[i].append(b)
    return block, [torch.cat(a) for a in inputs], [torch.cat(b) for b in outputs]


def train(side=12, seed=0):
    """One step on side x side image tokens: (input, norm weights, gradients of all three)."""
    gen = torch.Generator().manual_seed(seed)
    n = side * side
    w = torch.randn(3 * WIDTH, WIDTH, generator=gen) * WIDTH ** -0.5
    codes, scale = (torch.from_numpy(a).to(DEV) for a in quantize_int8_convrot_weight(w.numpy(), 128))
    x = torch.randn(n, WIDTH, generator=gen).to(DEV, torch.bfloat16).requires_grad_(True)
    norms = [torch.ones(DIM, device=DEV).requires_grad_(True) for _ in range(2)]
    i = torch.arange(n, device=DEV)
    positions = torch.stack([torch.zeros_like(i), i // side, i % side])  # time, height, width
    inv_freq, axis = qlin.rope_frequencies((16, 24, 24), device=DEV)
    qkv = qlin.int8_linear_trainable(x, codes, scale, None, True, 128)
    q, k, v = qkv.view(n, 3 * HEADS, DIM).split(HEADS, 1)
    q, k = qlin.qk_norm_rope_trainable(q, k, *norms, positions, inv_freq, axis, interleaved=True)
    y = torch.nn.functional.scaled_dot_product_attention(*(t.transpose(0, 1).float() for t in (q, k, v)))
    loss = y.square().mean()
    return x, norms, torch.autograd.grad(loss, [x, *norms])


def main():
    _, inputs, outputs = serve()
    print("served", [tuple(o.shape) for o in outputs], "finite:", all(bool(o.isfinite().all()) for o in outputs))
    _, _, grads = train()
    print("trained, gradients", [tuple(g.shape) for g in grads], "finite:", all(bool(g.isfinite().all()) for g in grads))


if __name__ == "__main__":
    main()
