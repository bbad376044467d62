"""The example that runs the attention side together: a served request's outputs are those of causal attention over all its
tokens at once, and the trainer's gradients those of the same step in plain torch."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("attention_block",
                                                  os.path.join(ROOT, "mac-kernels-public_amd", "examples", "attention_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def turned(x, angle):
    """x [tokens, heads, D] (float64) rotated in halves by angle [tokens, D / 2]."""
    u, v = x.chunk(2, -1)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    return torch.cat([u * c - v * s, u * s + v * c], -1)


def normed(x, w):
    return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w


def test_served_requests():
    """Stage roundings to fp16 (the projection, q, k, v, the attention, the output: 2^-11 each) through two products with
    unit-variance weights leave a relative error of a few 2^-11: 4e-3 of the norm is allowed."""
    import qlin
    m = example()
    block, inputs, outputs = m.serve()
    h, kv, d = m.HEADS, m.KV_HEADS, m.DIM
    wqkv = qlin.dequantize_gguf(block.qkv, "Q4_K", ((h + 2 * kv) * d, m.WIDTH)).double().cpu()
    wout = qlin.dequantize_gguf(block.out, "Q4_K", (m.WIDTH, m.WIDTH)).double().cpu()
    for x, y in zip(inputs, outputs):
        x, n = x.double().cpu(), x.shape[0]
        q, k, v = (x @ wqkv.T).view(n, h + 2 * kv, d).split((h, kv, kv), 1)
        angle = torch.arange(n)[:, None] * block.inv_freq.double().cpu()
        q, k = turned(normed(q, block.q_norm.double().cpu()), angle), turned(normed(k, block.k_norm.double().cpu()), angle)
        k, v = (t.repeat_interleave(h // kv, 1) for t in (k, v))
        score = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
        p = torch.softmax(score.masked_fill(torch.ones(n, n).triu(1).bool(), -torch.inf), -1)
        want = torch.einsum("hqk,khd->qhd", p, v).reshape(n, m.WIDTH) @ wout.T + x
        rel = float((y.double().cpu() - want).norm() / want.norm())
        assert y.shape == want.shape and rel < 4e-3, rel


def test_training_step():
    """Against autograd through the float64 formulas with the projection's own bf16 output: the gradients of the norms' weights
    carry the bf16 roundings of q and k and of their gradients (2^-8 each, over many terms): 2e-2 of the norm."""
    import qlin
    m = example()
    x, norms, grads = m.train()
    assert all(bool(g.isfinite().all()) for g in grads) and grads[0].shape == x.shape
    gen = torch.Generator().manual_seed(0)
    w = torch.randn(3 * m.WIDTH, m.WIDTH, generator=gen) * m.WIDTH ** -0.5
    from qlin.quantize import quantize_int8_convrot_weight
    codes, scale = (torch.from_numpy(a).to(m.DEV) for a in quantize_int8_convrot_weight(w.numpy(), 128))
    wd = qlin.dequantize_int8_convrot_weight(codes, scale, 128).double().cpu()
    xd = x.detach().double().cpu().requires_grad_(True)
    n, side = x.shape[0], 12
    i = torch.arange(n)
    pos = torch.stack([torch.zeros_like(i), i // side, i % side]).double()
    freq, axis = qlin.rope_frequencies((16, 24, 24))
    angle = (pos[axis.long()] * freq.double()[:, None]).T
    leaves = [torch.ones(m.DIM, dtype=torch.float64).requires_grad_(True) for _ in range(2)]
    q, k, v = (xd @ wd.T).view(n, 3 * m.HEADS, m.DIM).split(m.HEADS, 1)

    def turned_pairs(t):
        u, w_ = t[..., 0::2], t[..., 1::2]
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        return torch.stack([u * c - w_ * s, u * s + w_ * c], -1).flatten(-2)

    q, k = turned_pairs(normed(q, leaves[0])), turned_pairs(normed(k, leaves[1]))
    p = torch.softmax(torch.einsum("qhd,khd->hqk", q, k) * m.DIM ** -0.5, -1)
    loss = torch.einsum("hqk,khd->hqd", p, v).square().mean()
    want = torch.autograd.grad(loss, [xd, *leaves])
    for got, ref in zip(grads, want):
        rel = float((got.double().cpu() - ref).norm() / ref.norm())
        assert rel < 2e-2, rel
