"""The example that runs the MLP side together, against the formulas in 64 bits over the dequantized weights."""
import importlib.util
import os

import pytest
import torch
from mlp_ref import act, norm

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("mlp_block", os.path.join(ROOT, "mac-kernels-public_amd", "examples", "mlp_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def weights(m, block):
    import qlin
    return [qlin.dequantize_int8_convrot_weight(q, s, m.GROUP).double().cpu()
            for q, s in ((block.gate_up, block.gate_up_scale), (block.down, block.down_scale))]


def mlp(x, residual, w, gate_up, down):
    y, h = norm(x, residual, w)
    gate, up = (y @ gate_up.T).chunk(2, -1)
    return (act(gate, "silu")[0] * up) @ down.T, h


def test_served_rows():
    """Rows in 8 bits: half a step of top / 127 at most, 0.29 steps in the mean; top is at most 4.5 times a normal row's mean magnitude
    here, so each of the two roundings is 1.1% of its row, the first one grows to at most twice that through the gated
    product, and bf16 adds 2^-9 four times: 4e-2 of what the MLP adds to the residual is allowed, a norm over each row."""
    m = example()
    block, inputs, outputs = m.serve()
    wg, wd = weights(m, block)
    for (x, r), y in zip(inputs, outputs):
        add, h = mlp(x.double().cpu(), r.double().cpu(), block.norm.double().cpu(), wg, wd)
        got = y.double().cpu() - h
        rel = ((got - add).norm(dim=-1) / add.norm(dim=-1)).max()
        assert y.shape == add.shape and float(rel) < 4e-2, float(rel)


def test_one_captured_step():
    """A single token's step captured into a graph, replayed over new rows between eager ones."""
    m = example()
    block = m.Block()
    x, r = m.rows(1, 20)
    block.step(x, r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.step(x, r)
    for seed in range(3):
        a, b = m.rows(1, 30 + seed)
        x.copy_(a)
        r.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, block.step(a, b))


def test_training_step():
    """The gradients pass through the roundings of the rows: they are those of the formulas at a point 1 to 3% away (see above),
    and the frozen linears' gradients round dy to fp16 rows: 6e-2 of each gradient's norm is allowed."""
    m = example()
    block, leaves, grads = m.train()
    wg, wd = weights(m, block)
    wide = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    add, h = mlp(*wide, wg, wd)
    want = torch.autograd.grad((add + h).square().mean(), wide)
    for got, ref in zip(grads, want):
        rel = float((got.double().cpu() - ref).norm() / ref.norm())
        assert got.shape == ref.shape and rel < 6e-2, rel
