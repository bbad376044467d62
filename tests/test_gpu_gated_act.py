"""Gated activation in 16, 32 and 8 bits, and its gradient, against the formulas in 64 bits."""
import pytest
import torch
from mlp_ref import BF16, DEV, F16, F32, U, act, check_codes, half_step, layouts, qlin, rand, rotated, rounded, sigma_bound, within

pytestmark = pytest.mark.gpu
SIZES = [(1, 1), (3, 7), (2, 8), (5, 64), (4, 100), (300, 72), (3, 1000), (2, 4096), (3, 8200), (2, 13824), (2, 16392), (1, 33000)]
DTYPES = [F16, BF16, F32]
ACTS = ["silu", "gelu_tanh"]


def make(t, w, dtype, seed=0, scale=3.0):
    gate = rand(t, w, seed=seed, scale=scale).to(dtype)
    far = torch.tensor([0.0, -0.0, 20.0, -20.0, 100.0, -100.0, 300.0, -300.0, 1e4, -1e4]).to(dtype)
    n = min(w, far.numel())
    gate[0, :n] = far[:n]
    return gate.to(DEV), rand(t, w, seed=seed + 1, dtype=dtype).to(DEV)


def wide(*ts):
    return [None if t is None else t.double().cpu() for t in ts]


def least(z, *factors):
    """sigma below 2^-126 may come out as 0: z and the factors times that."""
    out = z.abs() * 2.0 ** -125
    for f in factors:
        out = out * f.abs()
    return out


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,w", SIZES)
def test_forward(t, w, dtype, kind):
    gate, up = make(t, w, dtype)
    for u in (up, None):
        y = qlin().gated_act(gate, u, act=kind)
        z, v = wide(gate, u)
        f, _, arg = act(z, kind)
        want = f if v is None else f * v
        more = want.abs() * (sigma_bound(arg, dtype) + 2 * U) + least(z, *([] if v is None else [v]))
        assert y.dtype == dtype
        within(y, want, rounded(dtype, want, more))


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [0, 4, 8, 16, 32, 64, 128, 256])
def test_int8(group, dtype, kind):
    """sigma is off by 2^-14 at most where it is above 2^-24 of the row's largest value's: 127 * 2^-14 < 0.008 of a step.  Through a
    rotation that is 2^-14 of the group's norm, at most 16 times the row's largest value: 2^-10 of the scale, 0.124 of a step,
    and what check_codes says."""
    for t, w in [(1, 4), (3, 20), (2, 100), (3, 1024), (2, 13824), (2, 16640), (1, 33024)] if group else SIZES:
        if group and w % group:
            continue
        gate, up = make(t, w, dtype, seed=w)
        gate.clamp_(-30, 30)
        for u in (up, None):
            q, s = qlin().gated_act_int8(gate, u, act=kind, convrot_groupsize=group)
            z, v = wide(gate, u)
            f = act(z, kind)[0]
            want = rotated(f if v is None else f * v, group)
            codes, scale, top = q.cpu().double(), s.cpu().double(), want.abs().amax(-1, keepdim=True)
            within(scale, top / 127, top / 127 * (2.0 ** -13 + 2.0 ** -10 if group else 2.0 ** -14))
            steps = torch.where(top > 0, want * 127 / torch.where(top > 0, top, 1.0), 0.0)
            assert float((codes - steps).abs().max()) <= (0.65 if group else 0.51)
            if group == 0 and dtype == F32:
                check_codes(q, s, want)


@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,w", SIZES)
def test_gradient(t, w, dtype, kind):
    gate, up = make(t, w, dtype, seed=2)
    dy = rand(t, w, seed=9, dtype=dtype).to(DEV)
    for u in (up, None):
        dgate, dup = qlin().gated_act_grad(dy, gate, u, act=kind)
        z, v, d = wide(gate, u, dy)
        f, df, arg = act(z, kind)
        s = torch.where(z == 0, 0.5, f / torch.where(z == 0, 1.0, z))
        # f' = s + z s (1 - s) t': the second term's size, in which 1 - s is off by U besides sigma's share
        c = act(z, kind)
        second = (c[1] - s).abs()
        rel = sigma_bound(arg, dtype)
        more = s * rel + second * (2 * rel + 8 * U) + (z * s).abs() * (1.0 if kind == "silu" else 1.6 * (1 + 0.135 * z ** 2)) * 4 * U
        scale = d.abs() * (1.0 if v is None else v.abs())
        want = d * df * (1.0 if v is None else v)
        within(dgate, want, rounded(dtype, want, scale * (more + 3 * U * df.abs()) + least(z * z * z, scale) + least(z, scale)))
        if u is None:
            assert dup is None
        else:
            want = d * f
            within(dup, want, rounded(dtype, want, want.abs() * (rel + 2 * U) + least(z, d)))
            base = dgate._base if dgate._base is not None else dgate
            assert base.shape == (t, 2 * w) and dup.data_ptr() == base.data_ptr() + w * base.element_size()


def test_gradient_against_differences():
    """Central differences of the fp32 forward call, element by element: the step's third-order term and the forward's rounding over
    the step stay below 2e-3."""
    e = 1e-2
    z = torch.linspace(-6, 6, 512, device=DEV)[None]
    up, dy = rand(1, 512, seed=1).to(DEV), torch.ones(1, 512, device=DEV)
    for kind in ACTS:
        Q = qlin()
        dgate, dup = Q.gated_act_grad(dy, z, up, act=kind)
        diff = (Q.gated_act(z + e, up, act=kind).double() - Q.gated_act(z - e, up, act=kind).double()) / (2 * e)
        assert float((diff - dgate.double()).abs().max()) <= 2e-3 * float(up.abs().max())
        diff = (Q.gated_act(z, up + e, act=kind).double() - Q.gated_act(z, up - e, act=kind).double()) / (2 * e)
        assert float((diff - dup.double()).abs().max()) <= 2e-3


@pytest.mark.parametrize("kind", ["rows", "odd", "columns"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(kind, dtype):
    Q = qlin()
    for w in (256, 1001, 4104):
        gate, up = make(6, w, dtype, seed=w)
        dy = rand(6, w, seed=3, dtype=dtype).to(DEV)
        a, b, c = (layouts(v, kind) for v in (gate, up, dy))
        assert torch.equal(Q.gated_act(gate, up), Q.gated_act(a, b))
        for x, y in zip(Q.gated_act_int8(gate, up), Q.gated_act_int8(a, b)):
            assert torch.equal(x, y)
        for x, y in zip(Q.gated_act_grad(dy, gate, up), Q.gated_act_grad(c, a, b)):
            assert torch.equal(x, y)
        both = torch.cat([gate, up], 1)
        assert torch.equal(Q.gated_act(*both.chunk(2, 1)), Q.gated_act(gate, up))
        y = Q.gated_act(gate.view(2, 3, w), up.view(2, 3, w))
        q, s = Q.gated_act_int8(gate.view(2, 3, w), up.view(2, 3, w))
        dg, du = Q.gated_act_grad(dy.view(2, 3, w), gate.view(2, 3, w), up.view(2, 3, w))
        assert y.shape == q.shape == dg.shape == du.shape == (2, 3, w) and s.shape == (2, 3, 1)


def test_trainable():
    Q = qlin()
    for dtype in DTYPES:
        gate, up = make(5, 264, dtype, seed=6)
        dy = rand(5, 264, seed=7, dtype=dtype).to(DEV)
        want = Q.gated_act_grad(dy, gate, up, act="gelu_tanh")
        lg, lu = gate.clone().requires_grad_(True), up.clone().requires_grad_(True)
        got = torch.autograd.grad(Q.gated_act_trainable(lg, lu, "gelu_tanh"), (lg, lu), dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        both = torch.cat([gate, up], 1).requires_grad_(True)
        y = Q.gated_act_trainable(both, act="gelu_tanh", packed=True)
        assert torch.equal(y, Q.gated_act(gate, up, act="gelu_tanh"))
        assert torch.equal(torch.autograd.grad(y, both, dy)[0], torch.cat(want, 1))
        got = torch.autograd.grad(Q.gated_act_trainable(lg), lg, dy)[0]
        assert torch.equal(got, Q.gated_act_grad(dy, gate)[0])
    with pytest.raises(ValueError):
        Q.gated_act_trainable(both, up, packed=True)
    with pytest.raises(ValueError):
        Q.gated_act_trainable(gate[:, :7], packed=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ACTS)
def test_rows_of_no_size_and_extremes(dtype, kind):
    Q = qlin()
    for shape in ((0, 64), (2, 0, 64)):
        x = torch.empty(shape, dtype=dtype, device=DEV)
        q, s = Q.gated_act_int8(x, x, act=kind)
        assert Q.gated_act(x, x, act=kind).shape == q.shape == Q.gated_act_grad(x, x, x, act=kind)[1].shape == shape and s.shape == (*shape[:-1], 1)
    inf, nan, big = float("inf"), float("nan"), float(torch.finfo(dtype).max)
    z = torch.tensor([[inf, nan, big, -big, 0.0, -0.0]], dtype=dtype, device=DEV)
    y = Q.gated_act(z, act=kind)[0].double().tolist()
    assert y[0] == inf and y[1] != y[1] and y[2] == big and y[3:] == [0.0, 0.0, 0.0]
    d = Q.gated_act_grad(torch.ones_like(z), z, act=kind)[0][0].double().tolist()
    assert d[0] == 1 and d[1] != d[1] and d[2:] == [1, 0, 0.5, 0.5]
    # rows of zeros and of tiny values; an infinity or a NaN stays in its row
    gate = torch.full((5, 64), 30.0, dtype=dtype, device=DEV)
    up = torch.zeros_like(gate)
    up[1] = torch.arange(64, device=DEV).to(dtype) * torch.finfo(dtype).tiny
    up[2, 5], up[3, 6], up[4] = inf, nan, rand(64, seed=1).to(dtype).to(DEV)
    q, s = Q.gated_act_int8(gate, up, act=kind)
    assert bool((q[0] == 0).all()) and float(s[0]) == 0 and q[1].tolist() == [round(i * 127 / 63) for i in range(64)]
    assert not bool(s[2].isfinite()) and not bool(s[3].isfinite())
    assert torch.equal(q[4], Q.gated_act_int8(gate[4:], up[4:], act=kind)[0][0])


def test_both_routes_agree(monkeypatch):
    from qlin import ops
    Q = qlin()
    gate, up = make(6, 520, BF16, seed=2)
    dy = rand(6, 520, seed=3, dtype=BF16).to(DEV)
    three = [v.view(2, 3, 520) for v in (dy, gate, up)]

    def all_of():
        a = [Q.gated_act(gate, up), Q.gated_act(three[1], act="gelu_tanh"), *Q.gated_act_int8(gate, up, convrot_groupsize=8)]
        return a + [*Q.gated_act_int8(three[1]), *Q.gated_act_grad(dy, gate, up), *Q.gated_act_grad(*three), Q.gated_act_grad(dy, gate)[0]]

    first = all_of()
    monkeypatch.setattr(ops, "_FAST", None)
    for a, b in zip(first, all_of()):
        assert torch.equal(a, b)


def test_captured():
    Q = qlin()
    gate, up = make(300, 1032, F16, seed=4)
    dy = rand(300, 1032, seed=5, dtype=F16).to(DEV)

    def step():
        return [Q.gated_act(gate, up), *Q.gated_act_int8(gate, up, convrot_groupsize=8), *Q.gated_act_grad(dy, gate, up)]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        gate.copy_(rand(300, 1032, seed=10 + turn, dtype=F16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
