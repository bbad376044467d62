"""Norm with the residual's addition, in 16, 32 and 8 bits, and its gradient, against the formulas in 64 bits."""
import pytest
import torch
from mlp_ref import BF16, DEV, F16, F32, U, check_codes, layouts, norm, qlin, rand, rotated, rounded, within

pytestmark = pytest.mark.gpu
SIZES = [(1, 1), (3, 7), (2, 8), (5, 64), (4, 100), (9, 256), (3, 1000), (2, 4096), (3, 5120), (2, 8200), (2, 16392), (1, 33000)]
KINDS = [(F16, F16), (BF16, BF16), (F32, F32), (BF16, F32), (F16, F32)]


def make(t, w, dtype, h_dtype, residual=True, seed=0):
    x = (rand(t, w, seed=seed) * torch.exp(0.3 * rand(w, seed=seed + 1))).to(dtype).to(DEV)
    r = rand(t, w, seed=seed + 2, dtype=h_dtype, scale=2.0).to(DEV) if residual else None
    return x, r, (1 + 0.2 * rand(w, seed=seed + 3)).to(dtype).to(DEV)


def wide(*ts):
    return [None if t is None else t.double().cpu() for t in ts]


def bound_y(dtype, y, w):
    """Squares of w values summed in runs of at most 32 and by trees: (32 + 16) roundings of the sum, half of them in rho; the sum, the
    quotient, the root and three products."""
    return rounded(dtype, y, 64 * U * y.abs())


@pytest.mark.parametrize("dtype,h_dtype", KINDS)
@pytest.mark.parametrize("t,w", SIZES)
def test_forward(t, w, dtype, h_dtype):
    x, r, g = make(t, w, dtype, h_dtype)
    for res in (r, None):
        for weight in (g, None, g.float()):
            y, h = qlin().add_rms_norm(x, res, weight)
            want, wh = norm(*wide(x, res, weight))
            assert y.dtype == dtype and h.dtype == (dtype if res is None else h_dtype)
            within(y, want, bound_y(dtype, want, w))
            if res is None:
                assert h is x
            else:
                within(h, wh, rounded(h_dtype, wh, U * wh.abs()))


@pytest.mark.parametrize("group", [0, 4, 8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype,h_dtype", KINDS)
def test_int8(group, dtype, h_dtype):
    for t, w in [(1, 4), (3, 20), (2, 100), (3, 1024), (2, 5120), (2, 16640), (1, 33024)] if group else SIZES:
        if group and w % group:
            continue
        x, r, g = make(t, w, dtype, h_dtype, seed=w)
        for res, weight in ((r, g), (None, g), (r, None)):
            q, s, h = qlin().add_rms_norm_int8(x, res, weight, convrot_groupsize=group)
            want, wh = norm(*wide(x, res, weight))
            assert q.dtype == torch.int8 and s.dtype == F32
            check_codes(q, s, rotated(want, group), group)
            if res is not None:
                within(h, wh, rounded(h_dtype, wh, U * wh.abs()))


@pytest.mark.parametrize("kind", ["rows", "odd", "columns"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_layouts(kind, dtype):
    """Rows of a larger tensor, at odd addresses, columns first: the same bits; and leading dimensions."""
    Q = qlin()
    for w in (256, 1001, 4104):
        x, r, g = make(6, w, dtype, dtype, seed=w)
        lx, lr = layouts(x, kind), layouts(r, kind)
        for a, b in zip(Q.add_rms_norm(x, r, g), Q.add_rms_norm(lx, lr, g)):
            assert torch.equal(a, b)
        for a, b in zip(Q.add_rms_norm_int8(x, r, g), Q.add_rms_norm_int8(lx, lr, g)):
            assert torch.equal(a, b)
        for a, b in zip(Q.add_rms_norm_grad(r, x, r, g), Q.add_rms_norm_grad(lr, lx, lr, g)):
            assert torch.equal(a, b)
        y, h = Q.add_rms_norm(x.view(2, 3, w), r.view(2, 3, w), g)
        assert y.shape == h.shape == (2, 3, w) and torch.equal(y.view(6, w), Q.add_rms_norm(x, r, g)[0])
        q, s, h = Q.add_rms_norm_int8(x.view(2, 3, w), r.view(2, 3, w), g)
        assert q.shape == (2, 3, w) and s.shape == (2, 3, 1)
        dx, dw = Q.add_rms_norm_grad(r.view(2, 3, w), None, x.view(2, 3, w), g)
        assert dx.shape == (2, 3, w) and dw.shape == (w,)


def grad(dy, dh, h, w, eps=1e-6):
    rho = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    g = dy if w is None else dy * w
    mean = (g * h).mean(-1, keepdim=True)
    dx = rho * (g - h * rho ** 2 * mean)
    size = rho * (g.abs() + h.abs() * rho ** 2 * (g * h).abs().mean(-1, keepdim=True))
    if dh is not None:
        dx, size = dx + dh, size + dh.abs()
    part = dy * h * rho
    return dx, size, part.sum(0), part.abs().sum(0)


@pytest.mark.parametrize("dtype,h_dtype", KINDS)
@pytest.mark.parametrize("t,w", SIZES + [(700, 264), (1030, 72)])
def test_gradient(t, w, dtype, h_dtype):
    """dx: the roundings of bound_y in each of its terms.  dw: a sum of t terms in runs, each with the roundings of rho."""
    x, r, g = make(t, w, dtype, h_dtype, seed=1)
    h = r if r is not None else x
    dy, dh = rand(t, w, seed=8, dtype=dtype).to(DEV), rand(t, w, seed=9, dtype=h_dtype).to(DEV)
    for d, weight in ((dh, g), (None, g.float()), (dh, None)):
        dx, dw = qlin().add_rms_norm_grad(dy, d, h, weight)
        wx, size, ww, total = grad(*wide(dy, d, h, weight))
        assert dx.dtype == h_dtype
        within(dx, wx, rounded(h_dtype, wx, 64 * U * size))
        if weight is None:
            assert dw is None
        else:
            assert dw.dtype == weight.dtype
            within(dw, ww, rounded(weight.dtype, ww, (64 + t) * U * total))
            again = qlin().add_rms_norm_grad(dy, d, h, weight)
            assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    assert qlin().add_rms_norm_grad(dy, dh, h, g, weight_grad=False)[1] is None


def test_gradient_against_differences():
    """Central differences of the fp32 forward call along random directions: the step's third-order term and the forward's own
    rounding over the step are below 2e-3 of the derivative."""
    Q = qlin()
    t, w, e = 6, 500, 1e-2
    x, r, g = make(t, w, F32, F32, seed=3)
    cy, ch = rand(t, w, seed=4).to(DEV), rand(t, w, seed=5).to(DEV)

    def loss(x, r, g):
        y, h = Q.add_rms_norm(x, r, g)
        return float((y.double() * cy).sum() + (h.double() * ch).sum())

    leaves = [v.clone().requires_grad_(True) for v in (x, r, g)]
    y, h = Q.add_rms_norm_trainable(*leaves)
    grads = torch.autograd.grad((y, h), leaves, (cy, ch))
    for i in range(3):
        d = torch.sign(grads[i])  # a direction along which the derivative is far from 0
        args = [[v + s * e * d if j == i else v for j, v in enumerate((x, r, g))] for s in (1, -1)]
        diff = (loss(*args[0]) - loss(*args[1])) / (2 * e)
        want = float((grads[i].double() * d).sum())
        assert abs(diff - want) <= 2e-3 * abs(want), (i, diff, want)


def test_trainable():
    """The gradients that reach x, the residual and the weight, with and without each, and frozen."""
    Q = qlin()
    for dtype, h_dtype in KINDS:
        x, r, g = make(5, 264, dtype, h_dtype, seed=6)
        dy, dh = rand(5, 264, seed=7, dtype=dtype).to(DEV), rand(5, 264, seed=8, dtype=h_dtype).to(DEV)
        lx, lr, lg = (v.clone().requires_grad_(True) for v in (x, r, g))
        y, h = Q.add_rms_norm_trainable(lx, lr, lg)
        dx, dw = Q.add_rms_norm_grad(dy, dh, h, g)
        got = torch.autograd.grad((y, h), (lx, lr, lg), (dy, dh), retain_graph=True)
        assert torch.equal(got[0], dx.to(dtype)) and torch.equal(got[1], dx) and torch.equal(got[2], dw)
        got = torch.autograd.grad(y, (lx, lr, lg), dy, retain_graph=True)
        assert torch.equal(got[1], Q.add_rms_norm_grad(dy, None, h, g)[0])
        got = torch.autograd.grad(h, (lx, lr), dh)  # y has no part in it
        assert torch.equal(got[1], dh) and torch.equal(got[0], dh.to(dtype))
        y, h = Q.add_rms_norm_trainable(lx, None, lg)
        assert h is lx
        got = torch.autograd.grad(y, (lx, lg), dy)
        want = Q.add_rms_norm_grad(dy, None, x, g)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        y, _ = Q.add_rms_norm_trainable(lx, r, g)  # frozen weight and residual
        assert torch.equal(torch.autograd.grad(y, lx, dy)[0], Q.add_rms_norm_grad(dy, None, h=Q.add_rms_norm(x, r, g)[1], weight=g)[0].to(dtype))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rows_of_no_size_and_extremes(dtype):
    Q = qlin()
    g = torch.ones(64, dtype=dtype, device=DEV)
    for shape in ((0, 64), (2, 0, 64)):
        x = torch.empty(shape, dtype=dtype, device=DEV)
        y, h = Q.add_rms_norm(x, x, g)
        q, s, _ = Q.add_rms_norm_int8(x, x, g)
        dx, dw = Q.add_rms_norm_grad(x, x, x, g)
        assert y.shape == h.shape == q.shape == dx.shape == shape and s.shape == (*shape[:-1], 1)
        assert bool((dw == 0).all())
    # a row of zeros: zeros, its scale too; a row of tiny values keeps its codes; infinities and NaN stay in their row
    x = torch.zeros(5, 64, dtype=dtype, device=DEV)
    x[1] = torch.arange(64, device=DEV).to(dtype) * torch.finfo(dtype).tiny
    x[2, 5] = float("inf")
    x[3, 6] = float("nan")
    x[4] = rand(64, seed=1).to(dtype).to(DEV)
    y, _ = Q.add_rms_norm(x, None, g)
    q, s, _ = Q.add_rms_norm_int8(x, None, g)
    assert bool((y[0] == 0).all()) and bool((q[0] == 0).all()) and float(s[0]) == 0
    assert q[1].tolist() == [round(i * 127 / 63) for i in range(64)]
    assert bool(y[2, 5].isnan()) and bool((y[2, :5] == 0).all()) and bool(y[3].isnan().all())
    assert not bool(s[2].isfinite()) and not bool(s[3].isfinite())
    assert torch.equal(y[4], Q.add_rms_norm(x[4:], None, g)[0][0]) and torch.equal(q[4], Q.add_rms_norm_int8(x[4:], None, g)[0][0])
    # eps alone holds a row of zeros
    assert bool(Q.add_rms_norm(x[:1], None, g, eps=0.0)[0].isnan().all())


def test_both_routes_agree(monkeypatch):
    """The C++ calls and the ctypes ones."""
    from qlin import ops
    Q = qlin()
    x, r, g = make(6, 520, BF16, F32, seed=2)
    dy = rand(6, 520, seed=3, dtype=BF16).to(DEV)

    def all_of():
        a = [*Q.add_rms_norm(x, r, g), *Q.add_rms_norm(x.view(2, 3, 520), None, None)]
        a += [*Q.add_rms_norm_int8(x, r, g, convrot_groupsize=8), *Q.add_rms_norm_int8(x.view(2, 3, 520), None, g)]
        return a + [*Q.add_rms_norm_grad(dy, r, r, g), *Q.add_rms_norm_grad(dy.view(2, 3, 520), None, x.view(2, 3, 520), g)]

    first = all_of()
    assert ops._FAST is not None
    monkeypatch.setattr(ops, "_FAST", None)
    for a, b in zip(first, all_of()):
        assert torch.equal(a, b)


def test_captured_and_on_other_streams():
    """A captured call replays over new values; a call on another stream than the default one."""
    Q = qlin()
    x, r, g = make(300, 1032, F16, F16, seed=4)
    dy = rand(300, 1032, seed=5, dtype=F16).to(DEV)

    def step():
        y, h = Q.add_rms_norm(x, r, g)
        return [y, h, *Q.add_rms_norm_int8(x, r, g)[:2], *Q.add_rms_norm_grad(dy, r, h, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [v.clone() for v in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        x.copy_(rand(300, 1032, seed=10 + turn, dtype=F16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
    x.copy_(make(300, 1032, F16, F16, seed=4)[0])
    for a, b in zip(eager, step()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,h_dtype", KINDS)
def test_gradient_of_many_long_rows(dtype, h_dtype):
    """Rows longer than a workgroup holds, more than there are workgroups: partial sums over rows in turn."""
    test_gradient(600, 16401, dtype, h_dtype)
