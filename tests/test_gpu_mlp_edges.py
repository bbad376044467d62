"""The MLP side's calls that its other tests do not make: every product shape, calls at once that need a workspace each, the norm's
gradient against the unrounded sum, and its training ops on other rows and gradients than contiguous ones."""
import pytest
import torch
from mlp_ref import BF16, DEV, F16, F32, U, half_step, qlin, rand, rounded, within
from test_gpu_add_norm import grad as norm_grad
from test_gpu_w8a8 import check, make

pytestmark = pytest.mark.gpu


# tiles of 32 x 16 and 64 x 32, the GEMM's 128 x 256, its 256 x 256 with one k-tile, two and three, whole rounds of these and the rest
@pytest.mark.parametrize("m,k,n", [(96, 1024, 1360), (90, 1040, 1360), (192, 512, 2704), (170, 272, 2700), (576, 1024, 11008), (570, 128, 11264), (2816, 128, 4096),
                                   (2800, 256, 4090), (2816, 384, 4096), (2080, 256, 8192), (2079, 3584, 8192)])
def test_product_shapes(m, k, n):
    s = make(m, k, n, seed=m)
    bias, res, rs = rand(n, seed=1, dtype=F16).to(DEV), rand(m, n, seed=2, dtype=BF16).to(DEV), rand(n, seed=3, dtype=BF16).to(DEV)
    check(qlin().w8a8_int8_linear(*s), *s)
    check(qlin().w8a8_int8_linear(*s, bias, BF16, residual=res, residual_scale=rs), *s, bias, res, rs)


def test_products_of_no_outputs_with_a_residual(monkeypatch):
    from qlin import ops
    for _ in range(2):
        x, sx, w, sw = make(6, 256, 40)
        y = qlin().w8a8_int8_linear(x.view(2, 3, 256), sx.view(2, 3, 1), w[:0], sw[:0], residual=torch.empty(2, 3, 0, dtype=F16, device=DEV))
        assert y.shape == (2, 3, 0) and y.dtype == F16
        monkeypatch.setattr(ops, "_FAST", None)


def products():
    """Calls that copy their operands into the workspace: K of no whole pieces, weights apart, both operands apart."""
    Q, out = qlin(), []
    for m, k, n, pad in ((300, 1000, 264, 0), (70, 1000, 33, 0), (600, 1024, 1100, 128), (300, 272, 512, 5)):
        for seed in (1, 2):
            x, sx, w, sw = make(m, k, n, seed=100 * seed + m)
            if pad:
                big = torch.zeros(n, k + pad, dtype=torch.int8, device=DEV)
                big[:, :k] = w
                w = big[:, :k]
            out.append((seed, lambda x=x, sx=sx, w=w, sw=sw: Q.w8a8_int8_linear(x, sx, w, sw)))
    return out


def gradients():
    """Gradients of the norm's weight, whose partial sums are in the workspace."""
    Q, out = qlin(), []
    for t, w in ((900, 264), (300, 5120), (300, 16401)):
        for seed in (1, 2):
            dy, h, g = (rand(*size, seed=10 * seed + i, dtype=BF16).to(DEV) for i, size in enumerate(((t, w), (t, w), (w,))))
            out.append((seed, lambda dy=dy, h=h, g=g: torch.cat([v.reshape(-1) for v in Q.add_rms_norm_grad(dy, None, h, g)])))
    return out


@pytest.mark.parametrize("calls", [products, gradients])
def test_calls_at_once_have_workspaces_of_their_own(calls):
    """Different operands on two streams, eager and as two graphs, each call's result that of the call alone."""
    from qlin import _lib
    assert _lib.load().qlin_workspace_size(_lib.OP_W8A8_LINEAR, 300, 264, 1000, 0, 0) > 0
    both = [[f for seed, f in calls() if seed == s] for s in (1, 2)]
    want = [[f() for f in fs] for fs in both]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append([f() for f in both[i]])
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    graphs, outs = [], []
    for fs in both:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([f() for f in fs])
        graphs.append(g)
    for _ in range(3):
        for out in outs:
            for v in out:
                v.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
            assert all(torch.equal(f(), b) for f, b in zip(both[i], want[i]))  # eager work between the replays


@pytest.mark.parametrize("dtype,h_dtype", [(F16, F16), (BF16, BF16), (BF16, F32), (F32, F32)])
def test_gradient_takes_the_sum_as_it_was_stored(dtype, h_dtype):
    """What that costs against the gradient through the unrounded sum: a relative e of each h, half a step of its dtype, is 2 e of dweight's
    terms (h's own and rho's) and 5 e of dx's (rho; h, rho^3 and the mean); next to nothing where the residual is fp32."""
    Q = qlin()
    t, w = 300, 1032
    x, r, g = rand(t, w, seed=1, dtype=dtype).to(DEV), rand(t, w, seed=2, dtype=h_dtype, scale=2.0).to(DEV), (1 + 0.2 * rand(w, seed=3)).to(DEV)
    dy, dh = rand(t, w, seed=4, dtype=dtype).to(DEV), rand(t, w, seed=5, dtype=h_dtype).to(DEV)
    lx, lr, lg = (v.clone().requires_grad_(True) for v in (x, r, g))
    y, h = Q.add_rms_norm_trainable(lx, lr, lg)
    _, dx, dw = torch.autograd.grad((y, h), (lx, lr, lg), (dy, dh))
    wide = [v.double().cpu() for v in (dy, dh, x, r, g)]
    wx, size, ww, total = norm_grad(wide[0], wide[1], wide[2] + wide[3], wide[4])
    e = half_step(h_dtype) * 1.05
    within(dx, wx, rounded(h_dtype, wx, (5 * e + 64 * U) * size))
    within(dw, ww, rounded(F32, ww, (2 * e + (64 + t) * U) * total))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_gradients_of_broadcast_and_strided_outputs(dtype):
    """sum().backward() hands an expanded gradient back, a transposed consumer a strided one."""
    Q = qlin()
    t, w = 6, 264
    x, r, g = (rand(*s, seed=i, dtype=dtype).to(DEV).requires_grad_(True) for i, s in enumerate(((t, w), (t, w), (w,))))
    ones = torch.ones(t, w, dtype=dtype, device=DEV)
    pattern = rand(w, t, seed=9, dtype=dtype).to(DEV)
    for f in (lambda: Q.add_rms_norm_trainable(x, r, g)[0], lambda: Q.gated_act_trainable(x, r), lambda: Q.gated_act_trainable(x.view(2, 3, w)).view(t, w)):
        leaves = [v for v in (x, r, g) if torch.autograd.grad(f().sum(), v, allow_unused=True)[0] is not None]
        got = torch.autograd.grad(f().sum(), leaves)
        want = torch.autograd.grad(f(), leaves, ones)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        got = torch.autograd.grad(f().t(), leaves, pattern)
        want = torch.autograd.grad(f(), leaves, pattern.t().contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("shape", [(1,), (5,), (2, 3), (0,), (2, 70)])
def test_trainable_product_of_other_rows(dtype, shape):
    from qlin.quantize import quantize_int8_convrot_weight
    Q = qlin()
    n, k = 96, 512
    codes, scale = (torch.from_numpy(a).to(DEV) for a in quantize_int8_convrot_weight(rand(n, k, seed=1, scale=k ** -0.5).numpy(), 128))
    x, dy = rand(*shape, k, seed=2, dtype=dtype).to(DEV).requires_grad_(True), rand(*shape, n, seed=3, dtype=dtype).to(DEV)
    y = Q.w8a8_linear_trainable(x, codes, scale, rand(n, seed=4, dtype=dtype).to(DEV), True, 128)
    assert y.shape == (*shape, n) and y.dtype == dtype
    dx, = torch.autograd.grad(y, x, dy)
    assert dx.dtype == dtype and torch.equal(dx, Q.int8_linear_grad_input(dy, codes, scale, True, 128, out_dtype=dtype))
    assert not Q.w8a8_linear_trainable(x.detach(), codes, scale, None, True, 128).requires_grad
