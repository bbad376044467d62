"""The product of int8 rows against the exact integer sums."""
import pytest
import torch
from mlp_ref import BF16, DEV, F16, F32, U, qlin, rand, rounded, within

pytestmark = pytest.mark.gpu
ROWS = [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 128, 200, 257, 333, 512]
SHAPES = [(1, 1), (7, 3), (64, 16), (100, 40), (128, 128), (192, 65), (256, 1), (272, 300), (1000, 77), (1024, 512), (4096, 256), (4100, 130)]


def make(m, k, n, seed=0, top=127):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-top, top + 1, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-top, top + 1, (n, k), generator=g, dtype=torch.int8)
    sx, sw = torch.rand(m, 1, generator=g) * 0.02 + 1e-3, (torch.rand(n, generator=g) * 0.02 + 1e-3) * k ** -0.5
    return [t.to(DEV) for t in (x, sx, w, sw)]


def check(y, x, sx, w, sw, bias=None, residual=None, rs=None):
    """Exact sums (float64 products of whole numbers); the epilogue rounds at most five times in fp32."""
    x, sx, w, sw = (t.cpu().double() for t in (x, sx, w, sw))
    base = x.reshape(-1, x.shape[-1]) @ w.T * sx.reshape(-1, 1) * sw.reshape(1, -1)
    size = base.abs()
    if bias is not None:
        base, size = base + bias.cpu().double(), size + bias.cpu().double().abs()
    if residual is not None:
        f = 1.0 if rs is None else rs.cpu().double()
        r = residual.cpu().double().reshape(base.shape)
        base, size = r + f * base, r.abs() + size * (f if rs is None else f.abs())
    within(y.reshape(base.shape), base, rounded(y.dtype, base, 6 * U * size))


@pytest.mark.parametrize("m", ROWS)
def test_shapes(m):
    for i, (k, n) in enumerate(SHAPES):
        s = make(m, k, n, seed=m + i)
        dt = (F16, BF16, F32)[i % 3]
        y = qlin().w8a8_int8_linear(*s, out_dtype=dt)
        assert y.shape == (m, n) and y.dtype == dt
        check(y, *s)


@pytest.mark.parametrize("m", [1, 3, 8, 16, 40, 64, 130, 600])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_bias_and_residual(m, dtype):
    for k, n in ((256, 100), (1000, 72), (2048, 264)):
        s = make(m, k, n, seed=m + n)
        bias, res, rs = rand(n, seed=1, dtype=dtype).to(DEV), rand(m, n, seed=2, dtype=dtype).to(DEV), rand(n, seed=3, dtype=dtype).to(DEV)
        for b, r, f in ((bias, None, None), (None, res, None), (bias, res, rs), (bias.float(), res.float(), rs.half())):
            y = qlin().w8a8_int8_linear(*s, b, dtype, residual=r, residual_scale=f)
            check(y, *s, b, r, f)


@pytest.mark.parametrize("m,k,n", [(1, 5120, 13824), (8, 13824, 1000), (64, 16384, 300), (64, 5120, 13824), (130, 13824, 5120), (250, 13824, 5120), (256, 4096, 4096), (512, 4096, 500), (333, 5120, 5120), (1200, 4096, 6144), (2500, 5120, 4864),
                                   (900, 1024, 4096), (800, 16384, 4100), (2048, 2048, 4096), (333, 4112, 4096), (1500, 4100, 1000)])
def test_large(m, k, n):
    s = make(m, k, n)
    bias = rand(n, seed=1, dtype=BF16).to(DEV)
    res = rand(m, n, seed=2, dtype=BF16).to(DEV)
    check(qlin().w8a8_int8_linear(*s, bias, BF16, residual=res), *s, bias, res)


@pytest.mark.parametrize("m", [1, 2, 9, 40, 300])
@pytest.mark.parametrize("k", [131071, 131056, 130944])
def test_largest_sums(m, k):
    """All codes at their ends: sums to just below 2^31, exact."""
    n = 20
    x, w = torch.full((m, k), -128, dtype=torch.int8, device=DEV), torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    x[:, -1] = 3
    w[:, -2] = 5
    sx, sw = torch.full((m, 1), 2.0 ** -20, device=DEV), torch.ones(n, device=DEV)
    check(qlin().w8a8_int8_linear(x, sx, w, sw, out_dtype=F32), x, sx, w, sw)


@pytest.mark.parametrize("m", [1, 2, 6, 20, 50, 150])
def test_layouts(m):
    """Rows of larger tensors, at odd addresses; three dimensions; scales in other shapes and dtypes: the same bits."""
    Q = qlin()
    for k, n in ((256, 70), (1024, 130), (1000, 33)):
        x, sx, w, sw = make(m, k, n, seed=k)
        want = Q.w8a8_int8_linear(x, sx, w, sw)
        for pad, first in ((16, 0), (48, 16), (5, 1), (128, 3)):
            bx, bw = (torch.zeros(t.shape[0], k + pad + first, dtype=torch.int8, device=DEV) for t in (x, w))
            bx[:, first:first + k], bw[:, first:first + k] = x, w
            vx, vw = bx[:, first:first + k], bw[:, first:first + k]
            for a, b in ((vx, w), (x, vw), (vx, vw)):
                assert torch.equal(Q.w8a8_int8_linear(a, sx, b, sw), want)
        assert torch.equal(Q.w8a8_int8_linear(x.t().contiguous().t(), sx, w.t().contiguous().t(), sw), want)
        y = Q.w8a8_int8_linear(x[None, :, None], sx[None, :, None], w, sw[:, None])
        assert y.shape == (1, m, 1, n) and torch.equal(y.view(m, n), want)
        one = Q.w8a8_int8_linear(x, sx, w, torch.full((1,), 0.5, device=DEV))
        assert torch.equal(one, Q.w8a8_int8_linear(x, sx.view(-1), w, torch.full((n,), 0.5, device=DEV)))
        half = sw.half()
        assert torch.equal(Q.w8a8_int8_linear(x, sx, w, half), Q.w8a8_int8_linear(x, sx, w, half.float()))
        big = torch.randn(m, n + 9, device=DEV).half()
        assert torch.equal(Q.w8a8_int8_linear(x, sx, w, sw, None, F16, residual=big[:, 3:3 + n]),
                           Q.w8a8_int8_linear(x, sx, w, sw, None, F16, residual=big[:, 3:3 + n].contiguous()))


def test_no_rows_or_outputs_and_scales_that_are_not_finite():
    Q = qlin()
    x, sx, w, sw = make(3, 256, 40)
    assert Q.w8a8_int8_linear(x[:0], sx[:0], w, sw).shape == (0, 40) and Q.w8a8_int8_linear(x, sx, w[:0], sw[:0]).shape == (3, 0)
    for m in (3, 80):
        x, sx, w, sw = make(m, 256, 40)
        want = Q.w8a8_int8_linear(x, sx, w, sw)
        sx[1] = float("nan")
        y = Q.w8a8_int8_linear(x, sx, w, sw)
        assert bool(y[1].isnan().all()) and torch.equal(y[2:], want[2:]) and torch.equal(y[0], want[0])


def test_behind_the_last_output_nothing_is_written():
    """Rows of a larger buffer through the C ABI: what stands around them stays."""
    from qlin import _lib
    for m in (1, 3, 20, 70, 300):
        x, sx, w, sw = make(m, 384, 50)
        big = torch.full((m + 2, 64), 7.0, dtype=F16, device=DEV)
        y = big[1:m + 1, 5:55]
        n = _lib.load().qlin_workspace_size(_lib.OP_W8A8_LINEAR, m, 50, 384, 0, 0)
        room = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
        d = _lib.desc
        st = _lib.load().qlin_w8a8_linear(d(x), d(sx), d(w), d(sw), None, None, None, d(y), room.data_ptr(), room.numel(),
                                          _lib.stream_of(x.device))
        assert st == 0
        check(y, x, sx, w, sw)
        y.fill_(7)
        assert bool((big == 7).all())


def test_both_routes_agree(monkeypatch):
    from qlin import ops
    Q = qlin()

    def all_of():
        out = []
        for m, k, n in ((1, 256, 40), (6, 1000, 33), (70, 512, 130), (300, 1024, 264)):
            s = make(m, k, n, seed=m)
            b, r, f = rand(n, seed=1).to(DEV), rand(m, n, seed=2, dtype=F16).to(DEV), rand(n, seed=3).to(DEV)
            out += [Q.w8a8_int8_linear(*s), Q.w8a8_int8_linear(*s, b, residual=r, residual_scale=f), Q.w8a8_int8_linear(*s, out_dtype=F32)]
        return out

    first = all_of()
    monkeypatch.setattr(ops, "_FAST", None)
    for a, b in zip(first, all_of()):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_captured_and_two_streams():
    """Captured calls replay over new rows, two graphs that share nothing; calls on two streams at once."""
    Q = qlin()
    cases = [make(m, k, n, seed=m) for m, k, n in ((1, 4096, 512), (9, 1000, 264), (40, 4096, 300), (200, 2048, 512))]
    run = lambda: [Q.w8a8_int8_linear(*s) for s in cases]  # noqa: E731
    run()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    for turn in range(3):
        for i, s in enumerate(cases):
            s[0].copy_(make(*s[0].shape, 8, seed=50 + turn + i)[0])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = run()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(run())
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_trainable():
    """The forward call over the quantized rows; the gradient is the frozen linear's."""
    Q = qlin()
    from qlin.quantize import quantize_int8_convrot_weight
    n, k = 96, 512
    codes, scale = (torch.from_numpy(a).to(DEV) for a in quantize_int8_convrot_weight(rand(n, k, seed=1, scale=k ** -0.5).numpy(), 128))
    x = rand(40, k, seed=2, dtype=BF16).to(DEV).requires_grad_(True)
    dy = rand(40, n, seed=3, dtype=BF16).to(DEV)
    y = Q.w8a8_linear_trainable(x, codes, scale, None, True, 128)
    q, s = Q.quantize_int8_rowwise(x.detach(), 128)
    assert torch.equal(y, Q.w8a8_int8_linear(q, s, codes, scale, out_dtype=BF16))
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], Q.int8_linear_grad_input(dy, codes, scale, True, 128))
    # near the linear over x itself: rows in 8 bits, at most half a step of a 127th of the largest value off, at random
    want = Q.int8_linear(x.detach(), codes, scale, convrot=True, convrot_groupsize=128)
    rel = float((y.detach().double() - want.double()).norm() / want.double().norm())
    assert rel < 2e-2, rel


def test_rows_far_apart():
    """Rows almost 2^24 bytes apart as they are, at 2^24 copied: the bits of packed rows.  (Sizes whose tiles are 256 x 256, K long and short.)"""
    Q = qlin()
    for k in (256, 3584):
        x, sx, w, sw = make(512, k, 32768, seed=k)
        want = Q.w8a8_int8_linear(x, sx, w, sw)
        buf = torch.empty(512 << 24, dtype=torch.int8, device=DEV)
        for ld in ((1 << 24) - 16, 1 << 24):
            far = buf.as_strided((512, k), (ld, 1))
            far.copy_(x)
            assert torch.equal(Q.w8a8_int8_linear(far, sx, w, sw), want)
            assert torch.equal(Q.w8a8_int8_linear(far[:40], sx[:40], w, sw), want[:40])
            assert torch.equal(Q.w8a8_int8_linear(far[:1], sx[:1], w[:100], sw[:100]), want[:1, :100])
