"""Outputs of the MLP side that are one of the call's inputs, through the C ABI: the bits of a call with memory of its own."""
import pytest
import torch
from mlp_ref import BF16, DEV, F16, F32, qlin, rand

pytestmark = pytest.mark.gpu
WIDTHS = [1, 7, 64, 1001, 4104, 8192, 16401, 33001]  # in registers and read twice; whole pieces and pieces that reach past the row


def call(name, *args):
    from qlin import _lib
    L = _lib.load()
    args = [_lib.desc(a) if torch.is_tensor(a) or a is None else a for a in args]
    assert getattr(L, name)(*args, _lib.stream_of(torch.device(DEV, 0))) == 0, L.qlin_last_error()


def rows(t, w, n, dtype, pad=0):
    """n tensors [t, w] of rows w + pad apart."""
    return [torch.cat([rand(t, w, seed=10 * w + i), torch.zeros(t, pad)], 1).to(dtype).to(DEV)[:, :w] for i in range(n)]


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("w", WIDTHS)
def test_norm(w, dtype, pad):
    for t in (1, 5):
        x, r, g = rows(t, w, 3, dtype, pad)
        g = g[0].clone()
        y, h = torch.empty_like(x), torch.empty_like(x)
        call("qlin_add_rms_norm", x, r, g, 1e-6, y, h)
        for ky, kh in (("x", None), (None, "r"), ("x", "r"), ("r", "x"), (None, "x"), ("r", None)):
            a = {"x": x.clone(), "r": r.clone(), None: torch.empty_like(x)}
            oy, oh = a[ky], a[kh] if kh else torch.empty_like(x)
            call("qlin_add_rms_norm", a["x"], a["r"], g, 1e-6, oy, oh)
            assert torch.equal(oy, y) and torch.equal(oh, h), (ky, kh)
        a = x.clone()
        call("qlin_add_rms_norm", x, None, g, 1e-6, y, None)
        call("qlin_add_rms_norm", a, None, g, 1e-6, a, None)
        assert torch.equal(a, y)
        for group in (0, 4):
            if group and w % group:
                continue
            q, s = torch.empty(t, w, dtype=torch.int8, device=DEV), torch.empty(t, 1, device=DEV)
            q2, s2 = torch.empty_like(q), torch.empty_like(s)
            call("qlin_add_rms_norm_int8", x, r, g, 1e-6, group, q, s, h)
            for over in (x, r):
                a, b = x.clone(), r.clone()
                oh = a if over is x else b
                call("qlin_add_rms_norm_int8", a, b, g, 1e-6, group, q2, s2, oh)
                assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(oh, h)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("t,w", [(3, 7), (900, 72), (5, 1001), (700, 4104), (300, 8192), (5, 16401), (300, 33001)])
def test_gradient_of_the_norm(t, w, dtype):
    from qlin import _lib
    dy, dh, h, g = rows(t, w, 4, dtype)
    g = g[0].clone()
    n = _lib.load().qlin_workspace_size(_lib.OP_ADD_RMS_NORM_GRAD, t, 0, w, 0, 0)
    room = torch.empty(n, dtype=torch.uint8, device=DEV)

    def grad(dy, dh, h, dx):
        dw = torch.empty_like(g)
        call("qlin_add_rms_norm_grad", dy, dh, h, g, 1e-6, dx, dw, room.data_ptr(), room.numel())
        return dx, dw

    want = grad(dy, dh, h, torch.empty_like(h))
    for i in range(3):
        a = [v.clone() for v in (dy, dh, h)]
        got = grad(*a, a[i])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i


@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("w", [1, 3, 7, 8, 1001, 4104, 33001])
def test_activation(w, dtype, pad):
    for t in (1, 300):
        gate, up, dy = rows(t, w, 3, dtype, pad)
        y, dg, du = (torch.empty_like(gate) for _ in range(3))
        call("qlin_gated_act", gate, up, 0, y)
        call("qlin_gated_act_grad", dy, gate, up, 1, dg, du)
        for i in range(2):
            a = [gate.clone(), up.clone()]
            call("qlin_gated_act", *a, 0, a[i])
            assert torch.equal(a[i], y)
        for i, j in ((1, 2), (2, 1), (0, 1), (0, 2), (1, 0), (2, 0)):
            a = [dy.clone(), gate.clone(), up.clone()]
            call("qlin_gated_act_grad", *a, 1, a[i], a[j])
            assert torch.equal(a[i], dg) and torch.equal(a[j], du), (i, j)


# tiles, rows of any alignment, the GEMM's shapes, rows that are copied, whole rounds and the rest (K short and long)
@pytest.mark.parametrize("m,k,n", [(1, 256, 40), (20, 512, 130), (333, 1024, 200), (20, 1000, 33), (64, 100, 70), (300, 1000, 264), (900, 1024, 4096),
                                   (2816, 128, 4096), (2080, 256, 8192), (2080, 3584, 8192)])
def test_product(m, k, n):
    from qlin import _lib
    gen = torch.Generator().manual_seed(m)
    x, w = (torch.randint(-127, 128, (r, k), generator=gen, dtype=torch.int8).to(DEV) for r in (m, n))
    sx, sw = torch.rand(m, 1, generator=gen).to(DEV), torch.rand(n, generator=gen).to(DEV) * k ** -0.5
    room = torch.empty(max(1, _lib.load().qlin_workspace_size(_lib.OP_W8A8_LINEAR, m, n, k, 0, 0)), dtype=torch.uint8, device=DEV)
    for dtype in (BF16, F32):
        for pad in (0, 5):
            r, = rows(m, n, 1, dtype, pad)
            y = torch.empty(m, n, dtype=dtype, device=DEV)
            call("qlin_w8a8_linear", x, sx, w, sw, None, r, None, y, room.data_ptr(), room.numel())
            a = torch.empty(m, n + pad, dtype=dtype, device=DEV)[:, :n]
            a.copy_(r)
            call("qlin_w8a8_linear", x, sx, w, sw, None, a, None, a, room.data_ptr(), room.numel())
            assert torch.equal(a, y)
