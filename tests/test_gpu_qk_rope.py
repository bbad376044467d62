"""Rotation of q and k by positions on several axes, the per-head norms with it, the form that writes a
paged cache and the gradients, against the formulas in float64 on the CPU.

Bounds.  Every output is rounded once: |err| <= u |y| with u = 2^-24, 2^-11, 2^-8 (fp32, fp16, bf16; half of the
smallest subnormal below their normal range).  The fp32 arithmetic before it: cos and sin to 2^-21, a sum of
squares of depth < 32 and a dozen products, together under 2^-18 of the pair's length.  The gradients add a second
sum of that depth: 2^-17 of |w g| + |x^| mean|w g x^|, times 1 / rms.  The weight gradients add up a few thousand
terms in partial sums: 2^-16 of the sum of the terms' sizes.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def qlin():
    import qlin as Q
    return Q


def rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def angles(positions, freq, axis):
    pos = positions.double() if positions.dim() == 2 else positions.double()[None]
    ax = torch.zeros(len(freq), dtype=torch.long) if axis is None else axis.long()
    return (pos[ax] * freq.double()[:, None]).T[:, None]  # [tokens, 1, pairs]


def halves(x, p, interleaved):
    return (x[..., 0:2 * p:2], x[..., 1:2 * p:2]) if interleaved else (x[..., :p], x[..., p:2 * p])


def joined(u, v, rest, interleaved):
    a = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([a, rest], -1)


def rotate(x, ang, interleaved):
    p = ang.shape[-1]
    u, v = halves(x, p, interleaved)
    c, s = ang.cos(), ang.sin()
    return joined(u * c - v * s, u * s + v * c, x[..., 2 * p:], interleaved)


def lengths_of_pairs(x, p, interleaved):
    """|(u, v)| at both values of each pair, |x| behind them."""
    u, v = halves(x, p, interleaved)
    n = (u * u + v * v).sqrt()
    return joined(n, n, x[..., 2 * p:].abs(), interleaved)


def normed(x, w, eps):
    unit = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return unit if w is None else unit * w.double()


def within(got, want, extra, what):
    got_d = got.double().cpu()
    tol = U[got.dtype] * want.abs() + extra + TINY[got.dtype]
    bad = ~((got_d - want).abs() <= tol)
    assert got_d.shape == want.shape and not bad.any(), \
        f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {((got_d - want).abs() / tol).max():.2f} of the bound"


def forward_ok(got, x, w, eps, ang, interleaved, what):
    y = x.double().cpu()
    if eps is not None:
        y = normed(y, w, eps)
    want = rotate(y, ang, interleaved)
    within(got, want, 2.0 ** -18 * lengths_of_pairs(y, ang.shape[-1], interleaved), what)


def grid_positions(axes, t, dtype=torch.int64, start=0):
    i = torch.arange(t)
    return torch.stack([(i // (7 ** a)) % 91 + start for a in range(axes)]).to(dtype)


# tokens, q heads, k heads, D, sizes per axis, interleaved
SHAPES = [
    (1, 32, 8, 128, (128,), False),       # one token of a decode step
    (1, 1, 1, 64, (64,), True),
    (5, 48, 48, 128, (16, 56, 56), True),  # image tokens
    (33, 3, 1, 128, (32, 48, 48), False),
    (7, 5, 5, 96, (24, 36, 36), True),
    (19, 6, 2, 80, (80,), False),
    (19, 6, 2, 80, (40,), False),         # half of each head rotates
    (9, 4, 4, 72, (24, 24, 24), True),    # pieces of 8 values
    (11, 2, 2, 64, (20, 24), False),      # 22 pairs: value by value
    (6, 3, 2, 7, (4,), True),             # odd heads
    (6, 3, 2, 5, (4,), False),
    (4, 2, 1, 1, (0,), False),            # nothing to rotate
    (17, 2, 2, 256, (256,), True),
    (3, 2, 2, 512, (512,), False),
    (3, 1, 2, 510, (254, 256), True),
    (301, 20, 4, 64, (64,), False),
    (2, 24, 24, 128, (0, 128), True),     # an axis that turns nothing
    (9000, 1, 2, 16, (16,), True),        # many tokens of few short heads
]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("t,hq,hk,d,sizes,inter", SHAPES)
def test_rotation_and_norms(t, hq, hk, d, sizes, inter, dtype):
    Q = qlin()
    freq, axis = Q.rope_frequencies(sizes)
    pos = grid_positions(len(sizes), t)
    q, k = rand(t, hq, d, seed=1, dtype=dtype), rand(t, hk, d, seed=2, dtype=dtype)
    wq, wk = 1 + 0.2 * rand(d, seed=3), (1 + 0.2 * rand(d, seed=4)).to(dtype)
    ang = angles(pos, freq, axis)
    dev = [x.to(DEV) for x in (q, k, pos, freq, axis)]
    yq, yk = Q.axis_rope(*dev, interleaved=inter)
    forward_ok(yq, q, None, None, ang, inter, "rotated q")
    forward_ok(yk, k, None, None, ang, inter, "rotated k")
    bq, bk = Q.axis_rope(yq, None, *dev[2:], interleaved=inter, inverse=True)
    assert bk is None
    forward_ok(bq, yq, None, None, -ang, inter, "turned back")
    nq, nk = Q.qk_norm_rope(dev[0], dev[1], wq.to(DEV), wk.to(DEV), *dev[2:], eps=1e-5, interleaved=inter)
    forward_ok(nq, q, wq, 1e-5, ang, inter, "q")
    forward_ok(nk, k, wk, 1e-5, ang, inter, "k")
    nq, nk = Q.qk_norm_rope(dev[0], None, None, None, *dev[2:], interleaved=inter)
    assert nk is None
    forward_ok(nq, q, None, 1e-6, ang, inter, "q without a weight")


@pytest.mark.parametrize("pdtype", [torch.int32, torch.int64, F32])
@pytest.mark.parametrize("start", [0, 4095, 1 << 20])
def test_positions(pdtype, start):
    """Far positions lose nothing: the angle is formed in 64 bits."""
    Q = qlin()
    t, d = 40, 128
    freq, axis = Q.rope_frequencies((64, 64), theta=5e5, shared=True)
    pos = grid_positions(2, t, pdtype, start)
    if pdtype == F32:
        pos = pos + 0.25
    q = rand(t, 2, d, seed=5)
    y, _ = Q.axis_rope(q.to(DEV), None, pos.to(DEV), freq.to(DEV), axis.to(DEV))
    forward_ok(y, q, None, None, angles(pos, freq, axis), False, "q")
    y, _ = Q.axis_rope(q.to(DEV), None, pos[1].to(DEV), freq.to(DEV))  # one axis as a vector
    forward_ok(y, q, None, None, angles(pos[1], freq, None), False, "one axis")
    wide = torch.zeros(2, 3 * t, dtype=pdtype)
    wide[:, ::3] = pos
    y2, _ = Q.axis_rope(q.to(DEV), None, wide.to(DEV)[:, ::3], freq.to(DEV), axis.to(DEV))
    y1, _ = Q.axis_rope(q.to(DEV), None, pos.to(DEV), freq.to(DEV), axis.to(DEV))
    assert torch.equal(y1, y2)


@pytest.mark.parametrize("t,d", [(70000, 512), (200000, 128)])
def test_many_tokens_of_one_head(t, d):
    """A workgroup's rows are of as many tokens as its LDS holds cosines of (the bounds of test_rotation_and_norms, in float64
    on the GPU)."""
    Q = qlin()
    freq, _ = Q.rope_frequencies(d, device=DEV)
    pos = torch.arange(t, device=DEV)
    q = torch.randn(t, 1, d, generator=torch.Generator(DEV).manual_seed(1), device=DEV, dtype=F32).half()
    y, _ = Q.axis_rope(q, None, pos, freq)
    dq, _, _, _ = Q.qk_norm_rope_grad(q, None, q, None, None, None, pos, freq)
    ang = (pos.double()[:, None] * freq.double())[:, None]
    x = q.double()
    assert bool(((y.double() - rotate(x, ang, False)).abs() <= 2.0 ** -11 * rotate(x, ang, False).abs()
                 + 2.0 ** -18 * lengths_of_pairs(x, d // 2, False) + TINY[F16]).all())
    rstd = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    g, unit, size = rotate(x, -ang, False), x * rstd, lengths_of_pairs(x, d // 2, False)
    want = rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
    tol = 2.0 ** -11 * want.abs() + 2.0 ** -17 * rstd * (size + unit.abs() * (size * unit.abs()).mean(-1, keepdim=True)) + TINY[F16]
    assert bool(((dq.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("d,sizes,inter", [(128, (64, 64), True), (128, (128,), False), (72, (24, 48), True), (72, (72,), False)])
def test_large_calls_are_their_parts(d, sizes, inter, dtype):
    """Rows of more than 32 MB are read in another way than small ones: the same bits as token by token slices."""
    Q = qlin()
    h, hk = 12, 4
    t = (40 << 20) // ((h + hk) * d * (4 if dtype == F32 else 2))
    freq, axis = (x.to(DEV) for x in Q.rope_frequencies(sizes))
    pos = grid_positions(len(sizes), t).to(DEV)
    gen = torch.Generator(DEV).manual_seed(1)
    qkv, g = (torch.randn(t, h + hk, d, generator=gen, device=DEV).to(dtype) for _ in range(2))
    w = (1 + 0.2 * rand(d, seed=3)).to(DEV)
    run = lambda a, b: Q.qk_norm_rope(qkv[a:b, :h], qkv[a:b, h:], w, w, pos[:, a:b], freq, axis, interleaved=inter)
    grad = lambda a, b: Q.qk_norm_rope_grad(g[a:b, :h], g[a:b, h:], qkv[a:b, :h], qkv[a:b, h:], w, w, pos[:, a:b], freq, axis,
                                            interleaved=inter)[:2]
    for call in (run, grad):
        whole, parts = call(0, t), [call(a, min(a + 501, t)) for a in range(0, t, 501)]
        for i in range(2):
            assert torch.equal(whole[i], torch.cat([p[i] for p in parts]))


def test_axis_entries_outside_count_as_the_nearest():
    Q = qlin()
    freq, axis = Q.rope_frequencies((32, 32))
    pos = grid_positions(2, 9).to(DEV)
    q = rand(9, 2, 64, seed=6).to(DEV)
    a, _ = Q.axis_rope(q, None, pos, freq.to(DEV), axis.to(DEV))
    axis = torch.where(axis == 0, -5, 1000).int()
    b, _ = Q.axis_rope(q, None, pos, freq.to(DEV), axis.to(DEV))
    assert torch.equal(a, b)


@pytest.mark.parametrize("d,hq,hk", [(128, 8, 2), (80, 3, 1), (36, 2, 2)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_strides(d, hq, hk, dtype):
    """Slices of a fused projection, heads before tokens, rows off the 16-byte grid, a strided last dimension and
    extra leading dimensions give the bits of contiguous tensors."""
    Q = qlin()
    t = 23
    freq, axis = (x.to(DEV) for x in Q.rope_frequencies((d // 2, d // 2 - d // 2 % 2)))
    freq, axis = freq[: d // 2], axis[: d // 2]
    pos = grid_positions(2, t).to(DEV)
    w = (1 + 0.2 * rand(d, seed=1)).to(DEV)
    qkv = rand(t, hq + 2 * hk, d, seed=2, dtype=dtype).to(DEV)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    want = Q.qk_norm_rope(q.contiguous(), k.contiguous(), w, w, pos, freq, axis)

    def same(got):
        for g, x in zip(got, want):
            assert torch.equal(g.reshape(x.shape), x)

    same(Q.qk_norm_rope(q, k, w, w, pos, freq, axis))
    same(Q.qk_norm_rope(q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1), w, w,
                        pos, freq, axis))
    odd = torch.zeros(t, hq + 2 * hk, d + 3, dtype=dtype, device=DEV)
    odd[..., 1:d + 1] = qkv
    same(Q.qk_norm_rope(odd[:, :hq, 1:d + 1], odd[:, hq:hq + hk, 1:d + 1], w, w, pos, freq, axis))
    wide = qkv.repeat_interleave(2, -1)[..., ::2]
    assert wide.stride(-1) == 2
    same(Q.qk_norm_rope(wide[:, :hq], wide[:, hq:hq + hk], w.repeat_interleave(2)[::2], w, pos, freq, axis))
    got = Q.qk_norm_rope(q.unsqueeze(0), k.unsqueeze(0), w, w, pos, freq, axis)
    assert got[0].shape == (1, t, hq, d)
    same(got)


@pytest.mark.parametrize("t", [0, 1])
def test_no_tokens_and_no_heads(t):
    Q = qlin()
    freq, axis = (x.to(DEV) for x in Q.rope_frequencies((64,)))
    pos = torch.zeros(1, t, dtype=torch.int64, device=DEV)
    q, k = torch.ones(t, 4, 64, device=DEV), torch.ones(t, 0, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    a, b = Q.qk_norm_rope(q, k, w, w, pos, freq, axis)
    assert a.shape == q.shape and b.shape == k.shape
    dq, dk, dwq, dwk = Q.qk_norm_rope_grad(q, k, q, k, w, w, pos, freq, axis)
    assert dq.shape == q.shape and dk.shape == k.shape and bool((dwk == 0).all())
    if t == 0:
        assert bool((dwq == 0).all())


def test_rows_that_are_not_finite():
    """Zero rows give zeros; an infinity or a NaN stays within its own head."""
    Q = qlin()
    freq, axis = (x.to(DEV) for x in Q.rope_frequencies((128,)))
    q = rand(3, 4, 128, seed=7, dtype=BF16).to(DEV)
    q[0, 1] = 0
    q[1, 2, 5] = float("nan")
    q[2, 3, 9] = float("inf")
    pos = torch.arange(3, device=DEV)
    y, _ = Q.qk_norm_rope(q, None, None, None, pos, freq)
    assert bool((y[0, 1] == 0).all()) and bool(y[1, 2].isnan().all()) and not bool(y[2, 3].isfinite().all())
    rest = torch.ones(3, 4, dtype=torch.bool)
    rest[1, 2] = rest[2, 3] = False
    assert bool(y[rest.to(DEV)].isfinite().all())


# ------------------------------------------------------------------------------------------------ the cache

@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("t,hq,hk,d,sizes,inter,page,dtype", [
    (1, 32, 8, 128, (128,), False, 16, BF16),
    (37, 10, 2, 128, (64,), False, 16, F16),
    (50, 4, 4, 80, (80,), True, 7, BF16),
    (21, 2, 1, 20, (12,), False, 1, F32),
    (130, 5, 1, 256, (256,), False, 100, F16),
])
def test_store(t, hq, hk, d, sizes, inter, page, dtype, layout):
    """Stored k and v are those of the plain call, in the slots' places; every other place keeps its bits."""
    Q = qlin()
    freq, axis = (x.to(DEV) for x in Q.rope_frequencies(sizes))
    pos = torch.arange(t, device=DEV, dtype=torch.int32) + 100
    qkv = rand(t, hq + 2 * hk, d, seed=8, dtype=dtype).to(DEV)
    q, k, v = qkv.split((hq, hk, hk), 1)
    w = (1 + 0.2 * rand(d, seed=9)).to(DEV)
    blocks = t // page + 3
    shape = (blocks, page, hk, d) if layout == "token" else (blocks, hk, page, d)

    def cache(seed):
        c = rand(*shape, seed=seed, dtype=dtype).to(DEV)
        return c if layout == "token" else c.transpose(1, 2)

    slots = torch.randperm(blocks * page, generator=torch.Generator().manual_seed(10))[:t].to(DEV)
    if t > 8:  # no place: padding, and slots past the cache
        slots[3], slots[5], slots[7] = -1, blocks * page, 1 << 40
    for sl, eps in ((slots, 1e-6), (slots.clamp(max=2 ** 31 - 1).int(), None)):
        kc, vc = cache(11), cache(12)
        wantk, wantv = kc.clone(), vc.clone()
        weights = (None, None) if eps is None else (w, w)
        if eps is None:
            yq, yk = Q.axis_rope(q, k, pos, freq, axis, interleaved=inter)
        else:
            yq, yk = Q.qk_norm_rope(q, k, w, w, pos, freq, axis, eps=eps, interleaved=inter)
        for i, s in enumerate(sl.tolist()):
            if 0 <= s < blocks * page:
                wantk[s // page, s % page], wantv[s // page, s % page] = yk[i], v[i]
        got = Q.qk_norm_rope_store(q, k, v, *weights, pos, freq, sl, kc, vc, axis, eps=eps, interleaved=inter)
        assert torch.equal(got, yq) and torch.equal(kc, wantk) and torch.equal(vc, wantv)


# ------------------------------------------------------------------------------------------------ gradients

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("t,hq,hk,d,sizes,inter", SHAPES + [(700, 12, 3, 128, (16, 56, 56), True)])
def test_gradients(t, hq, hk, d, sizes, inter, dtype):
    Q = qlin()
    eps = 1e-3
    freq, axis = Q.rope_frequencies(sizes)
    pos = grid_positions(len(sizes), t)
    ang = angles(pos, freq, axis)
    x = [rand(t, h, d, seed=13 + h, dtype=dtype) for h in (hq, hk)]
    g = [rand(t, h, d, seed=93 + h, dtype=dtype) for h in (hq, hk)]
    w = [1 + 0.2 * rand(d, seed=15), (1 + 0.2 * rand(d, seed=16)).to(dtype)]
    got = Q.qk_norm_rope_grad(*(a.to(DEV) for a in (*g, *x, *w, pos, freq, axis)), eps=eps, interleaved=inter)
    for i, name in enumerate("qk"):
        xd, gd, wd = x[i].double(), g[i].double(), w[i].double()
        leaves = xd.clone().requires_grad_(True), wd.clone().requires_grad_(True)
        dx, dw = torch.autograd.grad(rotate(normed(leaves[0], leaves[1], eps), ang, inter), leaves, gd)
        size = lengths_of_pairs(gd, ang.shape[-1], inter)  # |g| cannot grow beyond the pair's
        rstd = (xd.square().mean(-1, keepdim=True) + eps).rsqrt()
        unit = (xd * rstd).abs()
        wg = wd.abs() * size
        within(got[i], dx, 2.0 ** -17 * rstd * (wg + unit * (wg * unit).mean(-1, keepdim=True)), f"d{name}")
        within(got[2 + i], dw, 2.0 ** -16 * (size * unit).sum((0, 1)), f"d{name}_weight")
        assert got[2 + i].dtype == w[i].dtype
    # frozen weights, no weights and no k leave the same dq
    dev = [a.to(DEV) for a in (pos, freq, axis)]
    f = Q.qk_norm_rope_grad(g[0].to(DEV), None, x[0].to(DEV), None, w[0].to(DEV), None, *dev, eps=eps, interleaved=inter,
                            weight_grads=False)
    assert torch.equal(f[0], got[0]) and f[1] is None and f[2] is None and f[3] is None


def test_gradients_against_differences():
    """The trainable wrapper against central differences of the float64 forward, one direction at a time: step 1e-5
    leaves 1e-10 (truncation) and 1e-11 (rounding); the fp32 gradients are held to 1e-5 of their size."""
    Q = qlin()
    t, hq, hk, d, eps = 6, 3, 2, 48, 1e-6
    freq, axis = Q.rope_frequencies((16, 32))
    pos = grid_positions(2, t)
    ang = angles(pos, freq, axis)
    leaves = [rand(t, hq, d, seed=21), rand(t, hk, d, seed=22), 1 + 0.2 * rand(d, seed=23), 1 + 0.2 * rand(d, seed=24)]
    gq, gk = rand(t, hq, d, seed=25), rand(t, hk, d, seed=26)

    def loss(q, k, wq, wk):
        return ((rotate(normed(q, wq, eps), ang, True) * gq.double()).sum()
                + (rotate(normed(k, wk, eps), ang, True) * gk.double()).sum())

    dev = [a.to(DEV).requires_grad_(True) for a in leaves]
    yq, yk = Q.qk_norm_rope_trainable(*dev, pos.to(DEV), freq.to(DEV), axis.to(DEV), eps, True)
    grads = torch.autograd.grad((yq, yk), dev, (gq.to(DEV), gk.to(DEV)))
    for i, grad in enumerate(grads):
        for seed in range(4):
            step = rand(*leaves[i].shape, seed=30 + seed).double()
            at = [a.double() for a in leaves]
            hi, lo = list(at), list(at)
            hi[i], lo[i] = at[i] + 1e-5 * step, at[i] - 1e-5 * step
            want = float(loss(*hi) - loss(*lo)) / 2e-5
            got = float((grad.double().cpu() * step).sum())
            size = float((grad.double().cpu() * step).abs().sum())
            assert abs(got - want) <= 1e-5 * size + 1e-8, (i, seed, got, want)


def test_trainable_wrappers():
    Q = qlin()
    t, d = 12, 64
    freq, axis = (a.to(DEV) for a in Q.rope_frequencies((32, 32)))
    pos = grid_positions(2, t).to(DEV)
    q, k = (rand(t, h, d, seed=h, dtype=BF16).to(DEV).requires_grad_(True) for h in (4, 2))
    wq, wk = (torch.ones(d, device=DEV, dtype=BF16).requires_grad_(r) for r in (True, False))
    yq, yk = Q.qk_norm_rope_trainable(q, k, wq, wk, pos, freq, axis)
    want = Q.qk_norm_rope(q.detach(), k.detach(), wq.detach(), wk, pos, freq, axis)
    assert torch.equal(yq, want[0]) and torch.equal(yk, want[1])
    # a broadcast gradient (stride 0) and one of an unused output (zeros)
    (dq, dwq) = torch.autograd.grad(yq.sum(), (q, wq))
    ones = torch.ones_like(yq)
    ref = Q.qk_norm_rope_grad(ones, torch.zeros_like(yk), q.detach(), k.detach(), wq.detach(), wk, pos, freq, axis)
    assert torch.equal(dq, ref[0]) and torch.equal(dwq, ref[2]) and bool((ref[1] == 0).all())
    yq, yk = Q.axis_rope_trainable(q, k, pos, freq, axis)
    g = rand(t, 2, d, seed=40, dtype=BF16).to(DEV)
    (dk,) = torch.autograd.grad(yk, k, g)
    assert torch.equal(dk, Q.axis_rope(g, None, pos, freq, axis, inverse=True)[0])


def test_gradient_of_weights_is_the_same_every_time():
    Q = qlin()
    t, d = 500, 128
    freq, axis = (a.to(DEV) for a in Q.rope_frequencies((128,)))
    pos = torch.arange(t, device=DEV)
    q, g = rand(t, 24, d, seed=1).to(DEV), rand(t, 24, d, seed=2).to(DEV)
    w = torch.ones(d, device=DEV)
    first = Q.qk_norm_rope_grad(g, None, q, None, w, None, pos, freq)[2]
    for _ in range(5):
        assert torch.equal(first, Q.qk_norm_rope_grad(g, None, q, None, w, None, pos, freq)[2])


# ------------------------------------------------------------------------------------------------ routes, streams, graphs

def test_routes_agree(monkeypatch):
    from qlin import ops
    Q = qlin()
    t, d = 15, 96
    freq, axis = (a.to(DEV) for a in Q.rope_frequencies((48, 48)))
    pos = grid_positions(2, t).to(DEV)
    q, k, v = rand(t, 9, d, seed=1, dtype=F16).to(DEV).split((5, 2, 2), 1)
    w = torch.ones(d, device=DEV, dtype=F16)
    slots = torch.arange(t, device=DEV)

    def everything():
        kc, vc = torch.zeros(2, 8, 2, d, device=DEV, dtype=F16), torch.zeros(2, 8, 2, d, device=DEV, dtype=F16)
        out = [*Q.axis_rope(q, k, pos, freq, axis), *Q.qk_norm_rope(q, k, w, None, pos, freq, axis, interleaved=True)]
        out.append(Q.qk_norm_rope_store(q, k, v, w, w, pos, freq, slots, kc, vc, axis))
        out += [kc, vc, *Q.qk_norm_rope_grad(q, k, q, k, w, None, pos, freq, axis)]
        return out

    assert ops._FAST is not None
    fast = everything()
    monkeypatch.setattr(ops, "_FAST", None)
    for a, b in zip(fast, everything()):
        assert (a is None and b is None) or torch.equal(a, b)


def test_another_stream_and_a_graph():
    Q = qlin()
    t, d = 64, 128
    freq, axis = (a.to(DEV) for a in Q.rope_frequencies((128,)))
    pos = torch.arange(t, device=DEV)
    q, k = rand(t, 8, d, seed=1, dtype=BF16).to(DEV), rand(t, 2, d, seed=2, dtype=BF16).to(DEV)
    w = torch.ones(d, device=DEV, dtype=BF16)
    want = [*Q.qk_norm_rope(q, k, w, w, pos, freq), *Q.qk_norm_rope_grad(q, k, q, k, w, w, pos, freq)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [*Q.qk_norm_rope(q, k, w, w, pos, freq), *Q.qk_norm_rope_grad(q, k, q, k, w, w, pos, freq)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [*Q.qk_norm_rope(q, k, w, w, pos, freq), *Q.qk_norm_rope_grad(q, k, q, k, w, w, pos, freq)]
    for i in range(4):
        q.copy_(rand(t, 8, d, seed=50 + i, dtype=BF16))
        graph.replay()
        want = [*Q.qk_norm_rope(q, k, w, w, pos, freq), *Q.qk_norm_rope_grad(q, k, q, k, w, w, pos, freq)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
