"""Edges of the attention side: weights far below a row's largest, infinities, values that pass a rotation by, empty heads,
plans that are kept and saved, second derivatives, sizes at the ends of their ranges."""
import io

import pytest
import torch
from test_gpu_paged_attention import BF16, DEV, F16, check, make
from test_gpu_paged_plan import check as check_plan
from test_gpu_qk_rope import angles, grid_positions, rand, rotate

pytestmark = pytest.mark.gpu


def qlin():
    import qlin as Q
    return Q


# lengths, heads, kv heads, D, page, table width
PATHS = [
    ([500], 8, 2, 128, 16, 32),            # a workgroup takes the row
    ([250] * 200, 8, 8, 128, 16, 16),      # a wave does
    ([16384, 2000], 8, 2, 128, 16, None),  # split and joined
    ([2000], 8, 2, 128, 10, None),         # pages that end inside tiles
    ([500], 16, 1, 64, 16, 32),            # 9 to 16 heads of a kv head
    ([250] * 400, 48, 4, 128, 16, 16),
    ([16384], 12, 1, 128, 16, None),
    ([3000], 16, 1, 256, 12, None),
]


@pytest.mark.parametrize("gap", [14.0, 16.0, 17.5, 19.0, 24.0])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page,width", PATHS)
def test_a_token_far_above_the_rest(lengths, heads, kv_heads, dim, page, width, gap):
    """A row's first token `gap` nats above the others, with a value of zero, as trained heads have it: the output is what the
    others' small weights add up to, within the bound of test_gpu_paged_attention (fp16; bf16 has fp32's exponents)."""
    q, k, v, table, n = make(lengths, heads, kv_heads, dim, page, F16, width=width)
    q.zero_()
    q[..., 0] = 1
    k[..., 0] = torch.rand(k.shape[:3], generator=torch.Generator().manual_seed(5)).half().to(DEV) - 0.5
    v.copy_(1000 + 100 * v)
    first = table[:, 0].long()
    k[first, 0, :, 0] = gap
    v[first, 0] = 0
    s = (q, k, v, table, n)
    check(qlin().paged_attention(*s, scale=1.0), *s, scale=1.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page,width", PATHS + [([1], 8, 2, 128, 16, 4)])
def test_infinities_in_values(lengths, heads, kv_heads, dim, page, width, dtype):
    """An infinite value gives its infinity, opposite ones and a NaN give NaN, and no other value of the row changes."""
    q, k, v, table, n = make(lengths, heads, kv_heads, dim, page, dtype, width=width)
    inf, b, last = float("inf"), len(lengths) - 1, lengths[-1] - 1
    first, end = int(table[b, 0]), int(table[b, last // page])
    plain = v.clone()
    plain[first, 0, 0, 3:8] = 0
    plain[end, last % page, 0, 6] = 0
    v[first, 0, 0, 3:8] = torch.tensor([inf, -inf, inf, inf, float("nan")], dtype=dtype, device=DEV)
    v[end, last % page, 0, 6] = -inf
    got, want = (qlin().paged_attention(q, k, x, table, n) for x in (v, plain))
    check(want, q, k, plain, table, n)
    heads_of_0 = heads // kv_heads
    assert bool((got[b, :heads_of_0, 3] == inf).all()) and bool((got[b, :heads_of_0, 4] == -inf).all())
    assert bool((got[b, :heads_of_0, 5] == inf).all()) and bool(got[b, :heads_of_0, 7].isnan().all())
    sixth = got[b, :heads_of_0, 6]
    assert bool((sixth == -inf).all() if last == 0 else sixth.isnan().all())
    want[b, :heads_of_0, 3:8] = got[b, :heads_of_0, 3:8] = 0
    assert torch.equal(got, want)


def same_values(a, b):
    """Equal values, NaN where NaN is, zeros of the same sign."""
    return a.shape == b.shape and bool((((a == b) & (a.signbit() == b.signbit())) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rotated", [(128, 64), (128, 0), (72, 24), (20, 12), (7, 4)])
def test_values_behind_the_rotation_pass_as_they_are(d, rotated, inter, dtype):
    """Whatever they are, and without any effect on one another."""
    Q = qlin()
    t, h = 5, 3
    freq, _ = Q.rope_frequencies(rotated, device=DEV)
    pos = torch.arange(t, device=DEV)
    q = rand(t, h, d, seed=1, dtype=dtype).to(DEV)
    clean = Q.axis_rope(q, None, pos, freq, interleaved=inter)[0]
    q[:, 0, rotated + 1], q[:, 1, d - 1], q[:, 2, rotated] = float("nan"), float("-inf"), -0.0
    y = Q.axis_rope(q, None, pos, freq, interleaved=inter)[0]
    assert same_values(y[..., rotated:], q[..., rotated:]) and torch.equal(y[..., :rotated], clean[..., :rotated])
    # with the norms an infinite value makes its row's others zero; a NaN in a gradient stays in its own weight's sum
    y = Q.qk_norm_rope(q, None, None, None, pos, freq, interleaved=inter)[0][:, 1]
    assert bool(y[:, d - 1].isnan().all()) and bool((y[:, : d - 1] == 0).all())
    x, g, w = rand(t, h, d, seed=2, dtype=dtype).to(DEV), rand(t, h, d, seed=3, dtype=dtype).to(DEV), torch.ones(d, device=DEV)
    g[2, 1, rotated + 1] = float("nan")
    dw = Q.qk_norm_rope_grad(g, None, x, None, w, None, pos, freq, interleaved=inter)[2]
    assert dw.isnan().nonzero().flatten().tolist() == [rotated + 1]


def routes(monkeypatch):
    from qlin import ops
    assert ops._FAST is not None
    yield "C++"
    monkeypatch.setattr(ops, "_FAST", None)
    yield "ctypes"


def test_no_heads_in_more_dimensions(monkeypatch):
    Q = qlin()
    freq, pos, w = torch.ones(32, device=DEV), torch.zeros(6, dtype=torch.int64, device=DEV), torch.ones(64, device=DEV)
    slots, cache = torch.arange(6, device=DEV), torch.zeros(1, 16, 0, 64, device=DEV)
    for route in routes(monkeypatch):
        for hq, hk, d in ((4, 0, 64), (0, 2, 64), (0, 0, 64), (4, 2, 0)):
            q, k = torch.ones(2, 3, hq, d, device=DEV), torch.ones(2, 3, hk, d, device=DEV)
            f, v = (freq, w) if d else (freq[:0], w[:0])
            for got in (Q.axis_rope(q, k, pos, f), Q.qk_norm_rope(q, k, v, v, pos, f),
                        Q.qk_norm_rope_grad(q, k, q, k, v, v, pos, f)[:2]):
                assert got[0].shape == q.shape and got[1].shape == k.shape, route
            if hk == 0:
                assert Q.qk_norm_rope_store(q, k, k, v, v, pos, f, slots, cache, cache).shape == q.shape


def test_heads_of_no_values_are_refused(monkeypatch):
    Q = qlin()
    z = lambda *s: torch.zeros(s, dtype=F16, device=DEV)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)
    for _ in routes(monkeypatch):
        with pytest.raises(Q.NoCapableBackendError):
            Q.paged_attention(z(2, 8, 0), z(5, 16, 2, 0), z(5, 16, 2, 0), i(2, 4), i(2))
        with pytest.raises(ValueError):
            Q.paged_attention(z(), z(5, 16, 2, 64), z(5, 16, 2, 64), i(2, 4), i(2))


def test_a_plan_is_saved_and_its_lengths_kept(monkeypatch):
    """A plan's fields can be saved together, and a field that is kept keeps nothing of the others but their request tables."""
    Q = qlin()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    for route in routes(monkeypatch):
        table = torch.zeros(3, 400, dtype=torch.int32, device=DEV)
        plan = Q.paged_plan(ints([5, 0, 31]), ints([2000, 300, 1]), table, ints(list(range(200))), 16, 2301)
        f = io.BytesIO()
        torch.save(plan._asdict(), f)
        f.seek(0)
        back = torch.load(f, weights_only=True)
        assert all(torch.equal(back[n], getattr(plan, n)) for n in plan._fields), route
        for n in ("starts", "lengths", "used"):
            assert getattr(plan, n).untyped_storage().nbytes() <= 512, (route, n)


def test_a_wrong_length_over_pages_of_one_token():
    """2^31 - 1 new tokens in a table that holds 3 of them a row: the rest has no entry and takes no time either."""
    top = 2 ** 31 - 1
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    table = torch.full((3, 3), -7, dtype=torch.int32, device=DEV)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(2):
        begin.record()
        plan = qlin().paged_plan(ints([1, 2, 0]), ints([1, top, 2]), table, ints([10, 11, 12, 13]), 1, 6)
        end.record()
    torch.cuda.synchronize()
    assert table.tolist() == [[-7, 10, -7], [-7, -7, 11], [-1, -1, -7]]
    assert plan.starts.tolist() == [0, 1, top, top] and plan.used.tolist() == [top] and plan.lengths.tolist() == [2, top, 2]
    assert plan.slots.tolist() == [10, 11, -1, -1, -1, -1] and plan.rows.tolist() == [0, 1, 1, 1, 1, 1]
    assert begin.elapsed_time(end) < 50.0


@pytest.mark.parametrize("width", [0, 1, 5, 40])
@pytest.mark.parametrize("page", [1, 3, 16])
def test_plans_of_rows_that_are_too_short(page, width):
    import random
    r = random.Random(page * 100 + width)
    context, added = [r.randrange(60) for _ in range(70)], [r.choice((0, 1, r.randrange(90))) for _ in range(70)]
    for pages in (0, 17, 6000):
        check_plan(context, added, page, width, list(range(1000, 1000 + pages)), sum(added) + 5)


def test_second_derivatives():
    """The rotation's gradient has a gradient (by the outputs' gradients; the rotation is linear); the norms' has none and says so."""
    Q = qlin()
    t, h, d = 6, 2, 32
    freq, axis = Q.rope_frequencies((16, 16))
    pos = grid_positions(2, t)
    ang = angles(pos, freq, axis)
    x, scale = rand(t, h, d, seed=1), rand(t, h, d, seed=2)

    def penalty(rope, x, scale):
        y = rope(x)
        (g,) = torch.autograd.grad((y ** 3 * scale).sum(), x, create_graph=True)
        return torch.autograd.grad((g ** 2).sum(), x)[0]

    dev = [a.to(DEV) for a in (pos, freq, axis)]
    got = penalty(lambda a: Q.axis_rope_trainable(a, None, *dev)[0], x.to(DEV).requires_grad_(True), scale.to(DEV))
    want = penalty(lambda a: rotate(a, ang, False), x.double().requires_grad_(True), scale.double())
    assert float((got.double().cpu() - want).norm() / want.norm()) < 1e-5  # five fp32 stages of 2^-22 at most each
    with pytest.raises(RuntimeError):
        penalty(lambda a: Q.qk_norm_rope_trainable(a, None, None, None, *dev)[0], x.to(DEV).requires_grad_(True), scale.to(DEV))


def test_frozen_weights_have_no_gradient_formed(monkeypatch):
    from qlin import attention
    Q = qlin()
    t, d = 12, 64
    freq, pos = Q.rope_frequencies(64, device=DEV)[0], torch.arange(t, device=DEV)
    real, formed = attention.qk_norm_rope_grad, []

    def grad(*a, **k):
        out = real(*a, **k)
        formed.append([x is not None for x in out[2:]])
        return out

    monkeypatch.setattr(attention, "qk_norm_rope_grad", grad)
    q, k = (rand(t, h, d, seed=h).to(DEV).requires_grad_(True) for h in (4, 2))
    for learn in ((True, False), (False, True), (False, False), (True, True)):
        w = [torch.ones(d, device=DEV).requires_grad_(r) for r in learn]
        yq, yk = Q.qk_norm_rope_trainable(q, k, *w, pos, freq)
        (yq.square().sum() + yk.square().sum()).backward()
        assert formed.pop() == list(learn) and [x.grad is not None for x in w] == list(learn)
    for route in routes(monkeypatch):
        w = torch.ones(d, device=DEV)
        a = [x.detach() for x in (q, k, q, k)]
        both = real(*a, w, w, pos, freq)
        for flags in ((True, False), (False, True), (False, False)):
            out = real(*a, w, w, pos, freq, weight_grads=flags)
            for i in range(2):
                assert torch.equal(out[2 + i], both[2 + i]) if flags[i] else out[2 + i] is None, (route, flags)


def test_the_gradient_of_q_alone_takes_no_longer_than_with_k():
    Q = qlin()
    t, h, d = 9504, 40, 128
    freq, pos = Q.rope_frequencies(d, device=DEV)[0], torch.arange(t, device=DEV)
    x, g = (torch.randn(t, h, d, device=DEV, dtype=BF16) for _ in range(2))
    w = torch.ones(d, device=DEV)

    def us(k):
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            Q.qk_norm_rope_grad(g, g if k else None, x, x if k else None, w, w if k else None, pos, freq)
            b.record()
            b.synchronize()
            times.append(1000 * a.elapsed_time(b))
        return min(times)

    both, alone = us(True), us(False)
    assert alone < both, (alone, both)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", [
    ([4097, 20, 9000], 16, 1, 128, 16),    # split and joined
    ([3000, 5], 17, 1, 64, 16),            # two groups of a kv head, 9 and 8 heads
    ([3000, 70], 49, 1, 128, 16),          # four, the last one short
    ([300, 2000], 16, 1, 256, 16),
    ([300, 2000], 12, 1, 256, 100),
    ([257, 3000], 16, 1, 128, 12),
    ([100, 31], 34, 2, 64, 7),
])
def test_many_heads_of_a_kv_head(lengths, heads, kv_heads, dim, page, layout, dtype):
    s = make(lengths, heads, kv_heads, dim, page, dtype, layout)
    check(qlin().paged_attention(*s), *s)
    check(qlin().paged_attention(*s, window=290), *s, window=290)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_many_short_rows_of_many_heads(dtype):
    s = make([(i * 53) % 120 for i in range(300)], 64, 4, 256, 16, dtype)
    check(qlin().paged_attention(*s), *s)


@pytest.mark.parametrize("page,w", [(1 << 30, 2), (0x7FFFFF80, 1), (100, 0x7FFFFFFF // 100 + 1)])
def test_positions_to_the_end_of_32_bits(page, w):
    """A window at the end of a row of 2^30 tokens and more (every place of a block is the same memory)."""
    d, blocks = 64, 2
    k, v = (torch.randn(blocks, d, generator=torch.Generator().manual_seed(i)).half().to(DEV) for i in range(2))
    q = torch.randn(1, 4, d, generator=torch.Generator().manual_seed(2)).half().to(DEV)
    kc, vc = (x.as_strided((blocks, page, 1, d), (d, 0, d, 1)) for x in (k, v))
    table = torch.zeros(1, w, dtype=torch.int32, device=DEV)
    table[0, -1 if w < 8 else -4:] = 1
    most = 0x7FFFFF00  # positions that a kernel's tiles can count
    length = (1 << 30) + 5 if w == 2 else most - 3
    out = qlin().paged_attention(q, kc, vc, table, torch.tensor([length], dtype=torch.int32, device=DEV), window=5)
    assert torch.equal(out, v[1].expand(1, 4, d))


def test_more_workgroups_than_a_launch_has_threads_for():
    """1024 rows of 16640 kv heads are more than 2^24 workgroups of 256 threads."""
    rows, h, d = 1024, 16640, 8
    k, v = (torch.randn(1, 8, h, d, generator=torch.Generator(DEV).manual_seed(i), device=DEV).half() for i in range(2))
    q = torch.randn(rows, h, d, generator=torch.Generator(DEV).manual_seed(2), device=DEV).half()
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(rows, 1)
    lengths = torch.arange(rows, device=DEV, dtype=torch.int32) % 9
    out = qlin().paged_attention(q, k, v, table, lengths)
    some = [0, 1, 7, 8, 9, 500, 1007, 1008, 1023]
    check(out[some], q[some], k, v, table[some], lengths[some])


def test_a_window_past_every_length_is_none():
    """Up to the largest number there is: the same kernel, so the same bits."""
    s = make([1000, 1024, 3, 777] * 16, 8, 8, 128, 16, BF16)
    want = qlin().paged_attention(*s)
    for window in (1024, 1 << 40, 2 ** 63 - 1):
        assert torch.equal(qlin().paged_attention(*s, window=window), want), window
