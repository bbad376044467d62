"""qlin.paged_attention against softmax attention in float64 on the CPU.

Bound: |err| <= u |out| + e * sum_s p_s |v_s| with u = 2^-11 (fp16) or 2^-8 (bf16) for the one rounding of the
output, and e for the weights p: 2^-15 (two parts of 16 bits of a weight, its exponential and the sums) plus
2^-19 * max_s scale * sum_d |q_d k_sd| (an fp32 score of up to 256 products is off by that, and a weight by as much
relative to itself).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -126}


def qlin():
    import qlin as Q
    return Q


def make(lengths, heads, kv_heads, dim, page, dtype, layout="token", seed=0, width=None, spare=2, rest=float("nan")):
    """q, caches whose places outside the rows' tokens hold `rest`, block table (-1 where a row has no page), lengths."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    blocks = sum(need) + spare
    width = max(1, max(need, default=0)) if width is None else width
    order = torch.randperm(blocks, generator=gen).tolist()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    shape = (blocks, page, kv_heads, dim)
    k, v = (torch.full(shape, rest) for _ in range(2))
    for b, n in enumerate(lengths):
        for i in range(need[b]):
            table[b, i] = blk = order.pop()
            m = min(page, n - i * page)
            k[blk, :m], v[blk, :m] = torch.randn(m, kv_heads, dim, generator=gen), torch.randn(m, kv_heads, dim, generator=gen)
    q = 2 * torch.randn(len(lengths), heads, dim, generator=gen)
    q, k, v = (x.to(dtype).to(DEV) for x in (q, k, v))
    if layout == "head":
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    return q, k, v, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


def check(got, q, k, v, table, lengths, window=0, scale=None, what=""):
    q, k, v, table, got_d = q.double().cpu(), k.double().cpu(), v.double().cpu(), table.cpu(), got.double().cpu()
    b_, h_, d = q.shape
    hk, page = k.shape[2], k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    for b, n in enumerate(lengths.tolist()):
        n = max(0, min(n, table.shape[1] * page))
        first = max(0, n - window) if window else 0
        pages = table[b, : -(-n // page)].long()
        ok = ((pages >= 0) & (pages < k.shape[0])).repeat_interleave(page)[first:n]
        pages = pages.clamp(0, max(k.shape[0] - 1, 0))
        kk, vv = (x[pages].flatten(0, 1)[first:n][ok].transpose(0, 1) for x in (k, v))  # [hk, tokens, d]
        if kk.shape[1] == 0:
            assert bool((got_d[b] == 0).all()), f"{what} row {b}: no token, not zero"
            continue
        qq = q[b].view(hk, h_ // hk, d)
        p = torch.softmax(scale * qq @ kk.transpose(1, 2), -1)
        want, mass = (p @ vv).view(h_, d), (p @ vv.abs()).view(h_, d)
        size = (abs(scale) * qq.abs() @ kk.abs().transpose(1, 2)).amax(-1).view(h_, 1)
        tol = U[got.dtype] * want.abs() + (2.0 ** -15 + 2.0 ** -19 * size) * mass + TINY[got.dtype]
        err = (got_d[b] - want).abs()
        assert bool((err <= tol).all()), f"{what} row {b} ({n} tokens): worst {(err / tol).max():.2f} of the bound"


# lengths, heads, kv heads, D, page
CASES = [
    ([77], 32, 8, 128, 16),
    ([1], 1, 1, 128, 16),
    ([1, 2, 15, 16, 17, 31, 32, 33, 0, 127, 128, 129], 8, 2, 128, 16),
    ([300, 5, 1000], 16, 16, 64, 16),           # a head each
    ([300, 5, 1000], 40, 8, 128, 64),           # groups of 5
    ([257, 64], 16, 1, 128, 32),                # one kv head for 16
    ([257, 64], 24, 1, 128, 32),                # for 24
    ([100, 33], 48, 1, 64, 16),                 # for 48
    ([500, 1], 18, 2, 96, 16),                  # groups of 9
    ([130, 64, 700], 10, 2, 256, 16),
    ([63, 200], 4, 2, 8, 16),
    ([63, 200], 4, 4, 72, 8),
    ([63, 201], 4, 1, 80, 100),                 # pages that end inside tiles
    ([99, 100, 101], 8, 8, 128, 7),
    ([40, 41], 8, 4, 128, 1),
    ([4097, 20, 9000], 8, 2, 128, 16),          # split over the length and joined
    ([5000], 4, 1, 256, 48),
    ([6001], 2, 2, 64, 24),
    ([0, 0], 8, 2, 128, 16),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", CASES)
def test_attention(lengths, heads, kv_heads, dim, page, layout, dtype):
    """What lies behind a row's last token, in its last page and in the other pages, is NaN: it is never used."""
    s = make(lengths, heads, kv_heads, dim, page, dtype, layout)
    check(qlin().paged_attention(*s), *s)


@pytest.mark.parametrize("window", [1, 16, 31, 100, 4096])
@pytest.mark.parametrize("page", [16, 12])
def test_window(window, page):
    s = make([1, 15, 16, 17, 100, 101, 3000, 0], 8, 2, 128, page, BF16)
    check(qlin().paged_attention(*s, window=window), *s, window=window)


def test_pages_before_the_window_are_not_used():
    """A server frees the pages that a window has left behind: their entries and contents are anything."""
    q, k, v, table, lengths = make([1000], 8, 2, 128, 16, F16)
    want = qlin().paged_attention(q, k, v, table, lengths, window=100)
    gone = table[0, : 900 // 16].long()
    k[gone], v[gone] = float("nan"), float("inf")
    assert torch.equal(want, qlin().paged_attention(q, k, v, table, lengths, window=100))
    table[0, : 900 // 16] = -1
    assert torch.equal(want, qlin().paged_attention(q, k, v, table, lengths, window=100))


@pytest.mark.parametrize("width", [16, 17, 32, 33, 70, 128, 129, 300])
@pytest.mark.parametrize("rows", [1, 5, 70, 300])
def test_whole_rows_and_split_ones(rows, width):
    """Tables with room for rows that one workgroup takes and for rows that are split, whatever the lengths are."""
    lengths = [(i * 137) % (width * 16) for i in range(rows)]
    lengths[0] = width * 16 - 3
    s = make(lengths, 4, 2, 64, 16, F16, width=width)
    check(qlin().paged_attention(*s), *s)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,longest", [
    (300, 8, 8, 128, 20), (150, 32, 8, 128, 100), (400, 8, 8, 64, 130), (220, 48, 4, 96, 64), (200, 8, 4, 256, 33),
    (230, 16, 8, 72, 500),
])
def test_many_short_rows(rows, heads, kv_heads, dim, longest, dtype):
    """So many that a wave takes each, empty ones among them; the last in a window too."""
    lengths = [(i * 53) % (longest + 1) for i in range(rows)]
    s = make(lengths, heads, kv_heads, dim, 16, dtype)
    check(qlin().paged_attention(*s), *s)
    check(qlin().paged_attention(*s, window=19), *s, window=19)


@pytest.mark.parametrize("rows", [1, 65, 1030])
def test_many_rows(rows):
    lengths = [(i * 37) % 90 for i in range(rows)]
    lengths[-1] = 3000
    s = make(lengths, 4, 1, 64, 16, BF16)
    check(qlin().paged_attention(*s), *s)


@pytest.mark.parametrize("scale", [0.5, 1e-3, -0.1, 0.0])
def test_scale(scale):
    s = make([200, 3], 8, 2, 128, 16, F16)
    check(qlin().paged_attention(*s, scale=scale), *s, scale=scale)


def test_large_scores():
    """Scores of several hundred: one token holds all the weight, no exponential overflows."""
    q, k, v, table, lengths = make([700, 2500], 8, 2, 128, 16, BF16)
    q = (q * 50).contiguous()
    check(qlin().paged_attention(q, k, v, table, lengths), q, k, v, table, lengths)


def test_a_prompt_of_shared_rows():
    """A prompt's tokens as rows with one expanded table row and lengths 1, 2, ..."""
    n, page = 50, 16
    q, k, v, table, _ = make([n], 8, 2, 128, page, F16)
    q = torch.randn(n, 8, 128, generator=torch.Generator().manual_seed(3)).half().to(DEV)
    rows, lengths = table.expand(n, -1), torch.arange(1, n + 1, dtype=torch.int32, device=DEV)
    check(qlin().paged_attention(q, k, v, rows, lengths), q, k, v, rows, lengths)


def test_entries_outside_the_cache_are_absent():
    q, k, v, table, lengths = make([300, 40, 20], 8, 2, 128, 16, F16)
    table[0, 3], table[0, 7], table[1, 0], table[2, 0], table[2, 1] = -1, 10 ** 9, -5, k.shape[0], -2 ** 31
    check(qlin().paged_attention(q, k, v, table, lengths), q, k, v, table, lengths)
    s = make([300, 40], 8, 2, 128, 10, F16)
    s[3][0, 3], s[3][1, 1] = -1, 10 ** 9
    check(qlin().paged_attention(*s), *s)


def test_lengths_past_the_table_and_below_zero():
    q, k, v, table, lengths = make([64, 32], 8, 2, 128, 16, F16)
    lengths = torch.tensor([10 ** 9, -3], dtype=torch.int32, device=DEV)
    check(qlin().paged_attention(q, k, v, table, lengths), q, k, v, table, lengths)


def test_values_that_are_not_finite():
    """A NaN or an infinity in a row's own tokens shows in that row's head group alone."""
    q, k, v, table, lengths = make([100, 100], 8, 2, 128, 16, F16)
    v[table[0, 2].long(), 3, 1, 5] = float("inf")
    k[table[1, 1].long(), 0, 0] = float("nan")
    out = qlin().paged_attention(q, k, v, table, lengths)
    bad = ~out.isfinite()
    assert bool(bad[0, 4:, 5].all()) and int(bad[0].sum()) == 4 and bool(bad[1, :4].all()) and int(bad[1].sum()) == 4 * 128


def test_strides_and_out():
    s = make([77, 200], 8, 2, 128, 16, BF16)
    q, k, v, table, lengths = s
    want = qlin().paged_attention(*s)
    fused = torch.zeros(2, 8 + 4, 128, dtype=BF16, device=DEV)
    fused[:, :8] = q
    wide = torch.full((2, 40), -3, dtype=torch.int32, device=DEV)
    wide[:, : table.shape[1]] = table
    both = torch.stack([k, v], 1)                       # k and v of a block side by side
    out = torch.zeros(2, 9, 136, dtype=BF16, device=DEV)
    got = qlin().paged_attention(fused[:, :8], both[:, 0], both[:, 1], wide[:, : table.shape[1]], lengths, out=out[:, :8, :128])
    assert torch.equal(got, want) and got.data_ptr() == out.data_ptr()
    assert bool((out[:, 8] == 0).all()) and bool((out[..., 128:] == 0).all())
    assert torch.equal(qlin().paged_attention(q.repeat_interleave(2, -1)[..., ::2], k, v, table, lengths), want)


def test_a_cache_of_more_than_32_bits_of_values():
    """Blocks past 2^31 values and 2^32 bytes."""
    page, hk, d = 16, 8, 128
    blocks = (1 << 32) // (page * hk * d) + 40          # 8.6 GB a cache
    k = torch.empty(blocks, page, hk, d, dtype=F16, device=DEV)
    v = torch.empty_like(k)
    table = torch.tensor([[blocks - 1, 1, blocks // 2 + 3], [0, blocks - 30, 7]], dtype=torch.int32, device=DEV)
    for b in table.flatten().tolist():
        k[b], v[b] = torch.randn(page, hk, d).half().to(DEV), torch.randn(page, hk, d).half().to(DEV)
    q = torch.randn(2, 16, d).half().to(DEV)
    lengths = torch.tensor([45, 33], dtype=torch.int32, device=DEV)
    out = qlin().paged_attention(q, k, v, table, lengths)
    used = table.flatten().long()
    small = torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3)
    check(out, q, k[used], v[used], small, lengths)
    # stored there through the slots
    pos = torch.zeros(3, dtype=torch.int32, device=DEV)
    slots = torch.tensor([(blocks - 1) * page + 3, 5, (blocks // 2) * page], device=DEV)
    x = torch.randn(3, hk, d).half().to(DEV)
    freq, _ = qlin().rope_frequencies(128, device=DEV)
    qlin().qk_norm_rope_store(x, x, x, None, None, pos, freq, slots, k, v, eps=None)
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(k[s // page, s % page], x[i]) and torch.equal(v[s // page, s % page], x[i])


def test_routes_streams_and_graphs(monkeypatch):
    from qlin import ops
    Q = qlin()
    s = make([4097, 20, 900], 8, 2, 128, 16, BF16)
    want = Q.paged_attention(*s)
    for _ in range(3):
        assert torch.equal(Q.paged_attention(*s), want)
    with monkeypatch.context() as m:
        m.setattr(ops, "_FAST", None)
        assert torch.equal(Q.paged_attention(*s), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = Q.paged_attention(*s)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = Q.paged_attention(*s)
    for i in range(4):  # other lengths and queries, other eager calls between
        s[4].copy_(torch.tensor([4097 - 900 * i, 20 - i, 900 - 7 * i], dtype=torch.int32))
        s[0].copy_(torch.randn(s[0].shape, generator=torch.Generator().manual_seed(i)).to(BF16))
        graph.replay()
        want = Q.paged_attention(*s)
        torch.cuda.synchronize()
        assert torch.equal(got, want), i


def test_empty_calls():
    Q = qlin()
    q, k, v, table, lengths = make([5], 8, 2, 128, 16, F16)
    assert Q.paged_attention(q[:0], k, v, table[:0], lengths[:0]).shape == (0, 8, 128)
    assert bool((Q.paged_attention(q, k, v, table[:, :0], lengths) == 0).all())
    assert bool((Q.paged_attention(q, k[:0], v[:0], table, lengths) == 0).all())
    assert math.isclose(128 ** -0.5, 0.08838834764831845)
