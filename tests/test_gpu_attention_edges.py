"""Edges of the attention side: weights far below a row's largest, infinities, values that pass a rotation by, empty heads,
plans that are kept and saved, second derivatives, sizes at the ends of their ranges."""

import pytest
import torch
from test_gpu_paged_attention import BF16, DEV, F16, check, make

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
