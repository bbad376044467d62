"""qlin.paged_plan against the definition in Python integers, and what it does when lists and tables are too short."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def qlin():
    import qlin as Q
    return Q


def reference(context, added, table, free, page, n):
    """The plan in Python integers; `table` (lists) is changed in place."""
    slots, positions, rows, starts, lengths, used = [], [], [], [0], [], 0
    for b, (c, a) in enumerate(zip(context, added)):
        c, a = max(c, 0), max(a, 0)
        old, now = -(-c // page), -(-(c + a) // page)
        for at in range(old, now):
            if at < len(table[b]):
                table[b][at] = free[used] if used < len(free) else -1
            used += 1
        for p in range(c, c + a):
            block, index = -1, used - (now - old) + p // page - old
            if p // page < len(table[b]):
                block = table[b][p // page] if p // page < old else free[index] if index < len(free) else -1
            slots.append(block * page + p % page if block >= 0 else -1)
            positions.append(p)
            rows.append(b)
        starts.append(starts[-1] + a)
        lengths.append(c + a)
    pad = [-1] * (n - len(slots))
    return slots[:n] + pad, positions[:n] + pad, rows[:n] + pad, starts, lengths, [used]


def check(context, added, page, width, free, n, seed=0, pad=0):
    r = random.Random(seed)
    table = [[r.randrange(1 << 20) if i * page < c else -7 for i in range(width)] for c in context]
    want_table = [list(row) for row in table]
    want = reference(context, added, want_table, free, page, n)
    whole = torch.full((len(context), width + pad), -9, dtype=torch.int32)
    whole[:, :width] = torch.tensor(table, dtype=torch.int32).reshape(len(context), width)
    t = whole.to(DEV)[:, :width]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    plan = qlin().paged_plan(ints(context), ints(added), t, ints(free), page, n)
    for name, got, w in zip(plan._fields, plan, want):
        assert got.tolist() == w, name
    assert t.tolist() == want_table


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("b", [1, 3, 64, 257])
@pytest.mark.parametrize("new", [1, 40])
def test_plan(b, new, page):
    r = random.Random(b * page + new)
    context = [r.choice((0, 1, page - 1, page, page + 1, r.randrange(300))) for _ in range(b)]
    added = [r.choice((0, 1, new, r.randrange(new + 1))) for _ in range(b)]
    free = r.sample(range(1 << 20, 1 << 21), sum(-(-(c + a) // page) - -(-c // page) for c, a in zip(context, added)) + 2)
    check(context, added, page, 400, free, sum(added), pad=3)


def test_more_places_than_tokens_and_fewer():
    check([5, 0, 31], [2, 3, 1], 16, 4, [100, 101, 102], 64)
    check([5, 0, 31], [2, 3, 1], 16, 4, [100, 101, 102], 4)
    check([5, 0, 31], [2, 3, 1], 16, 4, [100, 101, 102], 0)


def test_short_free_list_and_short_rows():
    check([0, 14, 3], [40, 20, 60], 16, 8, [9, 8, 7], 120)       # the list runs out: pages and slots of -1
    check([0, 14, 3], [40, 20, 60], 16, 8, [], 120)
    check([0, 14, 3], [40, 20, 60], 16, 2, list(range(50)), 120)  # pages past the rows have no entry
    check([0, 14], [40, 20], 16, 0, list(range(50)), 60)


def test_edges():
    check([], [], 16, 4, [1, 2], 3)
    check([0, 0, 0], [0, 0, 0], 16, 4, [1, 2], 0)
    check([-5, 3], [4, -2], 16, 4, [1, 2], 6)                     # negative counts as 0
    check([100], [3000], 16, 250, list(range(300)), 3000)         # one request, many workgroups


def test_most_requests():
    r = random.Random(1)
    b = 4096
    context, added = [r.randrange(40) for _ in range(b)], [r.randrange(4) for _ in range(b)]
    check(context, added, 16, 4, list(range(6000)), sum(added))
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
    with pytest.raises(qlin().NoCapableBackendError):
        qlin().paged_plan(i32(4097), i32(4097), i32(4097, 1), i32(1), 16, 1)


def test_lengths_at_the_end_of_32_bits():
    """Sums past 32 bits stay at the largest value and nothing outside the tables is touched."""
    top = 2 ** 31 - 1
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    table = torch.full((2, 3), -7, dtype=torch.int32, device=DEV)
    plan = qlin().paged_plan(ints([top - 1, top]), ints([1, 5]), table, ints([4]), 1 << 20, 6)
    assert plan.lengths.tolist() == [top, top] and plan.starts.tolist() == [0, 1, 6]
    assert plan.positions.tolist() == [top - 1] + [top] * 5 and plan.slots.tolist() == [-1] * 6
    assert bool((table == -7).all())


def test_routes_stream_and_graph(monkeypatch):
    from qlin import ops
    Q = qlin()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    context, added, free = ints([5, 0, 31]), ints([2, 3, 1]), ints([100, 101, 102])
    fresh = lambda: torch.zeros(3, 4, dtype=torch.int32, device=DEV)
    t1, t2 = fresh(), fresh()
    a = Q.paged_plan(context, added, t1, free, 16, 8)
    with monkeypatch.context() as m:
        m.setattr(ops, "_FAST", None)
        b = Q.paged_plan(context, added, t2, free, 16, 8)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(t1, t2)
    t3 = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = Q.paged_plan(context, added, t3, free, 16, 8)
    for i in range(4):
        context.copy_(ints([5 + i, i, 31 + i]))
        t3.zero_()
        graph.replay()
        t4 = fresh()
        d = Q.paged_plan(context, added, t4, free, 16, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(c, d)), i
