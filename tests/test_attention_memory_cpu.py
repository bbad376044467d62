"""Memory that a plan's tensors may not share, refused before any launch."""
import pytest
import torch

I32, I64 = torch.int32, torch.int64


def plan(**over):
    from qlin import _lib
    z = lambda *s, dtype=I32: torch.zeros(*s, dtype=dtype)
    a = dict(context=z(3), added=z(3), free=z(4), table=z(3, 4), slots=z(9, dtype=I64), positions=z(9), rows=z(9), starts=z(4),
             lengths=z(3), used=z(1))
    a.update(over)
    d = _lib.desc
    return _lib.load().qlin_paged_plan(d(a["context"]), d(a["added"]), d(a["free"]), 16, d(a["table"]), d(a["slots"]),
                                       d(a["positions"]), d(a["rows"]), d(a["starts"]), d(a["lengths"]), d(a["used"]), None)


def slices(n, *places):
    m = torch.zeros(n, dtype=I32)
    return [m[a:b] for a, b in places]


def cases():
    x = torch.zeros(3, dtype=I32)
    yield "lengths in place of context", dict(context=x, lengths=x)
    yield "lengths in place of added", dict(added=x, lengths=x)
    a, b = slices(20, (0, 3), (2, 6))
    yield "starts over the end of added", dict(added=a, starts=b)
    a, b = slices(20, (0, 9), (8, 17))
    yield "rows over positions", dict(positions=a, rows=b)
    m = torch.zeros(9, dtype=I64)
    yield "positions over slots", dict(slots=m, positions=m.view(I32)[9:])
    t = torch.zeros(3, 6, dtype=I32)
    yield "free blocks in the table", dict(table=t[:, :4], free=t[1, :4])
    yield "used in the table's last entry", dict(table=t[:, :4], used=t[2, 3:4])
    yield "context over two rows' gap and the next row", dict(table=t[:, :4], context=t.view(-1)[5:8])
    w = torch.zeros(30, dtype=I32)
    yield "starts runs into the table", dict(table=w[6:18].view(3, 4), starts=w[3:7])


@pytest.mark.parametrize("what,over", list(cases()), ids=lambda v: v if isinstance(v, str) else "")
def test_shared_memory_is_refused(what, over):
    assert plan(**over) == 2  # QLIN_EINVAL


def test_memory_beside_one_another_is_not():
    """Neighbours in one allocation, between a table's rows and around it: nothing to refuse (QLIN_EHIP without a GPU, or done)."""
    m = torch.zeros(200, dtype=I32)
    t = torch.zeros(3, 8, dtype=I32)
    over = dict(context=t[0, 4:7], added=t[1, 4:7], lengths=t[2, 4:7], table=t[:, :4], positions=m[:9], rows=m[9:18], starts=m[18:22],
                used=m[22:23], free=m[23:27])
    if torch.cuda.is_available():
        pytest.skip("host memory is not for a launch")
    assert plan(**over) == 3
    w = torch.zeros(30, dtype=I32)
    assert plan(table=w[6:18].view(3, 4), starts=w[2:6], context=w[18:21]) == 3
    x = torch.zeros(3, dtype=I32)
    assert plan(context=x, added=x) == 3  # two inputs may be one
