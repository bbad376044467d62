"""The attention side without a GPU: what its entry points refuse before any launch, and the frequencies."""
import pytest
import torch

F16, F32, I32, I64 = torch.float16, torch.float32, torch.int32, torch.int64


def lib():
    from qlin import _lib
    return _lib, _lib.load()


def z(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


def rope_args(**over):
    a = dict(q=z(3, 4, 64), k=z(3, 2, 64), pos=z(1, 3, dtype=I32), freq=z(32, dtype=F32), axis=z(32, dtype=I32), flags=0,
             qo=z(3, 4, 64), ko=z(3, 2, 64))
    a.update(over)
    return a


def rope(**over):
    L, lb = lib()
    a = rope_args(**over)
    d = L.desc
    return lb.qlin_axis_rope(d(a["q"]), d(a["k"]), d(a["pos"]), d(a["freq"]), d(a["axis"]), a["flags"], d(a["qo"]), d(a["ko"]), None)


INVALID, DECLINED = 3 - 1, 1  # QLIN_EINVAL, QLIN_EUNSUPPORTED


@pytest.mark.parametrize("over,status", [
    (dict(q=None), INVALID),
    (dict(q=z(3, 64)), INVALID),                               # not [tokens, heads, D]
    (dict(q=z(3, 4, 64, dtype=I32)), DECLINED),
    (dict(q=z(3, 4, 1024), qo=z(3, 4, 1024)), DECLINED),        # heads too long
    (dict(k=z(2, 2, 64)), INVALID),                             # other tokens
    (dict(k=z(3, 2, 32)), INVALID),                             # other heads
    (dict(k=z(3, 2, 64, dtype=F32)), DECLINED),                 # another dtype
    (dict(k=z(3, 2, 128)[..., ::2]), DECLINED),                 # strided heads
    (dict(qo=z(3, 3, 64)), INVALID),
    (dict(qo=z(3, 4, 64, dtype=F32)), DECLINED),
    (dict(ko=None), INVALID),
    (dict(k=None), INVALID),
    (dict(freq=None), INVALID),
    (dict(freq=z(33, dtype=F32)), INVALID),                     # more pairs than a head holds
    (dict(freq=z(32)), DECLINED),
    (dict(axis=z(31, dtype=I32)), INVALID),
    (dict(axis=z(32, dtype=I64)), DECLINED),
    (dict(pos=None), INVALID),
    (dict(pos=z(1, 4, dtype=I32)), INVALID),
    (dict(pos=z(4, dtype=I32)), INVALID),
    (dict(pos=z(0, 3, dtype=I32)), INVALID),                    # no axis
    (dict(pos=z(1, 3)), DECLINED),
    (dict(flags=4), INVALID),
])
def test_rotation_refuses(over, status):
    assert rope(**over) == status


@pytest.mark.parametrize("over,status", [
    (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID),
    (dict(wq=z(63)), INVALID),
    (dict(wq=z(64, dtype=I32)), DECLINED),
    (dict(wk=z(128)[::2]), DECLINED),
    (dict(k=None, ko=None), INVALID),                            # k's weight without k
])
def test_norms_refuse(over, status):
    L, lb = lib()
    a = dict(rope_args(), wq=z(64), wk=z(64), eps=1e-6)
    a.update(over)
    d = L.desc
    assert lb.qlin_qk_norm_rope(d(a["q"]), d(a["k"]), d(a["wq"]), d(a["wk"]), a["eps"], d(a["pos"]), d(a["freq"]), d(a["axis"]),
                                0, d(a["qo"]), d(a["ko"]), None) == status


@pytest.mark.parametrize("over,status", [
    (dict(v=z(3, 4, 64)), INVALID),
    (dict(v=None), INVALID),
    (dict(k=None), INVALID),
    (dict(kc=z(5, 16, 4, 64)), INVALID),
    (dict(kc=z(5, 0, 2, 64), vc=z(5, 0, 2, 64)), INVALID),       # pages of no token
    (dict(vc=z(4, 16, 2, 64)), INVALID),                         # the caches differ
    (dict(vc=z(5, 16, 2, 64, dtype=F32)), DECLINED),
    (dict(kc=z(5, 16, 2, 128)[..., ::2]), DECLINED),
    (dict(slots=z(4, dtype=I64)), INVALID),
    (dict(slots=z(3)), DECLINED),
    (dict(eps=-1.0), INVALID),                                   # weights without the norms
    (dict(eps=float("nan")), INVALID),
])
def test_store_refuses(over, status):
    L, lb = lib()
    a = dict(rope_args(), v=z(3, 2, 64), wq=z(64), wk=None, eps=1e-6, slots=z(3, dtype=I64), kc=z(5, 16, 2, 64), vc=z(5, 16, 2, 64))
    a.update(over)
    d = L.desc
    assert lb.qlin_qk_norm_rope_store(d(a["q"]), d(a["k"]), d(a["v"]), d(a["wq"]), d(a["wk"]), a["eps"], d(a["pos"]), d(a["freq"]),
                                      d(a["axis"]), 0, d(a["slots"]), d(a["qo"]), d(a["kc"]), d(a["vc"]), None) == status


@pytest.mark.parametrize("over,status", [
    (dict(gq=z(3, 3, 64)), INVALID),
    (dict(gk=None), INVALID),
    (dict(dk=None), INVALID),
    (dict(dq=z(3, 4, 64, dtype=F32)), DECLINED),
    (dict(dwq=z(63)), INVALID),
    (dict(eps=-1.0), INVALID),
    (dict(ws=16), 4),                                            # QLIN_EWORKSPACE
])
def test_gradient_refuses(over, status):
    L, lb = lib()
    a = dict(rope_args(), gq=z(3, 4, 64), gk=z(3, 2, 64), dq=z(3, 4, 64), dk=z(3, 2, 64), wq=z(64), dwq=z(64), eps=1e-6, ws=1 << 20)
    a.update(over)
    d, room = L.desc, torch.zeros(1 << 20, dtype=torch.uint8)
    assert lb.qlin_qk_norm_rope_grad(d(a["gq"]), d(a["gk"]), d(a["q"]), d(a["k"]), d(a["wq"]), None, a["eps"], d(a["pos"]),
                                     d(a["freq"]), d(a["axis"]), 0, d(a["dq"]), d(a["dk"]), d(a["dwq"]), None, room.data_ptr(),
                                     a["ws"], None) == status


@pytest.mark.parametrize("over,status", [
    (dict(page=0), INVALID),
    (dict(context=z(3, 1, dtype=I32)), INVALID),
    (dict(context=z(3, dtype=I64)), DECLINED),
    (dict(added=z(2, dtype=I32)), INVALID),
    (dict(free=z(4, dtype=I64)), DECLINED),
    (dict(table=z(2, 4, dtype=I32)), INVALID),
    (dict(table=z(3, 4, dtype=I64)), DECLINED),
    (dict(table=z(3, 8, dtype=I32)[:, ::2]), DECLINED),
    (dict(table=z(1, 4, dtype=I32).expand(3, -1)), INVALID),      # rows that share their memory
    (dict(slots=z(9, dtype=I32)), DECLINED),
    (dict(rows=z(8, dtype=I32)), INVALID),
    (dict(starts=z(3, dtype=I32)), INVALID),
    (dict(used=z(2, dtype=I32)), INVALID),
])
def test_plan_refuses(over, status):
    L, lb = lib()
    a = dict(context=z(3, dtype=I32), added=z(3, dtype=I32), free=z(4, dtype=I32), page=16, table=z(3, 4, dtype=I32),
             slots=z(9, dtype=I64), positions=z(9, dtype=I32), rows=z(9, dtype=I32), starts=z(4, dtype=I32),
             lengths=z(3, dtype=I32), used=z(1, dtype=I32))
    a.update(over)
    d = L.desc
    assert lb.qlin_paged_plan(d(a["context"]), d(a["added"]), d(a["free"]), a["page"], d(a["table"]), d(a["slots"]),
                              d(a["positions"]), d(a["rows"]), d(a["starts"]), d(a["lengths"]), d(a["used"]), None) == status


@pytest.mark.parametrize("over,status", [
    (dict(q=z(2, 8, 64, dtype=F32)), DECLINED),
    (dict(q=z(2, 8)), INVALID),
    (dict(q=z(2, 8, 60), out=z(2, 8, 60), kc=z(5, 16, 2, 60), vc=z(5, 16, 2, 60)), DECLINED),
    (dict(q=z(2, 8, 264), out=z(2, 8, 264), kc=z(5, 16, 2, 264), vc=z(5, 16, 2, 264)), DECLINED),
    (dict(kc=z(5, 16, 3, 64), vc=z(5, 16, 3, 64)), INVALID),      # 8 heads over 3
    (dict(kc=z(5, 16, 0, 64), vc=z(5, 16, 0, 64)), INVALID),
    (dict(vc=z(5, 8, 2, 64)), INVALID),
    (dict(kc=z(5, 16, 2, 64, dtype=torch.bfloat16)), DECLINED),
    (dict(kc=z(5, 16, 2, 68)[..., :64]), DECLINED),               # rows off the 16-byte grid
    (dict(table=z(3, 4, dtype=I32)), INVALID),
    (dict(table=z(2, 4, dtype=I64)), DECLINED),
    (dict(lengths=z(3, dtype=I32)), INVALID),
    (dict(lengths=z(2, dtype=I64)), DECLINED),
    (dict(window=-1), INVALID),
    (dict(out=z(2, 8, 32)), INVALID),
])
def test_attention_refuses(over, status):
    L, lb = lib()
    a = dict(q=z(2, 8, 64), kc=z(5, 16, 2, 64), vc=z(5, 16, 2, 64), table=z(2, 4, dtype=I32), lengths=z(2, dtype=I32), window=0,
             out=z(2, 8, 64))
    a.update(over)
    d, room = L.desc, torch.zeros(1 << 24, dtype=torch.uint8)
    assert lb.qlin_paged_attention(d(a["q"]), d(a["kc"]), d(a["vc"]), d(a["table"]), d(a["lengths"]), 1.0, a["window"], d(a["out"]),
                                   room.data_ptr(), room.numel(), None) == status


def test_python_entry_points_refuse():
    """Host tensors and dtypes that the C ABI has no name for are declined as the linears' are, in both routes."""
    import qlin
    from qlin import ops
    q, k, c = z(3, 4, 64), z(3, 2, 64), z(5, 16, 2, 64)
    f, p, s, t = z(32, dtype=F32), z(3, dtype=I32), z(3, dtype=I64), z(3, 4, dtype=I32)
    calls = [lambda: qlin.axis_rope(q, k, p, f), lambda: qlin.qk_norm_rope(q, k, None, None, p, f),
             lambda: qlin.qk_norm_rope_store(q, k, k, None, None, p, f, s, c, c),
             lambda: qlin.qk_norm_rope_grad(q, k, q, k, None, None, p, f), lambda: qlin.paged_plan(p, p, t, p, 16, 3),
             lambda: qlin.paged_attention(q, c, c, t, p)]
    fast = ops._FAST
    try:
        for route in (fast, None):
            ops._FAST = route
            for call in calls:
                with pytest.raises(qlin.NoCapableBackendError):
                    call()
            with pytest.raises(ValueError):
                qlin.qk_norm_rope_store(q, k, k, None, None, p, f, s, c, c, eps=-1e-6)
    finally:
        ops._FAST = fast


def test_query_and_workspace():
    L, lb = lib()
    query = lambda op, n, k, param, a=L.DT_F16, b=L.DT_F16: lb.qlin_query(op, 4, n, k, param, a, b)
    assert query(L.OP_PAGED_ATTENTION, 32, 128, 8) == 0 and query(L.OP_PAGED_ATTENTION, 32, 128, 8, L.DT_BF16, L.DT_BF16) == 0
    for bad in ((32, 132, 8), (32, 264, 8), (32, 128, 5), (32, 128, 0), (32, 128, 8, L.DT_F32, L.DT_F32), (32, 128, 8, L.DT_F16, L.DT_BF16)):
        assert query(L.OP_PAGED_ATTENTION, *bad) == 1
    assert query(L.OP_QK_NORM_ROPE_GRAD, 96, 128, 0) == 0 and query(L.OP_QK_NORM_ROPE_GRAD, 96, 513, 0) == 1
    size = lambda op, m, n, k, param: lb.qlin_workspace_size(op, m, n, k, param, L.DT_F16)
    # two parts of a split row a workgroup: 2 x 512 workgroups x 4 heads x (128 values, maximum and sum)
    assert size(L.OP_PAGED_ATTENTION, 8, 32, 128, 8) >= 2 * 512 * 4 * 130 * 4
    assert size(L.OP_PAGED_ATTENTION, 8, 32, 128, 0) == 0
    assert size(L.OP_QK_NORM_ROPE_GRAD, 1056, 96, 128, 0) <= 1024 * 128 * 4


def test_frequencies():
    import qlin
    f, a = qlin.rope_frequencies((16, 56, 56), 1e4)
    assert f.dtype == F32 and a.dtype == I32 and a.tolist() == [0] * 8 + [1] * 28 + [2] * 28
    assert f[0] == f[8] == f[36] == 1.0
    assert torch.allclose(f[8:36].double(), 1e4 ** (-torch.arange(28, dtype=torch.float64) / 28), rtol=1e-7)
    g, b = qlin.rope_frequencies((32, 48, 48), 1e6, shared=True)
    assert torch.allclose(g.double(), 1e6 ** (-torch.arange(64, dtype=torch.float64) / 64), rtol=1e-7)
    assert b.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    assert qlin.rope_frequencies(128)[0].shape == (64,) and qlin.rope_frequencies((0, 4))[1].tolist() == [1, 1]
    for bad in ((3,), (), (-2,)):
        with pytest.raises(ValueError):
            qlin.rope_frequencies(bad)


def test_registry_lists_them():
    import qlin
    have = qlin.registry.capabilities()
    for name in ("axis_rope", "qk_norm_rope", "qk_norm_rope_store", "qk_norm_rope_grad", "paged_plan", "paged_attention"):
        assert name in have and qlin.registry.get_implementation(name) is getattr(qlin, name)
