"""The MLP side without a GPU: what its entry points refuse before any launch."""
import pytest
import torch

F16, BF16, F32, I8, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int8, torch.int32
INVALID, DECLINED, NO_ROOM = 2, 1, 4  # QLIN_EINVAL, QLIN_EUNSUPPORTED, QLIN_EWORKSPACE


def lib():
    from qlin import _lib
    return _lib, _lib.load()


def z(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


BAD_INPUT = [
    (dict(x=None), INVALID),
    (dict(x=z(64)), INVALID),                                 # not [rows, values]
    (dict(x=z(3, 64, dtype=I32)), DECLINED),
    (dict(x=z(3, 128)[:, ::2]), DECLINED),                    # strided values
    (dict(r=z(3, 63)), INVALID),
    (dict(r=z(2, 64)), INVALID),
    (dict(r=z(3, 64, dtype=BF16), h=z(3, 64, dtype=BF16)), DECLINED),
    (dict(r=None), INVALID),                                  # h without a residual
    (dict(h=None), INVALID),
    (dict(h=z(3, 64, dtype=F32)), DECLINED),                  # not the residual's dtype
    (dict(h=z(1, 64).expand(3, 64)), INVALID),                # rows that overlap
    (dict(w=z(63)), INVALID),
    (dict(w=z(128)[::2]), DECLINED),
    (dict(w=z(64, dtype=I8)), DECLINED),
    (dict(w=z(4, 32)[:2]), INVALID),                          # no vector
    (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID),
]


@pytest.mark.parametrize("over,status", BAD_INPUT + [
    (dict(y=z(3, 65)), INVALID),
    (dict(y=z(3, 64, dtype=F32)), DECLINED),
    (dict(y=z(1, 64).expand(3, 64)), INVALID),
    (dict(x=z(1, (1 << 20) + 1), r=None, h=None, w=None, y=z(1, (1 << 20) + 1)), DECLINED),
])
def test_norm_refuses(over, status):
    L, lb = lib()
    a = dict(x=z(3, 64), r=z(3, 64), w=z(64), eps=1e-6, y=z(3, 64), h=z(3, 64))
    a.update(over)
    d = L.desc
    assert lb.qlin_add_rms_norm(d(a["x"]), d(a["r"]), d(a["w"]), a["eps"], d(a["y"]), d(a["h"]), None) == status


@pytest.mark.parametrize("over,status", BAD_INPUT + [
    (dict(q=z(3, 64)), DECLINED),
    (dict(q=z(3, 63, dtype=I8)), INVALID),
    (dict(s=z(3, 1)), DECLINED),
    (dict(s=z(2, dtype=F32)), INVALID),
    (dict(s=None), INVALID),
    (dict(group=12), DECLINED),
    (dict(group=512), DECLINED),
    (dict(group=128), INVALID),                               # 64 values are no multiple of it
    (dict(x=z(3, 0), r=z(3, 0), h=z(3, 0), w=None, q=z(3, 0, dtype=I8)), DECLINED),  # no values, no scale
])
def test_norm_to_int8_refuses(over, status):
    L, lb = lib()
    a = dict(x=z(3, 64), r=z(3, 64), w=z(64), eps=1e-6, group=0, q=z(3, 64, dtype=I8), s=z(3, 1, dtype=F32), h=z(3, 64))
    a.update(over)
    d = L.desc
    assert lb.qlin_add_rms_norm_int8(d(a["x"]), d(a["r"]), d(a["w"]), a["eps"], a["group"], d(a["q"]), d(a["s"]), d(a["h"]),
                                     None) == status


@pytest.mark.parametrize("over,status", [
    (dict(dy=None), INVALID),
    (dict(h=None), INVALID),
    (dict(h=z(3, 64, dtype=BF16), dh=None, dx=z(3, 64, dtype=BF16)), DECLINED),
    (dict(h=z(3, 63)), INVALID),
    (dict(dh=z(3, 64, dtype=F32)), DECLINED),
    (dict(dh=z(4, 64)), INVALID),
    (dict(dx=z(3, 64, dtype=F32)), DECLINED),
    (dict(dx=None), INVALID),
    (dict(w=z(65)), INVALID),
    (dict(dw=z(63)), INVALID),
    (dict(dw=z(64, dtype=I32)), DECLINED),
    (dict(eps=-1e-9), INVALID),
    (dict(room=16), NO_ROOM),
])
def test_norm_gradient_refuses(over, status):
    L, lb = lib()
    a = dict(dy=z(3, 64), dh=z(3, 64), h=z(3, 64), w=z(64), eps=1e-6, dx=z(3, 64), dw=z(64), room=1 << 16)
    a.update(over)
    d, room = L.desc, torch.zeros(1 << 16, dtype=torch.uint8)
    assert lb.qlin_add_rms_norm_grad(d(a["dy"]), d(a["dh"]), d(a["h"]), d(a["w"]), a["eps"], d(a["dx"]), d(a["dw"]), room.data_ptr(),
                                     a["room"], None) == status


BAD_GATES = [
    (dict(gate=None), INVALID),
    (dict(gate=z(3, 64, dtype=I8)), DECLINED),
    (dict(gate=z(3, 128)[:, ::2]), DECLINED),
    (dict(up=z(3, 63)), INVALID),
    (dict(up=z(3, 64, dtype=F32)), DECLINED),
    (dict(act=2), DECLINED),
    (dict(act=-1), DECLINED),
]


@pytest.mark.parametrize("over,status", BAD_GATES + [
    (dict(y=None), INVALID),
    (dict(y=z(3, 64, dtype=F32)), DECLINED),
    (dict(y=z(2, 64)), INVALID),
])
def test_activation_refuses(over, status):
    L, lb = lib()
    a = dict(gate=z(3, 64), up=z(3, 64), act=0, y=z(3, 64))
    a.update(over)
    d = L.desc
    assert lb.qlin_gated_act(d(a["gate"]), d(a["up"]), a["act"], d(a["y"]), None) == status


@pytest.mark.parametrize("over,status", BAD_GATES + [
    (dict(q=z(3, 64)), DECLINED),
    (dict(q=z(2, 64, dtype=I8)), INVALID),
    (dict(s=z(4, dtype=F32)), INVALID),
    (dict(group=3), DECLINED),
    (dict(group=256), INVALID),
    (dict(gate=z(3, 0), up=z(3, 0), q=z(3, 0, dtype=I8)), DECLINED),
])
def test_activation_to_int8_refuses(over, status):
    L, lb = lib()
    a = dict(gate=z(3, 64), up=z(3, 64), act=0, group=0, q=z(3, 64, dtype=I8), s=z(3, dtype=F32))
    a.update(over)
    d = L.desc
    assert lb.qlin_gated_act_int8(d(a["gate"]), d(a["up"]), a["act"], a["group"], d(a["q"]), d(a["s"]), None) == status


@pytest.mark.parametrize("over,status", BAD_GATES + [
    (dict(dy=None), INVALID),
    (dict(dy=z(3, 64, dtype=F32)), DECLINED),
    (dict(dy=z(3, 32)), INVALID),
    (dict(dgate=None), INVALID),
    (dict(dup=None), INVALID),
    (dict(up=None), INVALID),
    (dict(dup=z(3, 64, dtype=F32)), DECLINED),
])
def test_activation_gradient_refuses(over, status):
    L, lb = lib()
    a = dict(dy=z(3, 64), gate=z(3, 64), up=z(3, 64), act=1, dgate=z(3, 64), dup=z(3, 64))
    a.update(over)
    d = L.desc
    assert lb.qlin_gated_act_grad(d(a["dy"]), d(a["gate"]), d(a["up"]), a["act"], d(a["dgate"]), d(a["dup"]), None) == status


MANY = dict(x=z(300, 256, dtype=I8), sx=z(300, 1, dtype=F32), y=z(300, 20))


@pytest.mark.parametrize("over,status", [
    (dict(x=None), INVALID),
    (dict(x=z(3, 256)), DECLINED),
    (dict(x=z(256, dtype=I8)), INVALID),
    (dict(x=z(3, 255, dtype=I8)), INVALID),
    (dict(w=z(20, 256)), DECLINED),
    (dict(w=z(20, 512, dtype=I8)[:, ::2]), DECLINED),
    (dict(sx=z(3, 1)), DECLINED),
    (dict(sx=z(4, 1, dtype=F32)), INVALID),
    (dict(sw=z(20)), DECLINED),
    (dict(sw=z(19, dtype=F32)), INVALID),
    (dict(b=z(19)), INVALID),
    (dict(b=z(20, dtype=I8)), DECLINED),
    (dict(r=z(3, 19)), INVALID),
    (dict(r=z(3, 20, dtype=I8)), DECLINED),
    (dict(rs=z(20)), INVALID),                                # without a residual
    (dict(r=z(3, 20), rs=z(19)), INVALID),
    (dict(y=z(3, 21)), INVALID),
    (dict(y=z(3, 20, dtype=I8)), DECLINED),
    (dict(y=z(1, 20).expand(3, 20)), INVALID),
    (dict(x=z(3, 0, dtype=I8), w=z(20, 0, dtype=I8)), DECLINED),
    (dict(x=z(1, 131072, dtype=I8), w=z(2, 131072, dtype=I8), sx=z(1, dtype=F32), sw=z(2, dtype=F32), y=z(1, 2)), DECLINED),
    (dict(sx=z(4, 4, dtype=F32)[:2, :2].expand(2, 2)), INVALID),
    (dict(x=z(4, 256, dtype=I8), y=z(4, 20), sx=z(2, 4, dtype=F32)[:, :2]), INVALID),   # four scales, but no vector
    (dict(x=z(1, 256, dtype=I8).expand(1 << 28, 256), sx=z(1, 1, dtype=F32)), DECLINED),
    (dict(x=z(1, 256, dtype=I8).expand(1 << 27, 256), w=z(1, 256, dtype=I8).expand(1 << 10, 256), sx=z(1, 1, dtype=F32)), DECLINED),
    (dict(w=z(1, 256, dtype=I8).expand(1 << 26, 256), sw=z(1, dtype=F32)), DECLINED),
    (dict(MANY, x=z(300, 250, dtype=I8), w=z(20, 250, dtype=I8)), NO_ROOM),   # rows that are not whole are copied
    (dict(MANY, w=z(20, 257, dtype=I8)[:, :256]), NO_ROOM),
])
def test_linear_refuses(over, status):
    L, lb = lib()
    a = dict(x=z(3, 256, dtype=I8), sx=z(3, 1, dtype=F32), w=z(20, 256, dtype=I8), sw=z(20, dtype=F32), b=None, r=None, rs=None, y=z(3, 20))
    a.update(over)
    d = L.desc
    assert lb.qlin_w8a8_linear(d(a["x"]), d(a["sx"]), d(a["w"]), d(a["sw"]), d(a["b"]), d(a["r"]), d(a["rs"]), d(a["y"]), None, 0,
                               None) == status


def test_tensors_on_the_cpu_are_declined(monkeypatch):
    """By both routes; QLIN_DISABLE declines too, and the registry lists the capabilities."""
    import qlin
    from qlin import ops
    x, w8 = z(3, 64), z(20, 64, dtype=I8)
    calls = [lambda: qlin.add_rms_norm(x, x, None), lambda: qlin.add_rms_norm_int8(x), lambda: qlin.add_rms_norm_grad(x, None, x),
             lambda: qlin.gated_act(x, x), lambda: qlin.gated_act_int8(x), lambda: qlin.gated_act_grad(x, x, x),
             lambda: qlin.w8a8_int8_linear(z(3, 64, dtype=I8), z(3, 1, dtype=F32), w8, z(20, dtype=F32))]
    for fast in (ops._FAST, None):
        monkeypatch.setattr(ops, "_FAST", fast)
        for call in calls:
            with pytest.raises(qlin.NoCapableBackendError, match="ROCm"):
                call()
    with pytest.raises(qlin.NoCapableBackendError, match="relu"):
        qlin.gated_act(x, act="relu")
    monkeypatch.setenv("QLIN_DISABLE", "1")
    for call in calls:
        with pytest.raises(qlin.NoCapableBackendError, match="QLIN_DISABLE"):
            call()
    have = qlin.registry.capabilities()
    assert {"add_rms_norm", "add_rms_norm_int8", "add_rms_norm_grad", "gated_act", "gated_act_int8", "gated_act_grad",
            "w8a8_int8_linear"} <= set(have)


def test_workspaces():
    L, lb = lib()
    a = lambda v: (v + 255) // 256 * 256  # noqa: E731
    size = lambda m, n, k, param=0: lb.qlin_workspace_size(L.OP_W8A8_LINEAR, m, n, k, param, 0)  # noqa: E731
    assert size(300, 20, 250) == size(300, 20, 250, 3) >= a(300 * 256) + a(20 * 256)   # rows that are not whole are copied
    assert size(300, 4096, 256) == size(64, 300, 250) == 0
    assert size(3000, 4096, 256, L.W8A8_W_ROWS) == a(4096 * 256) and size(3000, 4096, 256, L.W8A8_X_ROWS) == a(3000 * 256)
    assert size(9504, 4096, 4096, L.W8A8_W_APART) == a(4096 * 4096) and size(9504, 4096, 4096) == 0
    assert lb.qlin_workspace_size(L.OP_ADD_RMS_NORM_GRAD, 5, 0, 100, 0, L.DT_F16) >= 400


def test_rows_far_apart_are_copied():
    """Offsets in a tile are 32 bits: strides of 2^24 bytes and more go through the workspace, by both routes' rule and the library's."""
    from qlin import mlp
    L, lb = lib()
    far = lambda ld: torch.empty(0, dtype=I8).as_strided((2, 0), (ld, 1))  # noqa: E731
    assert mlp._aligned(far((1 << 24) - 16)) and not mlp._aligned(far(1 << 24)) and not mlp._aligned(far(40))
    assert 255 * ((1 << 24) - 16) + 128 < 1 << 32


def test_query():
    L, lb = lib()
    ask = lambda op, m, n, k, a, b: lb.qlin_query(op, m, n, k, 0, a, b)  # noqa: E731
    assert ask(L.OP_W8A8_LINEAR, 8, 4096, 131071, L.DT_I8, L.DT_BF16) == 0
    for bad in ((8, 4096, 131072, L.DT_I8, L.DT_BF16), (8, 4096, 0, L.DT_I8, L.DT_BF16), (8, 4096, 64, L.DT_F16, L.DT_F16), (8, 1 << 26, 64, L.DT_I8, L.DT_F16),
                (1 << 28, 8, 64, L.DT_I8, L.DT_F16), (1 << 27, 1 << 10, 64, L.DT_I8, L.DT_F16), (8, 4096, 64, L.DT_I8, L.DT_I8)):
        assert ask(L.OP_W8A8_LINEAR, *bad) == DECLINED
    assert ask(L.OP_ADD_RMS_NORM_GRAD, 8, 0, 1 << 20, L.DT_F16, L.DT_F32) == ask(L.OP_ADD_RMS_NORM_GRAD, 8, 0, 1, L.DT_BF16, L.DT_BF16) == 0
    assert ask(L.OP_ADD_RMS_NORM_GRAD, 8, 0, (1 << 20) + 1, L.DT_F16, L.DT_F16) == ask(L.OP_ADD_RMS_NORM_GRAD, 8, 0, 64, L.DT_F16, L.DT_BF16) == DECLINED
