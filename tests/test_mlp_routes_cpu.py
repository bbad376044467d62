"""The MLP side's ctypes route without a GPU: what it refuses before the library is asked for a workspace."""
import ctypes

import pytest
import torch

F16, F32, F64, I8 = torch.float16, torch.float32, torch.float64, torch.int8


@pytest.fixture
def route(monkeypatch):
    """The ctypes route with tensors of the CPU let through to its checks."""
    import qlin
    from qlin import mlp, ops
    monkeypatch.setattr(ops, "_FAST", None)
    monkeypatch.setattr(mlp, "_check_device", lambda *a: None)
    return qlin


def z(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("dtype", [F64, torch.int16, torch.complex64, torch.bool])
def test_dtypes_that_the_library_does_not_know_are_declined(route, dtype):
    """Also where the dtype would be looked up for the workspace's size first."""
    x, w, odd = z(3, 64), z(64), z(3, 64, dtype=dtype)
    calls = [lambda: route.add_rms_norm(odd, None, w), lambda: route.add_rms_norm_int8(odd, None, w), lambda: route.add_rms_norm_grad(odd, None, x, w),
             lambda: route.add_rms_norm_grad(odd, None, odd, w), lambda: route.gated_act(odd), lambda: route.gated_act_int8(odd),
             lambda: route.gated_act_grad(odd, odd),
             lambda: route.w8a8_int8_linear(odd, z(3, 1, dtype=F32), z(20, 64, dtype=I8), z(20, dtype=F32)),
             lambda: route.w8a8_int8_linear(z(3, 64, dtype=I8), z(3, 1, dtype=F32), z(20, 64, dtype=dtype), z(20, dtype=F32))]
    for call in calls:
        with pytest.raises(route.NoCapableBackendError):
            call()


def test_a_residual_of_no_outputs():
    """Rows of a linear without outputs have a residual without values."""
    from qlin import ops
    for shape in ((3, 0), (2, 3, 0), (0, 0)):
        r, rs = ops._residual_args("linear", z(*shape), z(0), shape, 0)
        assert r.shape == (shape[0] if len(shape) == 2 else 6, 0) and rs.shape == (0,)
    r, _ = ops._residual_args("linear", z(2, 0, 5), None, (2, 0, 5), 5)
    assert r.shape == (0, 5)


def test_a_gradient_of_no_values_needs_no_workspace():
    """qlin_workspace_size is 0 for it: a null workspace is taken, with pointers that are there."""
    from qlin import _lib
    L = _lib.load()
    room = torch.zeros(8)

    def of(*shape):
        t = _lib.QlinTensor(data=room.data_ptr(), dtype=_lib.DT_F16, ndim=len(shape))
        for i, n in enumerate(shape):
            t.shape[i], t.stride[i] = n, 1
        return t

    rows, weight = of(3, 0), of(0)
    assert L.qlin_workspace_size(_lib.OP_ADD_RMS_NORM_GRAD, 3, 0, 0, 0, _lib.DT_F16) == 0
    a = ctypes.addressof
    assert L.qlin_add_rms_norm_grad(a(rows), None, a(rows), a(weight), 1e-6, a(rows), a(weight), None, 0, None) == 0
