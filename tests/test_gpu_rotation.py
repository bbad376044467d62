"""Rotated 8-bit rows of the norm and the activation: their sums, their range, rows that are not finite, rows at any address."""
import pytest
import torch
from mlp_ref import BF16, DEV, F16, F32, U, act, layouts, qlin, rand, rotated, sigma_bound
from rotation_ref import GROUPS, check_rotated, check_whole, whole_rows

pytestmark = pytest.mark.gpu
DTYPES = [F16, BF16, F32]
WIDTHS = [256, 1024, 8192, 16640, 33024]  # in registers, a thread four and eight runs, and read twice


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("w", WIDTHS)
def test_sums_of_whole_numbers(group, w):
    """silu(32) is 32 in fp32.  The norm's scale has rho's roundings besides (bound_y of its tests: 64 U)."""
    v = whole_rows(3, w, group, seed=w + group)
    q, s = qlin().gated_act_int8(torch.full_like(v, 32.0, device=DEV), v.to(DEV), convrot_groupsize=group)
    check_whole(q, s, v, group, 32.0, 0)
    q, s, _ = qlin().add_rms_norm_int8(v.to(DEV), None, None, convrot_groupsize=group)
    rho = (v.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    check_whole(q, s, v, group, rho, 64)


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [4, 32, 128, 256])
def test_activation(group, dtype, kind):
    """A value is off by its sigma and two products before the rotation."""
    for t, w in ((3, 1024), (2, 13824), (2, 16640), (1, 33024)):
        gate, up = rand(t, w, seed=w, scale=3.0).to(dtype).to(DEV), rand(t, w, seed=w + 1, dtype=dtype).to(DEV)
        for u in (up, None):
            q, s = qlin().gated_act_int8(gate, u, act=kind, convrot_groupsize=group)
            z = gate.double().cpu()
            f, _, arg = act(z, kind)
            v = f if u is None else f * u.double().cpu()
            check_rotated(q, s, v, v.abs() * (sigma_bound(arg, dtype) + 2 * U) + 2.0 ** -120, group)


@pytest.mark.parametrize("dtype,h_dtype", [(F16, F16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("group", [4, 32, 128, 256])
def test_norm(group, dtype, h_dtype):
    """A value is off by the addition's and the weight's rounding, the scale by rho's besides, which is taken off first."""
    for t, w in ((3, 1024), (2, 5120), (2, 16640)):
        x, r, g = rand(t, w, seed=w, dtype=dtype), rand(t, w, seed=w + 1, dtype=h_dtype, scale=2.0), (1 + 0.2 * rand(w, seed=3)).to(dtype)
        q, s, _ = qlin().add_rms_norm_int8(x.to(DEV), r.to(DEV), g.to(DEV), convrot_groupsize=group)
        h = x.double() + r.double()
        rho = (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        v = h * g.double()
        check_rotated(q, s.double().cpu() / rho, v, v.abs() * 66 * U, group)


def loud(t, w, dtype, seed):
    return (rand(t, w, seed=seed).clamp(-1.9, 1.9) * 2.0 ** 27).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", GROUPS)
def test_rows_near_the_largest_values(group, dtype):
    """Values of up to 2^127 whose rotated ones stay below 2^127.3 here, their sums without the factor 1 / sqrt(G) up to 16 times that: the scale
    is finite and right.  Through the norm by its weight."""
    for w in (1024, 16640, 33024):
        up = loud(2, w, dtype, w + group) * 0.25
        q, s = qlin().gated_act_int8(torch.full_like(up, 2.0 ** 100), up, convrot_groupsize=group)
        v = up.double().cpu() * 2.0 ** 100
        assert bool(s.isfinite().all()) and float(rotated(v, group).abs().max()) < 2.0 ** 127.9
        check_rotated(q, s, v, v.abs() * 4 * U, group)
        x, g = rand(2, w, seed=w, dtype=dtype).to(DEV), torch.full((w,), 2.0 ** 125, device=DEV)
        q, s, _ = qlin().add_rms_norm_int8(x, None, g, convrot_groupsize=group)
        h = x.double().cpu()
        rho = (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        assert bool(s.isfinite().all())
        check_rotated(q, s.double().cpu() / rho, h * 2.0 ** 125, h.abs() * 2.0 ** 125 * 66 * U, group)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", GROUPS)
def test_rows_that_are_not_finite_and_tiny_rows(group, dtype):
    """An infinity or a NaN makes its row's scale not finite and leaves the other rows as they are; whole numbers of the smallest normal
    value keep their codes: their sums are exact, in units of 2^-130 at the least."""
    for w in (1024, 768, 33024):
        up = rand(6, w, seed=w, dtype=dtype).to(DEV)
        clean = up.clone()
        up[1, 5], up[2, w - 3], up[3, 7] = float("inf"), float("nan"), -float("inf")
        up[4] = 0
        tiny = torch.arange(w, device=DEV).remainder(61).to(dtype)
        up[5] = tiny * torch.finfo(dtype).tiny
        gate = torch.full_like(up, 32.0)
        q, s = qlin().gated_act_int8(gate, up, convrot_groupsize=group)
        q0, s0 = qlin().gated_act_int8(gate, clean, convrot_groupsize=group)
        assert not bool(s[1:4].isfinite().any()) and torch.equal(q[0], q0[0]) and torch.equal(s[0], s0[0])
        assert bool((q[4] == 0).all()) and float(s[4]) == 0
        want = rotated(tiny.double().cpu()[None], group)
        top = float(want.abs().max())
        assert float((q[5].cpu().double() - want * 127 / top).abs().max()) <= 0.5 + 130 * U
        q, s, _ = qlin().add_rms_norm_int8(up, None, None, convrot_groupsize=group)
        q0, s0, _ = qlin().add_rms_norm_int8(clean, None, None, convrot_groupsize=group)
        assert not bool(s[1:4].isfinite().any()) and torch.equal(q[0], q0[0]) and torch.equal(s[0], s0[0])
        assert bool((q[4] == 0).all()) and float(s[4]) == 0
        assert float((q[5].cpu().double() - want * 127 / top).abs().max()) <= 0.5 + 130 * U


@pytest.mark.parametrize("kind", ["rows", "odd", "columns"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(kind, dtype):
    """Rows of a larger tensor, at odd addresses, columns first: the bits of rows one behind the other."""
    Q = qlin()
    for w, groups in ((256, (4, 256)), (1000, (4, 8)), (4112, (16,)), (5376, (256,)), (13824, (64, 256)), (16640, (4,))):
        gate, up = rand(5, w, seed=w, scale=3.0).to(dtype).to(DEV), rand(5, w, seed=w + 1, dtype=dtype).to(DEV)
        g = (1 + 0.2 * rand(w, seed=2)).to(dtype).to(DEV)
        a, b = layouts(gate, kind), layouts(up, kind)
        for group in groups:
            for x, y in zip(Q.gated_act_int8(gate, up, convrot_groupsize=group), Q.gated_act_int8(a, b, convrot_groupsize=group)):
                assert torch.equal(x, y)
            for res, other in ((up, b), (None, None)):
                for x, y in zip(Q.add_rms_norm_int8(gate, res, g, convrot_groupsize=group), Q.add_rms_norm_int8(a, other, g, convrot_groupsize=group)):
                    assert torch.equal(x, y)


@pytest.mark.parametrize("pad", [1, 2, 4, 8])
def test_codes_at_any_address(pad):
    """Through the C ABI: codes in rows of a larger buffer, which stays as it was around them."""
    from qlin import _lib
    L, d = _lib.load(), _lib.desc
    for w, group in ((1024, 256), (1000, 0), (1000, 8), (13824, 128), (33024, 4)):
        gate, up = rand(4, w, seed=w, dtype=BF16).to(DEV), rand(4, w, seed=1, dtype=BF16).to(DEV)
        want, ws = qlin().gated_act_int8(gate, up, convrot_groupsize=group)
        wn, wns, wh = qlin().add_rms_norm_int8(gate, up, None, convrot_groupsize=group)
        for op in ("act", "norm"):
            big = torch.full((6, w + 2 * pad + 16), 99, dtype=torch.int8, device=DEV)
            q, s, h = big[1:5, pad:pad + w], torch.empty(4, device=DEV), torch.empty_like(gate)
            if op == "act":
                assert L.qlin_gated_act_int8(d(gate), d(up), 0, group, d(q), d(s), _lib.stream_of(q.device)) == 0
                assert torch.equal(q, want) and torch.equal(s[:, None], ws)
            else:
                assert L.qlin_add_rms_norm_int8(d(gate), d(up), None, 1e-6, group, d(q), d(s), d(h), _lib.stream_of(q.device)) == 0
                assert torch.equal(q, wn) and torch.equal(s[:, None], wns) and torch.equal(h, wh)
            q.fill_(99)
            assert bool((big == 99).all())
