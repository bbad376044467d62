"""The norm's sums over rows near the longest ones, in fp32."""
import pytest
import torch
from mlp_ref import DEV, F32, U, norm, qlin, rand, rounded, within
from test_gpu_add_norm import grad as norm_grad

pytestmark = pytest.mark.gpu
LONGEST = 1 << 20


@pytest.mark.parametrize("w", [LONGEST, LONGEST - 3, 300000])
def test_sums_of_very_long_rows(w):
    """Equal values whose squares are lost in part when they are added to a sum of a thousand of them: the sums' roundings have to stay
    those of bound_y's tests, (32 + 16) and fewer than 64 in any case.  In the gradient rho has half of a sum's 64 roundings, mean(g h)
    its own 64 and twice rho's, and six more operations: 64 + 64 + 32 + 20 of the terms' size."""
    Q = qlin()
    value = 1 + 0.45 * 2.0 ** -14
    x = torch.full((2, w), value, device=DEV)
    x[1] = rand(w, seed=1).to(DEV)
    y, _ = Q.add_rms_norm(x)
    want, _ = norm(x.double().cpu(), None, None)
    within(y, want, rounded(F32, want, 64 * U * want.abs()))
    for group in (0, 4):
        if group and w % group:
            continue
        _, s, _ = Q.add_rms_norm_int8(x[:1], None, None, convrot_groupsize=group)
        top = float(x[0, 0].double())  # the rotation of four equal values: 2 v / 2
        rho = 1 / (top ** 2 + 1e-6) ** 0.5
        within(s, torch.full((1, 1), top * rho / 127, dtype=torch.float64), top * rho / 127 * 64 * U)
    dy = torch.ones(2, w, device=DEV)
    dy[1] = rand(w, seed=2).to(DEV)
    dx, dw = Q.add_rms_norm_grad(dy, None, x, torch.ones(w, device=DEV))
    wx, size, ww, total = norm_grad(dy.double().cpu(), None, x.double().cpu(), torch.ones(w, dtype=torch.float64))
    within(dx, wx, rounded(F32, wx, 180 * U * size))
    within(dw, ww, rounded(F32, ww, 66 * U * total))
