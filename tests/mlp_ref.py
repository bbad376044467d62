"""The MLP side's formulas in 64 bits, and what the tests share."""
import math

import torch

DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = 2.0 ** -24            # half a step of fp32, relative
H4 = ((1, 1, 1, -1), (1, 1, -1, 1), (1, -1, 1, 1), (-1, 1, 1, 1))
SMALLEST = {F16: 2.0 ** -25, BF16: 2.0 ** -126, F32: 2.0 ** -126}  # what an output below the normal numbers may lose


def qlin():
    import qlin as Q
    return Q


def rand(*shape, seed=0, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, bound):
    """got (any float dtype) is within bound of want (float64), element by element."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    bound = bound.cpu() if torch.is_tensor(bound) else torch.full_like(want, bound)
    assert got.shape == want.shape, (got.shape, want.shape)
    off = (got - want).abs() - bound
    assert not bool((~(off <= 0)).any()), f"{float(off.max())} past the bound, of {float(want.abs().max())}"


def rounded(dtype, want, more):
    """An output's bound: half a step of its dtype and `more`, what the fp32 arithmetic may add."""
    return half_step(dtype) * (want.abs() + more) + more + SMALLEST[dtype]


def rotated(v, g):
    if not g:
        return v
    h = torch.ones(1, 1, dtype=v.dtype)
    while h.shape[0] * 4 <= g:
        h = torch.kron(h, torch.tensor(H4, dtype=v.dtype))
    if h.shape[0] < g:
        h = torch.kron(torch.tensor(((1, 1), (1, -1)), dtype=v.dtype), h)
    return (v.reshape(-1, g) @ h.T / math.sqrt(g)).reshape(v.shape)


def norm(x, r, w, eps=1e-6):
    """(y, h) of float64 rows."""
    h = x if r is None else x + r
    y = h * (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    return (y if w is None else y * w), h


def check_codes(codes, scale, want, group=0):
    """codes [.., W] int8 with scale [.., 1] for the float64 rows `want`: the scale is the largest magnitude / 127, and a code is off
    by half a step and a slack at most.  In fp32 that is 127 * 16 * 2^-24 of a step; through the rotation a value is off by
    2^-17 of its group's norm, which is at most 16 times the row's largest value: 127 * 16 * 2^-17 = 0.0155 of a step, and
    16 * 2^-17 = 2^-13 of the scale."""
    slack = 0.018 if group else 0.001
    codes, scale, want = codes.cpu().double(), scale.cpu().double(), want.cpu()
    top = want.abs().amax(-1, keepdim=True)
    assert codes.shape == want.shape and scale.shape == top.shape
    within(scale, top / 127, top / 127 * (2.0 ** -13 if group else 200 * U) + 2.0 ** -149)
    steps = torch.where(top > 0, want * 127 / torch.where(top > 0, top, 1.0), 0.0)
    assert float((codes - steps).abs().max()) <= 0.5 + slack
    assert bool(((codes.abs().amax(-1, keepdim=True) == 127) == (top > 0)).all())


def act(z, kind):
    """(f, f', t) of float64 z."""
    if kind == "silu":
        t, dt = z, torch.ones_like(z)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        t, dt = c * (z + 0.044715 * z ** 3), c * (1 + 3 * 0.044715 * z ** 2)
    s = torch.sigmoid(t)
    return z * s, s + z * s * torch.sigmoid(-t) * dt, t


def sigma_bound(t, dtype):
    """What sigma's fp32 evaluation may be off by, relative: t's own roundings (4 half steps of |t|, which sigma takes over as
    they are where e^-t counts), then the exponential's, the sum's and the quotient's."""
    return (4 * t.abs().clamp(max=128) + (16 if dtype == F32 else 32)) * U


def layouts(x, kind):
    """x [T, W] with the same values in another place: rows of a larger tensor, at an odd address, or three dimensions."""
    t, w = x.shape
    if kind == "rows":
        big = torch.empty(t, w + 24, dtype=x.dtype, device=x.device)
        big[:, 8:8 + w] = x
        return big[:, 8:8 + w]
    if kind == "odd":
        big = torch.empty(t * (w + 1) + 1, dtype=x.dtype, device=x.device)[1:].view(t, w + 1)
        big[:, :w] = x
        return big[:, :w]
    if kind == "columns":
        return x.t().contiguous().t()
    return x
