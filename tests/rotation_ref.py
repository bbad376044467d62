"""Rows whose rotation is exact in fp32, and what the codes and scales of rotated rows may be off by."""
import math

import torch
from mlp_ref import F32, U, rotated, within

GROUPS = [4, 8, 16, 32, 64, 128, 256]


def whole_rows(t, w, group, seed=0):
    """fp32 rows of odd whole numbers as wide as the sums of a group's stay below 2^24: all of a rotation's sums are exact in fp32, in
    any order, and most values and half-rotated values need more than 16 bits."""
    most = 2 ** (24 - int(math.log2(group))) - 1
    v = torch.randint(-most // 2, most // 2, (t, w), generator=torch.Generator().manual_seed(seed)) * 2 + 1
    return v.clamp(-most, most).to(F32)


def check_whole(codes, scale, rows, group, factor, more):
    """codes and scale of rows (float64 whole numbers) times `factor`.  The largest magnitude is exact before the factor of an odd power of
    2's root, so that the scale has at most 3 roundings (that factor's own, its product, the quotient) and `more`; a code is the
    product with a quotient of one rounding, 127 * 2^-24 of a step, added to a whole number in one rounding to nearest."""
    codes, scale, want = codes.cpu().double(), scale.cpu().double(), rotated(rows.cpu().double(), group)
    top = want.abs().amax(-1, keepdim=True)
    within(scale, factor * top / 127, factor * top / 127 * (4 + more) * U)
    assert float((codes - want * 127 / top).abs().max()) <= 0.5 + 130 * U
    assert bool((codes.abs().amax(-1) == 127).all())


def check_rotated(codes, scale, v, off, group):
    """codes and scale of rows v (float64, before the rotation) whose values the kernel has within `off`.  The rotation: off through the
    sums as it is, its own roundings 70 * 2^-24 of a group's norm.  (A value of n1 or n2 <= 16 terms is a sum over three parts, the two
    lower ones 2^-8 of it: 17 additions of up to 2 half steps each with their share, 34.3 U times the terms' sum of magnitudes, which
    is at most sqrt(n1 n2) norms in the second product, through sqrt(n2) of it from sqrt(n1) in the first: both sqrt(G) norms,
    over sqrt(G).)"""
    g = v.reshape(-1, group)
    want = rotated(v, group)
    more = (off.reshape(-1, group).sum(-1, keepdim=True) / math.sqrt(group) + 70 * U * g.norm(dim=-1, keepdim=True)).expand(g.shape).reshape(v.shape)
    top, most = want.abs().amax(-1, keepdim=True), more.amax(-1, keepdim=True)
    assert float((most / top).max()) < 0.1
    within(scale, top / 127, 1.01 * most / 127 + top / 127 * 6 * U)
    codes = codes.cpu().double()
    room = 0.5 + 127 * (1.01 * (more / top + want.abs() * most / (top * (top - most))) + 8 * U)
    over = (codes - want * 127 / top).abs() - room
    assert float(over.max()) <= 0, float(over.max())


def model(v, group, parts, rounded_parts):
    """The rotation's sums of fp32 rows v in float64, each value as `parts` bf16 parts: truncated, or rounded to nearest."""
    def product(x, m):
        left, out = x.float(), torch.zeros_like(x)
        for _ in range(parts):
            part = left.to(torch.bfloat16).float() if rounded_parts else (left.view(torch.int32) & -65536).view(F32)
            left = left - part
            out = out + part.double() @ m
        return out
    n1 = min(group, 16)
    n2 = group // n1
    eye = lambda n: torch.eye(n, dtype=torch.float64)  # noqa: E731
    low, high = rotated(eye(n1), n1) * math.sqrt(n1), rotated(eye(n2), n2) * math.sqrt(n2)
    x = product(v.double().reshape(-1, n1), low.T).reshape(-1, n2, n1).transpose(1, 2)
    return product(x.reshape(-1, n2), high.T).reshape(-1, n1, n2).transpose(1, 2).reshape(v.shape)
