"""That the tests of rotated 8-bit rows see a rotation of too few parts: the kernel's products on the CPU, as three bf16 parts a value and as two."""
import math

import pytest
import torch
from mlp_ref import rotated
from rotation_ref import GROUPS, check_whole, model, whole_rows


def held(sums, group):
    """Codes and scale of unnormalized sums, in the kernel's roundings."""
    sums = sums.float()
    top = sums.abs().amax(-1, keepdim=True)
    codes = torch.round((sums.double() * (127 / top).double()))
    return codes.to(torch.int8), (top.double() / math.sqrt(group) / 127).float()


@pytest.mark.parametrize("group", GROUPS)
def test_three_parts_are_exact_and_two_are_seen(group):
    v = whole_rows(4, 2048, group, seed=group)
    want = rotated(v.double(), group) * math.sqrt(group)
    assert float((model(v, group, 3, False) - want).abs().max()) < 2.0 ** -20  # float64's own sums
    check_whole(*held(model(v, group, 3, False), group), v, group, 1.0, 0)
    for rounded_parts in (False, True):
        with pytest.raises(AssertionError):
            check_whole(*held(model(v, group, 2, rounded_parts), group), v, group, 1.0, 0)
