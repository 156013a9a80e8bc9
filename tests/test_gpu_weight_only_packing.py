"""Scales of 4-bit weights where they lie on a border of bf16."""

import pytest
import torch

from pir2_b200.weight_only import quantize_groups
from int4_reference import unpack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
def test_scales_are_the_nearest_to_the_true_seventh(group):
    """7 odd / 512 over 7 is halfway between two bf16 numbers and goes to the even
    one; a product with 1 / 7 as fp32 has it would leave the border."""
    odd = torch.arange(257, 512, 2, device="cuda", dtype=torch.float64)
    w = torch.zeros(128, 2 * group, device="cuda")
    w[:, 3] = (7 * odd / 512).float()
    w[:, group + 5] = -w[:, 3]
    packed, scales = quantize_groups(w, group)
    low = (odd - 1) / 2                       # of 256ths; the odd one goes up
    want = (low + low % 2) / 256
    assert torch.equal(scales.double(), torch.stack([want, want], 1))
    codes = unpack(packed)
    assert (codes[:, 3] == 7).all() and (codes[:, group + 5] == -7).all() and codes.abs().sum() == 128 * 14
