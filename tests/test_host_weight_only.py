"""Argument checks and the packing of 4-bit weights that need no GPU."""

import pytest
import torch

from pir2_b200 import _lib
from pir2_b200.weight_only import quantize_groups
from int4_reference import unpack


def test_arguments_that_are_refused():
    lib = _lib.lib()
    good = [4096, 256, 4096, 4096, 64, None, 2, 32, 256, 4096, 32, None, None]
    for at, value, status in (
        (0, None, _lib.EINVAL), (0, 4104, _lib.EALIGN), (1, 248, _lib.EINVAL), (1, 260, _lib.EALIGN), (2, None, _lib.EINVAL),
        (2, 4100, _lib.EALIGN), (3, None, _lib.EINVAL), (3, 4100, _lib.EALIGN), (4, 48, _lib.EINVAL), (4, 0, _lib.EINVAL),
        (5, 4097, _lib.EALIGN), (6, -1, _lib.EINVAL), (7, 0, _lib.EINVAL), (8, 0, _lib.EINVAL), (8, 200, _lib.EINVAL),
        (8, 1 << 21, _lib.EINVAL), (9, None, _lib.EINVAL), (9, 4097, _lib.EALIGN), (10, 31, _lib.EINVAL),
    ):
        args = list(good)
        args[at] = value
        assert lib.pir2b_gemm_w4a16(*args) == status, (at, value)
        assert b"gemm_w4a16" in lib.pir2b_last_error()
    args = list(good)
    args[6] = 0                       # no rows: nothing to do
    assert lib.pir2b_gemm_w4a16(*args) == _lib.OK


@pytest.mark.parametrize("group", [32, 64, 128])
def test_groups_are_packed_as_stated(group):
    w = torch.randn(5, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    w[2, :group] = 0
    packed, scales = quantize_groups(w, group)
    assert packed.shape == (5, 128) and packed.dtype == torch.uint8 and scales.shape == (5, 256 // group)
    codes = unpack(packed).double()
    assert codes.abs().max() == 7 and scales[2, 0] == 1
    back = codes.unflatten(1, (-1, group)) * scales.double()[..., None]
    most = w.double().unflatten(1, (-1, group)).abs().amax(-1, keepdim=True)
    assert ((back - w.double().unflatten(1, (-1, group))).abs() <= most * (0.5 / 7 + 2.0**-8)).all()
