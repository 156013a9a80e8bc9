"""Rows without a finite value but zeros, in the cache's formats, as its header
states them."""

import pytest
import torch

from pir2_b200 import _lib, ops
from pir2_b200.kv_cache import KVPages, Sequences

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize(
    "dtype,value", [(torch.uint8, 0.0), (torch.int8, 127.0), (torch.float8_e4m3fn, 448.0), (torch.bfloat16, float("inf"))],
    ids=["int4", "int8", "e4m3", "bf16"])
def test_rows_of_infinities_and_zeros(dtype, value, d, append):
    qkv = torch.zeros(3, 3, d, device="cuda", dtype=torch.bfloat16)
    qkv[0, 1:, 5], qkv[1, 1:] = float("inf"), -float("inf")
    qkv[2, 1:, 7], qkv[2, 1:, 40] = 2.0, float("inf")         # beside a finite value an infinity counts as it
    pages = KVPages.allocate(2, 1, d, page_size=16, dtype=dtype)
    sequences = Sequences(ints([0, 3]), ints([3]), ints([[1]]))
    if append:                                                # turned by no angle, k would be inf * 0: v alone
        ops.cache_append(qkv, pages, sequences, torch.ones(3, d // 2, device="cuda"), torch.zeros(3, d // 2, device="cuda"))
    else:
        ops.cache_write(qkv[:, 1:2], qkv[:, 2:], pages, sequences)
    k, v = ops.cache_read(pages, Sequences(ints([0, 3]), ints([3]), ints([[1]])), 3)
    assert _lib.device_status() == 0
    for back in (v,) if append else (k, v):
        want = torch.zeros(3, d, device="cuda", dtype=torch.bfloat16)
        want[0, 5], want[1] = value, -value
        assert torch.equal(back[:2, 0], want[:2])
        if dtype != torch.bfloat16:
            # 2 within half a step: a 14th of it and 2^-4 of the factor's rounding (int4), or 2^-8.
            near = 2 * (1 / 14 + 2.0**-4) if dtype == torch.uint8 else 2.0**-7
            assert abs(back[2, 0, 7].item() - 2) <= near and back[2, 0, 40] == back[2, 0, 7]
        elif value:
            assert back[2, 0, 7] == 2 and back[2, 0, 40] == float("inf")
