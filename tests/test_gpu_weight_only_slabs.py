"""4-bit products whose rows fit shared memory in several parts of K of which the
last is shorter."""

import pytest
import torch

from pir2_b200 import _lib, ops
from test_gpu_weight_only import check, rows, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64, 128])
# Parts of 1280 and 1024; three of 768 and 512; three of 1024 and 512; three of 1536 and 768; 3584 and 3328; the first again.
@pytest.mark.parametrize("m,n,k", [(40, 5000, 2304), (64, 777, 2816), (33, 6001, 3584), (20, 4100, 5376), (12, 4200, 6912), (100, 4100, 2304)])
def test_last_part_of_k_shorter_than_the_others(group, m, n, k):
    packed, scales = weights(n, k, group, seed=m)
    x, bias = rows(m, k, seed=n), rows(1, n, seed=1)[0]
    previous = _lib.set_w4_mode(2)
    try:
        out = ops.gemm_w4a16(x, packed, scales, bias)
        assert torch.equal(out, ops.gemm_w4a16(x, packed, scales, bias))
    finally:
        _lib.set_w4_mode(previous)
    check(out, x, packed, scales, bias)
