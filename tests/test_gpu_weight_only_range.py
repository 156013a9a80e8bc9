"""Products with 4-bit weights at the ends of the number range, against fp64:
sums of a group that pass fp32's largest number before their scale brings them
back, and rows of bf16's smallest numbers."""

import pytest
import torch

from pir2_b200 import _lib, ops
from int4_reference import pack, unpack

pytestmark = pytest.mark.gpu

SHAPES = [(5, 200, 512), (12, 777, 768), (40, 5000, 512)]


def dense(packed, scales):
    group = 2 * packed.shape[1] // scales.shape[1]
    return unpack(packed).double() * scales.double().repeat_interleave(group, dim=1)


@pytest.fixture(params=[0, 1, 2], ids=["chosen", "direct", "rows kept"])
def plan(request):
    """Both ways of running the same product."""
    previous = _lib.set_w4_mode(request.param)
    yield request.param
    _lib.set_w4_mode(previous)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_sums_of_a_group_beyond_the_range_that_their_scale_brings_back(group, m, n, k, plan):
    g = torch.Generator(device="cuda").manual_seed(m)
    codes = torch.randint(1, 8, (n, k), generator=g, device="cuda").to(torch.int8)
    codes[::2] = -8
    scales = torch.exp2(torch.randint(-20, -13, (n, k // group), generator=g, device="cuda").float()).to(torch.bfloat16)
    packed = pack(codes)
    x = torch.randn(m, k, generator=g, device="cuda").to(torch.bfloat16)
    x[0] = torch.finfo(torch.bfloat16).max                                 # 8 * 128 of them: 2^138
    x[1] = 2.0**126
    x[2] = torch.where(torch.arange(k, device="cuda") % group == 5, 2.0**126, 1.0)   # one in a group
    x[3] = 2.0**127 * torch.where(torch.rand(k, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    x[m - 1, k // 2 :] = 0                                                 # beside an ordinary row
    bias = torch.randn(n, generator=g, device="cuda").to(torch.bfloat16) if m % 2 else None
    out = ops.gemm_w4a16(x, packed, scales, bias)
    w = dense(packed, scales)
    want, mass = x.double() @ w.T, x.double().abs() @ w.abs().T
    if bias is not None:
        want, mass = want + bias.double(), mass + bias.double().abs()
    assert want.abs().max() < 2.0**128
    # As for ordinary rows: 2^-15 of the magnitudes for fp32 sums, half a step for bf16.
    far = ~((out.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-14 * mass)
    assert not far.any(), f"{int(far.sum())} values"
    assert _lib.device_status() == 0


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_results_beyond_the_range_are_infinities(m, n, k, plan):
    packed = pack(torch.full((n, k), -8, device="cuda", dtype=torch.int8))
    scales = torch.ones(n, k // 64, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    x[0, :], x[1, 3], x[2, 7] = 2.0**127, 2.0**126, -(2.0**124)
    out = ops.gemm_w4a16(x, packed, scales)
    assert (out[0] == -float("inf")).all() and (out[1] == -float("inf")).all()
    assert (out[2] == 2.0**127).all() and (out[3:] == 0).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_rows_of_the_smallest_numbers(group, m, n, k, plan):
    """Rows around bf16's smallest normal number and below it."""
    g = torch.Generator(device="cuda").manual_seed(n)
    codes = torch.randint(-8, 8, (n, k), generator=g, device="cuda").to(torch.int8)
    scales = torch.exp2(torch.randint(-4, 12, (n, k // group), generator=g, device="cuda").float()).to(torch.bfloat16)
    packed = pack(codes)
    power = torch.tensor([-126, -128, -120, -110, -100], device="cuda")[torch.arange(m, device="cuda") % 5]
    x = torch.ldexp(torch.randn(m, k, generator=g, device="cuda").double(), power[:, None].double()).to(torch.bfloat16)
    out = ops.gemm_w4a16(x, packed, scales)
    w = dense(packed, scales)
    want, mass = x.double() @ w.T, x.double().abs() @ w.abs().T
    # Sums are kept at 2^-10 of themselves, in steps of 2^-149: a product, a
    # group's and the result's addition each lose at most a step, 2^-139 of the
    # result, the first k of them times the group's scale (at most 2^11).  The
    # result's half step below bf16's normal numbers is 2^-134.
    lost = k * 2.0**-139 * 2.0**11 + 2 * (k // group + 16) * 2.0**-139 + 2.0**-134
    far = ~((out.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-14 * mass + lost)
    assert not far.any(), f"{int(far.sum())} values"
    # The bound says something: a typical result is far above it.
    assert (want.abs().median(dim=1).values > 16 * lost)[2::5].all()
    assert _lib.device_status() == 0
