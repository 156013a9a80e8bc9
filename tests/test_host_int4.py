"""The 4-bit cache's checks and arithmetic that need no GPU."""

import ctypes

import numpy as np
import pytest
import torch

from pir2_b200 import _lib
from int4_reference import pack, quantise4, unpack, values4


def pages(**changes):
    fields = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, k_page_stride=8 * 64 * 64, v_page_stride=8 * 64 * 64,
                  k_scale_page_stride=8 * 64, v_scale_page_stride=8 * 64, pages=4, page_size=64, kv_heads=8,
                  head_dim=128, format=_lib.CACHE_INT4, k_factor=4096, v_factor=4096, k_factor_page_stride=8 * 64 * 4,
                  v_factor_page_stride=8 * 64 * 4)
    fields.update(changes)
    return _lib.KVPagesStruct(**fields)


@pytest.mark.parametrize(
    "changes,text",
    [
        ({"k_factor": None}, b"factors"),
        ({"v_factor": None}, b"factors"),
        ({"k_factor": 4104}, b"factors"),
        ({"v_factor_page_stride": 8 * 64 * 4 - 16}, b"factors"),
        ({"k_factor_page_stride": 8 * 64 * 4 + 8}, b"factors"),
        ({"k_page_stride": 8 * 64 * 64 - 16}, b"stride"),
        ({"v_page_stride": 8 * 64 * 64 + 8}, b"aligned"),
        ({"k_scale": None}, b"scales"),
        ({"head_dim": 96}, b"head_dim"),
    ],
)
def test_pools_that_are_refused(changes, text):
    lib, p = _lib.lib(), pages(**changes)
    s = _lib.SequencesStruct(starts=4096, lengths=4096, table=4096, table_stride=4, batch=2, table_width=4)
    bad = (_lib.EINVAL, _lib.EALIGN)
    assert lib.pir2b_cache_attention(4096, 2048, 128, 2, 16, ctypes.byref(p), ctypes.byref(s), 1.0, 4096, 2048, None, None) in bad
    assert text in lib.pir2b_last_error()
    assert lib.pir2b_cache_write(4096, 1024, 128, 4096, 1024, 128, 2, ctypes.byref(p), ctypes.byref(s), None) in bad
    assert lib.pir2b_cache_read(ctypes.byref(p), ctypes.byref(s), 2, 4096, 4096, None) in bad


def test_quotients_of_the_4_bit_quantiser_give_the_codes_of_the_true_ones():
    """A code is v / f for a v of 8 and an f of 4 significant bits, computed as
    q = v y, q + (v - q f) y with y = 1 / f in fp32: for every pair of
    significands and every exponent whose code is not 0, and every border of two
    codes among them, it rounds as the true quotient does."""
    f32 = np.float32
    for top in range(8, 16):
        f = f32(top / 8)
        y = f32(1) / f
        for exponent in range(-4, 4):
            v = (np.arange(128, 256) / 128 * 2.0**exponent).astype(f32)
            q = v * y
            rest = (v.astype(np.float64) - q.astype(np.float64) * float(f)).astype(f32)
            q = (q.astype(np.float64) + rest.astype(np.float64) * float(y)).astype(f32)
            # v and f are whole numbers of 2^-11 and 2^-3: the true quotient's place from whole numbers.
            a, b = (v.astype(np.float64) * 2**11).astype(np.int64), int(f * 8) * 2**8
            low, rest = a // b, a % b
            true = low + ((2 * rest > b) | ((2 * rest == b) & (low % 2 == 1)))
            assert np.array_equal(np.rint(q).astype(np.int64), true)


def test_seventh_parts_round_to_the_nearest_factor():
    """m / 7 in fp32 and then to E4M3 is m / 7 to E4M3: no quotient of a bf16
    by 7 lies so near a border that the first rounding moves it across."""
    m = (torch.arange(128, 256).double() / 128)[None] * torch.pow(2.0, torch.arange(-12, 11).double())[:, None]
    got = (m.float() / torch.full_like(m.float(), 7.0)).to(torch.float8_e4m3fn).double()
    exponent = torch.frexp((m / 7).clamp(min=2.0**-6)).exponent - 1
    step = torch.pow(2.0, (exponent - 3).double())
    units = m / step                                                  # 7 times the quotient in steps, exact
    low = torch.floor(units / 7)
    twice = 2 * (units - 7 * low)
    want = (low + ((twice > 7) | ((twice == 7) & (low % 2 == 1))).double()) * step
    assert torch.equal(got, want)


@pytest.mark.parametrize("places", [-3, -2, -1, 1, 2, 3])
def test_codes_from_a_reciprocal_that_is_off(places):
    """The same codes where 1 / f is off by some places of its last bit, as an
    approximate reciprocal may be: the sum q + 1.5 2^23 rounds as the kernel's does."""
    f32 = np.float32
    for top in range(8, 16):
        f = f32(top / 8)
        y = (f32(1) / f).view(np.int32) + np.int32(places)
        y = y.view(f32)
        for exponent in range(-4, 4):
            v = (np.arange(128, 256) / 128 * 2.0**exponent).astype(f32)
            q = v * y
            rest = (v.astype(np.float64) - q.astype(np.float64) * float(f)).astype(f32)
            q = (q.astype(np.float64) + rest.astype(np.float64) * float(y)).astype(f32)
            a, b = (v.astype(np.float64) * 2**11).astype(np.int64), int(f * 8) * 2**8
            low, rest = a // b, a % b
            true = low + ((2 * rest > b) | ((2 * rest == b) & (low % 2 == 1)))
            assert np.array_equal(((q + f32(12582912)) - f32(12582912)).astype(np.int64), true)


def test_seventh_parts_by_a_product_and_one_step():
    """q = m fl(1/7), q + (m - 7 q) fl(1/7) is the correctly rounded m / 7 for every bf16 m."""
    f32 = np.float32
    m, y = np.arange(128, 256).astype(f32), f32(1) / f32(7)
    q = m * y
    rest = (m.astype(np.float64) - 7 * q.astype(np.float64)).astype(f32)
    q = (q.astype(np.float64) + rest.astype(np.float64) * float(y)).astype(f32)
    assert np.array_equal(q, m / f32(7))


@pytest.mark.parametrize(
    "changes,text",
    [
        ({"hq": 0}, b"query heads"),
        ({"hq": 1025}, b"query heads"),
        ({"eps": -1e-6}, b"eps"),
        ({"eps": float("inf")}, b"eps"),
        ({"eps": float("nan")}, b"eps"),
        ({"cos": None}, b"cos"),
        ({"sin": None}, b"cos"),
        ({"turns": 0}, b"cos"),
        ({"sin": 4100}, b"aligned"),
        ({"q_weight": 4098}, b"aligned"),
        ({"k_weight": 4104}, b"aligned"),
        ({"qkv": None}, b"qkv"),
        ({"qkv": 4104}, b"qkv"),
        ({"row": 32 * 128 + 4}, b"qkv"),
        ({"head": 12}, b"qkv"),
        ({"q_out": None}, b"q"),
        ({"q_row": 16 * 128 - 8}, b"q"),
        ({"k_out": 4104}, b"k"),
        ({"k_row": 8 * 128 - 8, "k_out": 4096}, b"k"),
        ({"rows": -1}, b"rows"),
    ],
)
def test_appends_that_are_refused(changes, text):
    args = dict(qkv=4096, row=32 * 128, head=128, rows=2, hq=16, q_weight=4096, k_weight=4096, eps=1e-6, cos=4096, sin=4096,
                turns=512, positions=None, q_out=4096, q_row=16 * 128, k_out=None, k_row=0)
    args.update(changes)
    lib, p = _lib.lib(), pages()
    s = _lib.SequencesStruct(starts=4096, lengths=4096, table=4096, table_stride=4, batch=2, table_width=4)
    order = ("qkv", "row", "head", "rows", "hq", "q_weight", "k_weight", "eps", "cos", "sin", "turns", "positions")
    status = lib.pir2b_cache_append(*[args[x] for x in order], ctypes.byref(p), ctypes.byref(s), args["q_out"], args["q_row"],
                                    args["k_out"], args["k_row"], None)
    assert status in (_lib.EINVAL, _lib.EALIGN)
    assert text in lib.pir2b_last_error()


def test_plain_form_of_the_format():
    x = torch.randn(5, 3, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    packed, scale, factor = quantise4(x)
    assert packed.shape == (5, 3, 64) and factor.shape == (5, 3, 4)
    assert torch.equal(pack(unpack(packed)), packed)
    # Half a step is a 14th of a group's largest value, and its factor's rounding 2^-4 of that value.
    far = (values4(packed, scale, factor) - x.double()).abs().unflatten(-1, (-1, 32))
    most = x.double().abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True)
    assert (far <= most * ((1 + 2.0**-4) / 14 + 2.0**-4)).all()
