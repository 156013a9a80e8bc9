"""Argument checks of the ragged-batch entry points that need no GPU: the C
ABI refuses bad shapes before any device call, and the Python handles refuse
host tensors."""

import ctypes

import numpy as np
import pytest
import torch

from pir2_b200 import _lib, ops
from pir2_b200.kv_cache import KVPages, Sequences


def pages(**changes):
    fields = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, k_page_stride=8 * 64 * 128, v_page_stride=8 * 64 * 128,
                  k_scale_page_stride=8 * 64, v_scale_page_stride=8 * 64, pages=4, page_size=64, kv_heads=8,
                  head_dim=128, format=_lib.CACHE_INT8)
    fields.update(changes)
    return _lib.KVPagesStruct(**fields)


def sequences(**changes):
    fields = dict(starts=4096, lengths=4096, table=4096, table_stride=4, batch=2, table_width=4)
    fields.update(changes)
    return _lib.SequencesStruct(**fields)


def attention(p, s, *, q=4096, q_row=2048, q_head=128, rows=2, hq=16, scale=1.0, out=4096, ldo=2048):
    return _lib.lib().pir2b_cache_attention(
        q, q_row, q_head, rows, hq, ctypes.byref(p), ctypes.byref(s), scale, out, ldo, None, None
    )


@pytest.mark.parametrize(
    "changes,status,text",
    [
        ({"page_size": 48}, _lib.EINVAL, b"page_size"),
        ({"head_dim": 96}, _lib.EINVAL, b"head_dim"),
        ({"format": 4}, _lib.EINVAL, b"format"),
        ({"pages": 0}, _lib.EINVAL, b"pages"),
        ({"kv_heads": 0}, _lib.EINVAL, b"kv heads"),
        ({"k": None}, _lib.EINVAL, b"k, v"),
        ({"k_page_stride": 64}, _lib.EINVAL, b"stride"),
        ({"k": 4104}, _lib.EALIGN, b"aligned"),
        ({"v_page_stride": 8 * 64 * 128 + 8}, _lib.EALIGN, b"aligned"),
        ({"k_scale": None}, _lib.EINVAL, b"scales"),
        ({"v_scale_page_stride": 8}, _lib.EINVAL, b"scales"),
    ],
)
def test_pools_that_are_refused(changes, status, text):
    lib, p, s = _lib.lib(), pages(**changes), sequences()
    assert attention(p, s) == status and text in lib.pir2b_last_error()
    assert lib.pir2b_cache_write(4096, 1024, 128, 4096, 1024, 128, 2, ctypes.byref(p), ctypes.byref(s), None) == status
    assert lib.pir2b_cache_read(ctypes.byref(p), ctypes.byref(s), 2, 4096, 4096, None) == status


@pytest.mark.parametrize(
    "changes", [{"starts": None}, {"lengths": None}, {"table": None}, {"batch": 0}, {"table_width": -1}, {"table_stride": 3}]
)
def test_sequences_that_are_refused(changes):
    assert attention(pages(), sequences(**changes)) == _lib.EINVAL


@pytest.mark.parametrize(
    "changes,status",
    [
        ({"rows": -1}, _lib.EINVAL),
        ({"hq": 12}, _lib.EINVAL),
        ({"hq": 0}, _lib.EINVAL),
        ({"scale": 0.0}, _lib.EINVAL),
        ({"scale": float("nan")}, _lib.EINVAL),
        ({"q": None}, _lib.EINVAL),
        ({"q": 4100}, _lib.EALIGN),
        ({"q_row": 2044}, _lib.EALIGN),
        ({"out": None}, _lib.EINVAL),
        ({"ldo": 2040}, _lib.EINVAL),
        ({"ldo": 2052}, _lib.EALIGN),
    ],
)
def test_queries_that_are_refused(changes, status):
    assert attention(pages(), sequences(), **changes) == status


def test_prompt_arguments_that_are_refused():
    lib = _lib.lib()
    good = [4096, 4096, 128, 4096, 4096, 128, 4096, 4096, 128, 4096, 2, 10, 16, 8, 128, 1.0, 4096, 2048, None]
    for at, value in ((0, None), (0, 4100), (1, 4), (3, None), (5, 2), (6, None), (9, None), (10, 0), (11, -1), (12, 12),
                      (13, 0), (14, 48), (15, -1.0), (16, None), (16, 4100), (17, 2000)):
        args = list(good)
        args[at] = value
        assert lib.pir2b_prompt_attention(*args) in (_lib.EINVAL, _lib.EALIGN), (at, value)
    args = list(good)
    args[11] = 0                      # no rows: nothing to do
    assert lib.pir2b_prompt_attention(*args) == _lib.OK


def test_host_tensors_are_refused():
    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        KVPages(k, k)
    with pytest.raises(ValueError, match="CUDA"):
        Sequences(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32))
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.prompt_attention(x, x, x, torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("limit", [127, 448])
def test_quotients_of_the_cache_quantiser_are_correctly_rounded(limit):
    """The quantiser divides a bf16 x by s = f32(1/L) * (a bf16) as q = x y,
    q + (x - q s) y with y = 1 / s: for every pair of significands and every
    exponent whose code is not 0 that is the correctly rounded quotient
    (fp64 holds x - q s exactly, as an FMA does)."""
    f = np.float32
    significand = f(1) + np.arange(128, dtype=f) / f(128)
    s = significand * (f(1) / f(limit))
    y = f(1) / s
    for shift in range(20):
        x = (significand * f(2.0**-shift))[:, None]
        q = x * y
        rest = (x.astype(np.float64) - q.astype(np.float64) * s).astype(f)
        q = (q.astype(np.float64) + rest.astype(np.float64) * y).astype(f)
        inside = x <= significand            # s belongs to the row's largest value
        assert np.array_equal(np.broadcast_to(x / s, q.shape)[inside], q[inside])
