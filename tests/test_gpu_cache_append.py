"""Norm, rotation and cache write of new tokens in one pass: q and k against
fp64, and the pages against cache_write of the same rows, bit for bit."""

import pytest
import torch

from pir2_b200 import _lib, ops
from pir2_b200.kv_cache import KVPages, Sequences, rotary_table
from ragged_reference import starts_of

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.int8, torch.float8_e4m3fn, torch.uint8]
IDS = ["bf16", "int8", "e4m3", "int4"]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(new, total, hq, hk, d, page, dtype, seed, norm=True):
    """(qkv, pool filled with noise, sequences, weights)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = sum(new)
    wide = torch.randn(rows, hq + 2 * hk + 1, d, generator=g, device="cuda")
    wide *= torch.exp(torch.randn(rows, 1, 1, generator=g, device="cuda"))
    qkv = wide.to(torch.bfloat16)[:, 1:]
    counts = [-(-t // page) for t in total]
    pages = KVPages.allocate(sum(counts) + 2, hk, d, page_size=page, dtype=dtype)
    for t in (pages.k, pages.v, pages.k_scale, pages.v_scale, pages.k_factor, pages.v_factor):
        if t is not None:
            raw = t.view(torch.uint8)
            raw.copy_(torch.randint(0, 120, raw.shape, generator=g, device="cuda", dtype=torch.uint8))
    order = torch.randperm(sum(counts) + 2, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(new), max(max(counts), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at : at + n]
        at += n
    weights = [torch.exp(0.3 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16) if norm else None for _ in range(2)]
    return qkv, pages, Sequences(starts_of(new), ints(total), table), weights


def state(pages):
    return [t for t in (pages.k, pages.v, pages.k_scale, pages.v_scale, pages.k_factor, pages.v_factor) if t is not None]


def as_bytes(t):
    return t.contiguous().view(torch.uint8)


def turned(x, weight, eps, cos, sin):
    """fp64 result and a bound of the fp32 error: every product and sum is off by
    2^-24 of it, a sum of squares of 128 in eight levels by 2^-21, all in all less
    than 2^-19 of the two terms that a channel adds."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    a, b = x.chunk(2, -1)
    cos, sin = cos.double()[:, None], sin.double()[:, None]
    y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    terms = torch.cat(((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()), -1)
    return y, terms * 2.0**-19


def near(got, want, slack):
    """Rounded once to bf16: half a step, 2^-8 of the value."""
    return ((got.double() - want).abs() <= 2.0**-8 * want.abs() + slack * (1 + 2.0**-8)).all()


def check(qkv, pages, sequences, weights, new, total, hq, hk, *, eps=1e-6, theta=1e4, positions=None, **given):
    rows, d = qkv.shape[0], qkv.shape[2]
    cos, sin = rotary_table(max(total) + 3, d, theta)
    expected = [t.clone() for t in state(pages)]
    source = qkv.clone()
    k_out = torch.empty(rows, hk, d, device="cuda", dtype=torch.bfloat16)
    q = ops.cache_append(qkv, pages, sequences, cos, sin, q_weight=weights[0], k_weight=weights[1], eps=eps,
                         positions=positions, k_out=k_out, **given)
    at = torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(new, total)]) if positions is None else positions.long()
    for got, part, weight in ((q, source[:, :hq], weights[0]), (k_out, source[:, hq : hq + hk], weights[1])):
        assert near(got, *turned(part, weight, eps, cos[at], sin[at]))
    # The pages: as cache_write puts the same rows.
    again = KVPages(*expected)
    ops.cache_write(k_out, source[:, hq + hk :], again, sequences)
    for got, want in zip(state(pages), expected):
        assert torch.equal(as_bytes(got), as_bytes(want))
    assert _lib.device_status() == 0
    return q


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads", [(16, 8, 128), (8, 1, 64), (5, 3, 128), (3, 3, 64), (32, 2, 128)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("new,past", [([1], [0]), ([1, 1, 1], [15, 16, 127]), ([0, 37, 700, 1], [5, 0, 60, 300])])
def test_rows_and_pages(dtype, heads, new, past):
    hq, hk, d = heads
    total = [n + p for n, p in zip(new, past)]
    for page, norm in ((16, True), (64, False)):
        qkv, pages, sequences, weights = make(new, total, hq, hk, d, page, dtype, seed=sum(total), norm=norm)
        check(qkv, pages, sequences, weights, new, total, hq, hk)


def test_values_next_to_borders_are_those_of_single_operations():
    """The same fp32 operations in torch, in the same order, give the same bits."""
    new, total = [200, 56], [230, 56]
    qkv, pages, sequences, weights = make(new, total, 16, 8, 128, 32, torch.uint8, seed=3)
    cos, sin = rotary_table(300, 128, 1e6)
    q = ops.cache_append(qkv, pages, sequences, cos, sin, q_weight=weights[0], k_weight=weights[1], eps=1e-6)
    at = torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(new, total)])
    x = qkv[:, :16].float()
    y = x[..., :64] * x[..., :64] + x[..., 64:] * x[..., 64:]
    y = y.unflatten(-1, (16, 4))
    y = (y[..., 0] + y[..., 2]) + (y[..., 1] + y[..., 3])
    while y.shape[-1] > 1:
        half = y.shape[-1] // 2
        y = y[..., :half] + y[..., half:]
    x = x * (1.0 / torch.sqrt(y / 128 + 1e-6)) * weights[0].float()
    a, b = x.chunk(2, -1)
    c, s = cos[at][:, None], sin[at][:, None]
    assert torch.equal(q, torch.cat((a * c - b * s, b * c + a * s), -1).to(torch.bfloat16))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_positions_of_their_own_and_rows_of_no_sequence(dtype):
    new, total = [3, 0, 9], [3, 20, 40]
    qkv, pages, sequences, weights = make(new, total, 4, 2, 128, 16, dtype, seed=7)
    check(qkv, pages, sequences, weights, new, total, 4, 2, positions=ints([11, 0, 5, 42, 42, 1, 2, 3, 4, 40, 30, 20]))
    more = torch.cat([qkv, qkv])                 # 12 rows behind the last sequence
    cos, sin = rotary_table(50, 128)
    out = torch.full((24, 4, 128), 3.0, device="cuda", dtype=torch.bfloat16)
    k_out = torch.full((24, 2, 128), 3.0, device="cuda", dtype=torch.bfloat16)
    before = [t.clone() for t in state(pages)]
    ops.cache_append(qkv, pages, sequences, cos, sin, q_weight=weights[0], k_weight=weights[1])
    after = [t.clone() for t in state(pages)]
    for t, x in zip(state(pages), before):
        t.copy_(x)
    ops.cache_append(more, pages, sequences, cos, sin, q_weight=weights[0], k_weight=weights[1], out=out, k_out=k_out)
    assert all(torch.equal(as_bytes(t), as_bytes(x)) for t, x in zip(state(pages), after))
    assert (out[12:] == 3).all() and (k_out[12:] == 3).all() and not (out[:12] == 3).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_in_place_in_a_replayed_graph(dtype):
    new, total = [2, 1], [30, 65]
    qkv, pages, sequences, weights = make(new, total, 8, 2, 64, 32, dtype, seed=5)
    cos, sin = rotary_table(80, 64)
    source = qkv.clone()
    want_k = torch.empty(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    want = ops.cache_append(qkv, pages, sequences, cos, sin, q_weight=weights[0], k_weight=weights[1], k_out=want_k)
    kept = [t.clone() for t in state(pages)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_append(qkv, pages, sequences, cos, sin, q_weight=weights[0], k_weight=weights[1], out=qkv[:, :8], k_out=qkv[:, 8:10])
    for t in state(pages):
        t.zero_()
    qkv.copy_(source)
    lengths = sequences.lengths.clone()
    sequences.lengths.copy_(ints([29, 60]))
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(qkv[:, :8], want)     # positions are read when the graph runs
    for t in state(pages):
        t.zero_()
    qkv.copy_(source)
    sequences.lengths.copy_(lengths)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(qkv[:, :8], want) and torch.equal(qkv[:, 8:10], want_k) and torch.equal(qkv[:, 10:], source[:, 10:])
    for b, (n, t) in enumerate(zip(new, total)):
        for p in range(t - n, t):
            slot = int(sequences.table[b, p // 32]), slice(None), p % 32
            for got, x in zip(state(pages), kept):
                whole = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[got.element_size()]
                assert torch.equal(got.view(whole)[slot], x.view(whole)[slot])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_values_that_are_not_finite_stay_in_their_rows(dtype):
    new, total = [6], [6]
    qkv, pages, sequences, weights = make(new, total, 2, 2, 128, 16, dtype, seed=9)
    cos, sin = rotary_table(8, 128)
    clean = ops.cache_append(qkv, pages, sequences, cos, sin, q_weight=weights[0], k_weight=weights[1]).clone()
    kept = [t.clone() for t in state(pages)]
    qkv[1, 0, 3], qkv[2, 3, 100], qkv[3, 4, 7], qkv[4, 5, 64] = float("nan"), float("inf"), float("inf"), float("nan")
    k_out = torch.empty(6, 2, 128, device="cuda", dtype=torch.bfloat16)
    q = ops.cache_append(qkv, pages, sequences, cos, sin, q_weight=weights[0], k_weight=weights[1], k_out=k_out)
    same = torch.ones(6, 2, dtype=torch.bool, device="cuda")
    same[1, 0] = False
    assert torch.equal(q[same], clean[same]) and not torch.isfinite(q[1, 0]).all()
    again = KVPages(*[t.clone() for t in kept])
    ops.cache_write(k_out, qkv[:, 4:], again, sequences)
    for got, want in zip(state(pages), state(again)):
        assert torch.equal(as_bytes(got), as_bytes(want))


def test_far_positions_past_the_table_and_bad_pages():
    new, total = [2], [131072]
    qkv, pages, sequences, weights = make(new, total, 2, 1, 128, 128, torch.uint8, seed=2)
    check(qkv, pages, sequences, weights, new, total, 2, 1, theta=1e6)
    kept = [t.clone() for t in state(pages)]
    cos, sin = rotary_table(131071, 128)         # the last row's position is one past it
    ops.cache_append(qkv, pages, sequences, cos, sin)
    assert _lib.device_status() == _lib.STATUS_BAD_POSITION
    last = int(sequences.table[0, -1])
    for t, x in zip(state(pages), kept):
        whole = {1: torch.uint8, 4: torch.int32}[t.element_size()]
        assert torch.equal(t.view(whole)[last, :, 127], x.view(whole)[last, :, 127])
    ops.cache_append(qkv, pages, sequences, cos, sin, positions=ints([-1, 0]))
    assert _lib.device_status() == _lib.STATUS_BAD_POSITION
    sequences.table[0, -1] = 5000
    ops.cache_append(qkv, pages, sequences, *rotary_table(131072, 128))
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE


def test_arguments_that_are_refused():
    qkv, pages, sequences, weights = make([2], [2], 2, 1, 64, 16, torch.int8, seed=1)
    cos, sin = rotary_table(4, 64)
    good = dict(q_weight=weights[0], k_weight=weights[1])
    assert ops.cache_append(qkv, pages, sequences, cos, sin, **good).shape == (2, 2, 64)
    assert ops.cache_append(qkv[:0], pages, sequences, cos, sin, **good).shape == (0, 2, 64)
    for arguments, changes in (
        ((qkv.float(), pages, sequences, cos, sin), {}),
        ((qkv[:, :2], pages, sequences, cos, sin), {}),
        ((qkv[..., :32], pages, sequences, cos, sin), {}),
        ((qkv, pages, sequences, cos[:, :16], sin), {}),
        ((qkv, pages, sequences, cos.double(), sin.double()), {}),
        ((qkv, pages, sequences, cos, sin[:2]), {}),
        ((qkv, pages, sequences, cos.cpu(), sin.cpu()), {}),
        ((qkv, pages, sequences, cos[:0], sin[:0]), {}),
        ((qkv, pages, sequences, cos, sin), {"q_weight": weights[0].float()}),
        ((qkv, pages, sequences, cos, sin), {"k_weight": weights[1][:32]}),
        ((qkv, pages, sequences, cos, sin), {"eps": float("nan")}),
        ((qkv, pages, sequences, cos, sin), {"positions": ints([0])}),
        ((qkv, pages, sequences, cos, sin), {"positions": ints([0, 1]).long()}),
        ((qkv, pages, sequences, cos, sin), {"out": qkv[:, :1]}),
        ((qkv, pages, sequences, cos, sin), {"k_out": qkv[:, 1:2].float()}),
        ((qkv, pages, sequences, cos, sin), {"k_out": torch.empty(2, 1, 68, device="cuda", dtype=torch.bfloat16)[:, :, 4:]}),
    ):
        with pytest.raises(ValueError, match="cache_append"):
            ops.cache_append(*arguments, **{**good, **changes})
    with pytest.raises(ValueError, match="rotary_table"):
        rotary_table(0, 64)
