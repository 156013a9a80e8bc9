"""Prompt and cache attention where values, masks and shapes are extreme,
against fp64."""

import pytest
import torch

from pir2_b200 import _lib, ops
from pir2_b200.kv_cache import KVPages, Sequences
from ragged_reference import attend, quantise, starts_of, tolerance, values

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.int8, torch.float8_e4m3fn]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def compare(out, q, k, v, scale):
    """One sequence: rows that see only finite keys and values against fp64,
    the others not finite."""
    n, hq, d = q.shape
    hidden = max(0, n - k.shape[0])          # rows before the first position see nothing
    want, mass, spoiled = attend(q[hidden:], k, v, scale)
    got = out.view(n, hq, d).double()
    assert (got[:hidden] == 0).all()
    got = got[hidden:]
    far = ((got - want).abs() > tolerance(want, mass)) | ~torch.isfinite(got)
    assert not (far & ~spoiled).any(), f"{int((far & ~spoiled).sum())} of {far.numel()} values"
    assert not torch.isfinite(got[spoiled]).any()
    assert _lib.device_status() == 0


def filled(k, v, page, dtype, width=None):
    """A pool that holds the rows k, v [n, hk, D] (fp32) of one sequence in
    pages of descending number: the pool, its table and what it holds."""
    n, hk, d = k.shape
    count = -(-n // page)
    width = count if width is None else width
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, :count] = torch.arange(count, 0, -1, dtype=torch.int32, device="cuda")
    stored, held = [], []
    for x in (k, v):
        codes, scale = quantise(x, dtype)
        held.append(values(codes, scale))
        for part in (codes, scale):
            if part is None:
                stored.append(None)
                continue
            raw = part.view(torch.uint8) if dtype == torch.float8_e4m3fn and part is codes else part
            rows = torch.zeros(count * page, *raw.shape[1:], dtype=raw.dtype, device="cuda")
            rows[:n] = raw
            pages = rows.view(count, page, *raw.shape[1:]).transpose(1, 2)
            pool = torch.zeros(count + 1, *pages.shape[1:], dtype=raw.dtype, device="cuda")
            pool[1:] = pages.flip(0)
            stored.append(pool.view(part.dtype))
    return KVPages(stored[0], stored[2], stored[1], stored[3]), table, held


# ------------------------------------------------------------- large values
# Scores of 0 for the first 128 keys and of `jump` (in log2) past them, so a
# weight taken relative to the first block's maximum is up to 2^jump.  The
# weighted sums of normalised weights stay below 2^104.
JUMPS = [(2.0**80, 43.0), (2.0**100, 15.0), (2.0**100, 30.0), (2.0**90, 60.0)]


@pytest.mark.parametrize("n,d", [(300, 64), (300, 128), (2100, 128)])
@pytest.mark.parametrize("big,jump", JUMPS)
def test_large_values_under_scores_that_grow(n, d, big, jump):
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.ones(n, 2, d, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(n, 1, d, device="cuda", dtype=torch.bfloat16)
    k[128:, :, 0] = jump
    v = (torch.rand(n, 1, d, generator=g, device="cuda") * big).to(torch.bfloat16)
    scale = 0.6931471805599453            # a score of 1 is a factor of 2
    compare(ops.prompt_attention(q, k, v, starts_of([n]), scale=scale), q, k, v, scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("new,total", [(1, 300), (90, 400), (200, 3000)])
@pytest.mark.parametrize("big,jump", JUMPS)
def test_large_values_in_the_cache_under_scores_that_grow(dtype, new, total, big, jump):
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.ones(new, 2, 128, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(total, 1, 128, device="cuda")
    k[128:, :, 0] = jump
    v = torch.rand(total, 1, 128, generator=g, device="cuda") * big
    pages, table, (hk, hv) = filled(k, v, 64, dtype)
    scale = 0.6931471805599453
    out = ops.cache_attention(q, pages, Sequences(starts_of([new]), ints([total]), table), scale=scale)
    compare(out, q, hk, hv, scale)


# ------------------------------------------- rows that see nothing, hidden infinities
@pytest.mark.parametrize("heads", [(16, 8, 128), (4, 4, 64), (9, 3, 64)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize(
    "new,total,bad,width",
    [(40, 20, 10, None), (40, 20, 19, None), (150, 100, 3, None), (900, 30, 7, None), (60, 33, 5, 200)],
)
def test_rows_before_the_first_token_beside_a_hidden_infinity(heads, new, total, bad, width):
    """More new rows than tokens: the first rows see nothing and give zeros,
    and what is hidden from them leaves no status."""
    hq, hk, d = heads
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(total, hk, d, generator=g, device="cuda") for _ in range(2))
    v[bad, :, 3] = float("inf")
    q = torch.randn(new, hq, d, generator=g, device="cuda").to(torch.bfloat16)
    pages, table, (kk, vv) = filled(k, v, 16, torch.bfloat16, width)
    out = ops.cache_attention(q, pages, Sequences(starts_of([new]), ints([total]), table))
    compare(out, q, kk, vv, d**-0.5)


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 6, 90])
@pytest.mark.parametrize("tiny", [2.0**-121, 2.0**-100, 2.0**100])
def test_keys_and_queries_of_opposite_magnitudes(dtype, new, tiny):
    """Scores of ordinary size from queries and keys near the ends of bf16's
    range."""
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn(100, 1, 128, generator=g, device="cuda") for _ in range(2))
    q = (torch.randn(new, 2, 128, generator=g, device="cuda") * tiny).to(torch.bfloat16)
    pages, table, (hk, hv) = filled(k / tiny, v, 32, dtype)
    out = ops.cache_attention(q, pages, Sequences(starts_of([new]), ints([100]), table))
    compare(out, q, hk, hv, 128**-0.5)
