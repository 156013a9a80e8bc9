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


# ------------------------------------------------ hidden values that are not finite
# Row i of the last new rows sees `bad` or does not; (new, total, table width in
# pages of 16): few rows of one and of two groups of 8, in one CTA, a cluster and
# pieces; one tile, two tiles, and both with the keys split.
HIDDEN = [
    (3, 40, None),
    (7, 40, None),
    (4, 1500, None),
    (7, 9001, None),
    (8, 30000, None),
    (40, 90, None),
    (40, 3001, None),
    (200, 411, None),
    (200, 5003, None),
    (300, 1000, 4000),
]


@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("heads", [(4, 2, 128), (4, 2, 64), (3, 1, 128)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("new,total,width", HIDDEN)
def test_values_hidden_from_some_rows_of_a_cache(new, total, width, heads, what):
    """A value or key in the cache that is not finite spoils the rows that see
    it, a value only in its own column, and no others."""
    hq, hk, d = heads
    g = torch.Generator(device="cuda").manual_seed(total)
    q = torch.randn(new, hq, d, generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.randn(total, hk, d, generator=g, device="cuda") for _ in range(2))
    first = total - new
    for back in sorted({1, 2, new // 2, new - 1}):        # hidden from the first rows, seen by `back` of them
        spoiled = v.clone()
        spoiled[total - back, hk - 1, 5] = what
        pages, table, (kk, vv) = filled(k, spoiled, 16, torch.bfloat16, width)
        sequences = Sequences(starts_of([new]), ints([total]), table)
        out = ops.cache_attention(q, pages, sequences)
        compare(out, q, kk, vv, d**-0.5)
        hit = ~torch.isfinite(out.view(new, hq, d))
        seen = torch.arange(first, total, device="cuda") >= total - back
        want = torch.zeros_like(hit)
        want[:, hq - hq // hk :, 5] = seen[:, None]
        assert torch.equal(hit, want)
    # A key: every row that sees it, whole, in the heads that read it.
    spoiled = k.clone()
    spoiled[total - 2, hk - 1, 5] = what
    pages, table, (kk, vv) = filled(spoiled, v, 16, torch.bfloat16, width)
    out = ops.cache_attention(q, pages, Sequences(starts_of([new]), ints([total]), table)).view(new, hq, d)
    other = hq - hq // hk
    finite = torch.isfinite(out)
    assert finite[: new - 2].all() and finite[:, :other].all()
    if what != what:
        assert not finite[new - 2 :, other:].any()
    compare(out[: new - 2], q[: new - 2], k[: total - 2].to(torch.bfloat16), v[: total - 2].to(torch.bfloat16), d**-0.5)


@pytest.mark.parametrize("n", [420, 2300])
@pytest.mark.parametrize("heads", [(4, 2, 128), (4, 2, 64), (6, 2, 64)], ids=lambda h: "x".join(map(str, h)))
def test_a_key_that_is_nan_spoils_the_rows_that_see_it(n, heads):
    hq, hk, d = heads
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(n, h, d, generator=g, device="cuda").to(torch.bfloat16) for h in (hq, hk, hk))
    k[n // 2, 1] = float("nan")
    out = ops.prompt_attention(q, k, v, starts_of([n])).view(n, hq, d)
    finite = torch.isfinite(out)
    assert finite[: n // 2].all() and finite[:, : hq // hk].all() and not finite[n // 2 :, hq // hk :].any()
    compare(out[: n // 2], q[: n // 2], k[: n // 2], v[: n // 2], d**-0.5)


# ------------------------------------------------------------- heads and lengths
@pytest.mark.parametrize("heads", [(64, 1, 64), (128, 1, 128), (128, 2, 64), (160, 1, 64), (256, 1, 128)],
                         ids=lambda h: "x".join(map(str, h)))
def test_many_heads_for_one_key_head(heads):
    """Groups of 64 to 256: a query tile is one box of two tokens, of one, or
    gathered, and its rows leave one by one."""
    hq, hk, d = heads
    g = torch.Generator(device="cuda").manual_seed(6)
    lengths = [1, 37, 0, 150]
    rows = sum(lengths)
    q = torch.randn(rows, hq, d, generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.randn(rows, hk, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    out = ops.prompt_attention(q, k, v, starts_of(lengths))
    at = 0
    for n in lengths:
        mine = slice(at, at + n)
        if n:
            compare(out[mine], q[mine], k[mine], v[mine], d**-0.5)
        at += n
    for dtype in DTYPES:
        pages, table, (kk, vv) = filled(k.float(), v.float(), 32, dtype)
        for new in (1, 9):
            out = ops.cache_attention(q[:new], pages, Sequences(starts_of([new]), ints([rows]), table))
            compare(out, q[:new], kk, vv, d**-0.5)


@pytest.mark.parametrize("lengths", [[2048], [2500], [2050, 2047], [4099]], ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("heads", [(2, 1, 64), (3, 1, 64), (6, 2, 128)], ids=lambda h: "x".join(map(str, h)))
def test_long_prompts_of_narrow_and_odd_heads(lengths, heads):
    hq, hk, d = heads
    g = torch.Generator(device="cuda").manual_seed(7)
    rows = sum(lengths)
    q, k, v = (torch.randn(rows, h, d, generator=g, device="cuda").to(torch.bfloat16) for h in (hq, hk, hk))
    out = ops.prompt_attention(q, k, v, starts_of(lengths))
    at = 0
    for n in lengths:
        mine = slice(at, at + n)
        compare(out[mine], q[mine], k[mine], v[mine], d**-0.5)
        at += n


@pytest.mark.parametrize("what", ["heads", "rows", "all"])
def test_broadcast_keys_and_values(what):
    """Strides of 0: one key head for all, or one row for all."""
    g = torch.Generator(device="cuda").manual_seed(8)
    q = torch.randn(200, 4, 128, generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.randn(200, 2, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    if what in ("heads", "all"):
        k, v = (x[:, :1].expand(200, 2, 128) for x in (k, v))
    if what in ("rows", "all"):
        k, v = (x[:1].expand(200, 2, 128) for x in (k, v))
    compare(ops.prompt_attention(q, k, v, starts_of([200])), q, k, v, 128**-0.5)


@pytest.mark.parametrize("batch,new,group,pieces", [(8, 8, 2, True), (9, 8, 2, True), (10, 8, 2, False), (18, 4, 2, True),
                                                    (9, 2, 8, True), (10, 2, 8, False), (18, 1, 4, True), (19, 1, 4, False)])
def test_units_of_rows_are_counted_whole(batch, new, group, pieces):
    """A call is cut into pieces (which need a workspace) where its units of 8
    or 16 rows have four places or more each on 148 SMs of two (four, 8-row)
    int8 CTAs: 8 kv heads of `batch` sequences, each one unit."""
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("counted for 148 SMs")
    pages = KVPages.allocate(2, 8, 128, page_size=128, dtype=torch.int8)
    table = torch.zeros(batch, 200, dtype=torch.int32, device="cuda")
    sequences = Sequences(starts_of([new] * batch), ints([200] * batch), table)
    size = _lib.lib().pir2b_cache_attention_workspace(batch * new, 8 * group, pages.address, sequences.address)
    assert (size > 0) == pieces


def test_one_prompt_of_8200_in_two_tiles():
    g = torch.Generator(device="cuda").manual_seed(9)
    q, k, v = (torch.randn(8200, h, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (2, 1, 1))
    k[5000, 0, 3] = 40.0                  # the reference moves
    compare(ops.prompt_attention(q, k, v, starts_of([8200])), q, k, v, 128**-0.5)
    v[8190, 0, 7] = float("inf")          # hidden from the last tile's first rows
    compare(ops.prompt_attention(q, k, v, starts_of([8200])), q, k, v, 128**-0.5)
