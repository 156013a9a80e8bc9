"""The paged K/V cache: quantised rows written and read back (bitwise), and
attention of new tokens over the pages against fp64."""

import pytest
import torch

from pir2_b200 import _lib, ops
from pir2_b200.kv_cache import KVPages, Sequences
from ragged_reference import attend, make_pool, quantise, starts_of, tolerance, values

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.int8, torch.float8_e4m3fn]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def bits(x):
    return x.contiguous().view(torch.uint8)


def new_rows(rows, hk, d, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, 2 * hk + 1, d, generator=g, device="cuda")
    x *= torch.exp(2 * torch.randn(rows, 1, 1, generator=g, device="cuda"))
    x = x.to(torch.bfloat16)
    return x[:, 1 : hk + 1], x[:, hk + 1 :]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("hk,d,page", [(8, 128, 64), (1, 64, 16), (3, 128, 32), (5, 64, 128)])
@pytest.mark.parametrize("new,past", [([1], [0]), ([1, 1, 1], [15, 16, 127]), ([0, 37, 200, 1], [5, 0, 60, 300])])
def test_write_and_read_back_bitwise(dtype, hk, d, page, new, past):
    total = [n + p for n, p in zip(new, past)]
    kc, vc, ks, vs, table, rows = make_pool(total, hk, d, page, dtype, seed=sum(total), poison=False)
    pages = KVPages(kc, vc, ks, vs)
    before = [None if t is None else t.clone() for t in (kc, vc, ks, vs)]
    k, v = new_rows(sum(new), hk, d, seed=9)
    k[0, 0] = 0                       # a row of zeros: scale 1
    starts = starts_of(new)
    ops.cache_write(k, v, pages, Sequences(starts, ints(total), table))
    back_k, back_v = ops.cache_read(pages, Sequences(starts_of(total), ints(total), table), sum(total))
    assert _lib.device_status() == 0
    # The pool as it has to be: the quantised rows in their slots, all else as before.
    for which, x, want_codes, want_scale, back in ((0, k, before[0], before[2], back_k), (1, v, before[1], before[3], back_v)):
        codes, scale = quantise(x, dtype)
        flat = want_codes.view(torch.uint8 if dtype != torch.bfloat16 else dtype)
        at = 0
        expected = []
        for b, (n, t) in enumerate(zip(new, total)):
            for i in range(n):
                p = t - n + i
                slot = int(table[b, p // page]), slice(None), p % page
                flat[slot] = codes[at + i].view(flat.dtype)
                if scale is not None:
                    want_scale[slot] = scale[at + i]
            at += n
            old = rows[b][which][: t - n]
            new_values = values(codes[at - n : at], None if scale is None else scale[at - n : at])
            expected.append(torch.cat([old, new_values]))
        got = (kc, vc)[which]
        assert torch.equal(bits(got), bits(want_codes))
        if scale is not None:
            assert torch.equal((ks, vs)[which], want_scale)
        assert torch.equal(back, torch.cat(expected).to(torch.bfloat16))


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=["int8", "e4m3"])
def test_write_of_values_that_are_not_finite(dtype):
    kc, vc, ks, vs, table, _ = make_pool([4], 2, 128, 16, dtype, seed=3, poison=False)
    k, v = (x.clone() for x in new_rows(4, 2, 128, seed=4))
    k[0, 0, 3], k[1, 1, 7], v[2, 0, 9], v[3] = float("nan"), float("inf"), -float("inf"), float("inf")
    ops.cache_write(k, v, KVPages(kc, vc, ks, vs), Sequences(starts_of([4]), ints([4]), table))
    page = int(table[0, 0])
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        codes, scale = quantise(x, dtype)
        assert torch.equal(torch.nan_to_num(s[page, :, :4].T, nan=-1.0), torch.nan_to_num(scale, nan=-1.0))
        assert torch.isnan(scale).sum() == (1 if x is k else 0)
        assert torch.equal(c[page, :, :4].transpose(0, 1).float(), codes.float())
    # A reader of the row with the NaN sees it, the others do not.
    q, _ = new_rows(1, 4, 128, seed=4)
    for length, spoiled in ((1, True), (4, True)):
        out = ops.cache_attention(q, KVPages(kc, vc, ks, vs), Sequences(starts_of([1]), ints([length]), table)).view(4, 128)
        assert torch.isnan(out[:2]).all() == spoiled and torch.isfinite(out[2:]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "int8", "e4m3"])
def test_pools_of_all_layers_in_one_allocation(dtype):
    """Pages of one layer lie apart; a large stride puts them past 2^31
    elements."""
    pages, hk, size, d = 6, 2, 64, 128
    apart = 450_000_000 // 16 * 16
    total = [300, 40]
    pool = torch.zeros(2 * hk * size * d + 5 * apart, device="cuda", dtype=dtype)
    k = pool.as_strided((pages, hk, size, d), (apart, size * d, d, 1))
    v = pool.as_strided((pages, hk, size, d), (apart, size * d, d, 1), hk * size * d)
    scales = [torch.ones(pages, 3, hk, size, device="cuda")[:, i] for i in (0, 2)] if dtype != torch.bfloat16 else []
    cache = KVPages(k, v, *scales)
    table = ints([[5, 0, 4, 1, 3], [2, -1, -1, -1, -1]])
    xk, xv = new_rows(sum(total), hk, d, seed=5)
    ops.cache_write(xk, xv, cache, Sequences(starts_of(total), ints(total), table))
    back = ops.cache_read(cache, Sequences(starts_of(total), ints(total), table), sum(total))
    held = []
    for x, got in zip((xk, xv), back):
        want = values(*quantise(x, dtype))
        assert torch.equal(got, want.to(torch.bfloat16))
        held.append(want)
    q, _ = new_rows(5, 4, d, seed=6)
    out = ops.cache_attention(q, cache, Sequences(starts_of([3, 2]), ints(total), table))
    check(out, q, [(held[0][:300], held[1][:300]), (held[0][300:], held[1][300:])], [3, 2], total)


def check(out, q, rows, new, total, scale=None):
    hq, d = q.shape[1], q.shape[2]
    at = 0
    for b, (n, t) in enumerate(zip(new, total)):
        mine = slice(at, at + n)
        got = out[mine].view(n, hq, d).double()
        hidden = max(0, n - t)        # rows before the first position see nothing
        want, mass, _ = attend(q[mine][hidden:], *rows[b], d**-0.5 if scale is None else scale)
        far = ((got[hidden:] - want).abs() > tolerance(want, mass)) | ~torch.isfinite(got[hidden:])
        assert not far.any(), f"{int(far.sum())} values of sequence {b}: {n} new of {t}"
        assert (got[:hidden] == 0).all()
        at += n
    assert _lib.device_status() == 0


CHUNKS = [
    ([1], [1]),
    ([1], [578]),
    ([1, 1, 1, 1], [16, 17, 1000, 63]),
    ([1, 0, 2, 5], [128, 7, 129, 700]),
    ([17], [561]),
    ([33, 1, 64], [33, 2000, 100]),
    ([130, 0, 257], [400, 0, 257]),
    ([5, 3, 1], [2, 0, 0]),            # rows that see no key
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("heads", [(16, 8, 128), (8, 1, 128), (6, 2, 64), (4, 4, 64)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("new,total", CHUNKS, ids=lambda x: "-".join(map(str, x)))
def test_attention_over_pages(dtype, heads, new, total):
    hq, hk, d = heads
    for page in (16, 128) if len(new) > 2 else (32, 64):
        kc, vc, ks, vs, table, rows = make_pool(total, hk, d, page, dtype, seed=hq + page)
        q, _ = new_rows(sum(new), hq, d, seed=page)
        q.div_(q.float().abs().amax(-1, keepdim=True)).mul_(3)
        out = ops.cache_attention(q, KVPages(kc, vc, ks, vs), Sequences(starts_of(new), ints(total), table))
        assert out.shape == (sum(new), hq * d)
        check(out, q, rows, new, total)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 6, 40, 300])
def test_attention_over_a_long_cache(dtype, new):
    total = [9001, 20011]
    kc, vc, ks, vs, table, rows = make_pool(total, 2, 128, 64, dtype, seed=11)
    q, _ = new_rows(2 * new, 4, 128, seed=12)
    q.div_(q.float().abs().amax(-1, keepdim=True)).mul_(3)
    sequences = Sequences(starts_of([new, new]), ints(total), table)
    out = ops.cache_attention(q, KVPages(kc, vc, ks, vs), sequences)
    check(out, q, rows, [new, new], total)
    assert torch.equal(out, ops.cache_attention(q, KVPages(kc, vc, ks, vs), sequences))


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("heads", [(2, 1, 128), (9, 3, 64)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("new", [[1, 1, 0, 1, 1], [1, 2, 0, 3, 4]], ids=["one", "few"])
def test_few_sequences_one_of_them_long(dtype, heads, new):
    """Units of rows of every length from none to many pieces."""
    hq, hk, d = heads
    total = [29990, 0, 5, 300, 4003]
    kc, vc, ks, vs, table, rows = make_pool(total, hk, d, 32, dtype, seed=hq)
    q, _ = new_rows(sum(new), hq, d, seed=31)
    q.div_(q.float().abs().amax(-1, keepdim=True)).mul_(3)
    sequences = Sequences(starts_of(new), ints(total), table)
    out = ops.cache_attention(q, KVPages(kc, vc, ks, vs), sequences)
    check(out, q, rows, new, total)
    assert torch.equal(out, ops.cache_attention(q, KVPages(kc, vc, ks, vs), sequences))


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("batch", [41, 128, 129])
@pytest.mark.parametrize("new", [1, 37, 70])
def test_many_sequences_of_uneven_lengths(dtype, batch, new):
    """More units of rows than run at once: they are taken by length."""
    fresh = [0 if b % 11 == 5 else 1 + (b * 7) % new if new > 1 else 1 for b in range(batch)]
    fresh[2] = 3 * new
    total = [(n * 5 + b * 17) % 90 for b, n in enumerate(fresh)]
    total[1], total[batch // 2], total[batch - 1] = 1500, 1101, 700
    kc, vc, ks, vs, table, rows = make_pool(total, 16, 64, 64, dtype, seed=batch)
    q, _ = new_rows(sum(fresh), 16, 64, seed=new)
    q.div_(q.float().abs().amax(-1, keepdim=True)).mul_(3)
    out = ops.cache_attention(q, KVPages(kc, vc, ks, vs), Sequences(starts_of(fresh), ints(total), table))
    check(out, q, rows, fresh, total)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "int8", "e4m3"])
def test_a_batch_of_many_kinds_of_rows(dtype):
    """Single tokens and whole prompts in one call, most sequences empty."""
    new = [1, 1, 0, 200, 1, 0, 7, 1, 40, 0, 1, 1]
    total = [400, 3, 50, 200, 1300, 0, 90, 64, 41, 9, 1, 800]
    kc, vc, ks, vs, table, rows = make_pool(total, 4, 128, 16, dtype, seed=21)
    q, _ = new_rows(sum(new), 8, 128, seed=22)
    q.div_(q.float().abs().amax(-1, keepdim=True)).mul_(3)
    out = ops.cache_attention(q, KVPages(kc, vc, ks, vs), Sequences(starts_of(new), ints(total), table))
    check(out, q, rows, new, total)


def test_many_sequences_of_one_row():
    total = [1 + (37 * i) % 300 for i in range(200)]
    kc, vc, ks, vs, table, rows = make_pool(total, 2, 128, 32, torch.int8, seed=31)
    q, _ = new_rows(200, 4, 128, seed=32)
    q.div_(q.float().abs().amax(-1, keepdim=True)).mul_(3)
    out = ops.cache_attention(q, KVPages(kc, vc, ks, vs), Sequences(starts_of([1] * 200), ints(total), table))
    check(out, q, rows, [1] * 200, total)


def test_sharp_scores_and_a_table_wider_than_needed():
    total = [777]
    kc, vc, ks, vs, table, rows = make_pool(total, 2, 128, 16, torch.int8, seed=41)
    wide = torch.full((1, 2048), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    for new in (2, 90):
        q, _ = new_rows(new, 4, 128, seed=42)
        q.mul_(50)
        out = ops.cache_attention(q, KVPages(kc, vc, ks, vs), Sequences(starts_of([new]), ints(total), wide), scale=0.3)
        check(out, q, rows, [new], total, scale=0.3)


def test_bad_indices_are_skipped_and_reported():
    total = [40]
    kc, vc, ks, vs, table, _ = make_pool(total, 2, 64, 16, torch.int8, seed=51, poison=False)
    pages = KVPages(kc, vc, ks, vs)
    before = [t.clone() for t in (kc, vc, ks, vs)]
    for bad_table, bad_length in ((table * 0 + 10_000, 40), (table * 0 - 1, 40), (table, 4000)):
        sequences = Sequences(starts_of([2]), ints([bad_length]), bad_table.contiguous())
        k, v = new_rows(2, 2, 64, seed=52)
        ops.cache_write(k, v, pages, sequences)
        assert _lib.device_status() == _lib.STATUS_BAD_PAGE
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip((kc, vc, ks, vs), before))
        for rows in (2, 100):
            q, _ = new_rows(rows, 4, 64, seed=53)
            ops.cache_attention(q, pages, Sequences(starts_of([rows]), ints([bad_length]), bad_table.contiguous()))
            assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    k, v = ops.cache_read(pages, Sequences(starts_of([40]), ints([40]), (table * 0 - 1).contiguous()), 40)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    assert (k == 0).all() and (v == 0).all()


def test_write_attend_in_a_graph_with_lengths_that_grow():
    """One captured step (write the new rows, attend) replayed while the
    sequences grow in place."""
    hq, hk, d, page = 4, 2, 128, 16
    cache = KVPages.allocate(40, hk, d, page_size=page, dtype=torch.int8)
    table = torch.randperm(40, device="cuda", dtype=torch.int32)[:30].view(2, 15).contiguous()
    lengths = ints([0, 0])
    starts = starts_of([1, 1])
    sequences = Sequences(starts, lengths, table)
    q = torch.zeros(2, hq, d, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.zeros(2, hk, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    out = torch.zeros(2, hq * d, device="cuda", dtype=torch.bfloat16)

    def step():
        lengths.add_(1)
        ops.cache_write(k, v, cache, sequences)
        ops.cache_attention(q, cache, sequences, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        lengths.zero_()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lengths.zero_()
    held = [([], []), ([], [])]
    g = torch.Generator(device="cuda").manual_seed(61)
    for i in range(40):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        graph.replay()
        for b in range(2):
            for mine, x in zip(held[b], (k, v)):
                mine.append(values(*quantise(x[b], torch.int8)))
        if i in (0, 1, 16, 39):
            rows = [tuple(torch.stack(x) for x in held[b]) for b in range(2)]
            check(out, q, rows, [1, 1], [i + 1, i + 1])


def test_refusals():
    k = torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.int8)
    s = torch.ones(4, 2, 16, device="cuda")
    for args, match in [
        ((k.float(), k.float(), s, s), "bf16, int8"),
        ((k, k[:2], s, s), "k and v"),
        ((k, k), "need k_scale"),
        ((k.bfloat16(), k.bfloat16(), s, s), "take none"),
        ((k[:, :, :8], k[:, :, :8], s[:, :, :8], s[:, :, :8]), "page_size"),
        ((k[..., :32], k[..., :32], s, s), "head_dim"),
        ((k.transpose(0, 1), k.transpose(0, 1), s.transpose(0, 1), s.transpose(0, 1)), "contiguous"),
        ((k, k, s.double(), s), "fp32"),
        ((k, k, s, s[:, :1]), "fp32"),
        ((k.cpu(), k.cpu(), s.cpu(), s.cpu()), "CUDA"),
    ]:
        with pytest.raises(ValueError, match=match):
            KVPages(*args)
    table, lengths, starts = ints([[0, 1]]), ints([20]), starts_of([3])
    for args, match in [
        ((starts.long(), lengths, table), "int32"),
        ((starts, lengths.cpu(), table), "CUDA"),
        ((starts, lengths, table[0]), "int32"),
        ((starts, ints([1, 2]), table), "entries"),
        ((starts[:1], lengths, table), "entries"),
        ((starts, lengths, table[:, :0]), "column"),
    ]:
        with pytest.raises(ValueError, match=match):
            Sequences(*args)
    pages, sequences = KVPages(k, k.clone(), s, s.clone()), Sequences(starts, lengths, table)
    rows = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="kv_heads"):
        ops.cache_write(rows[:, :1], rows[:, :1], pages, sequences)
    with pytest.raises(ValueError, match="bf16"):
        ops.cache_write(rows.float(), rows.float(), pages, sequences)
    with pytest.raises(ValueError, match="multiple of"):
        ops.cache_attention(torch.zeros(3, 3, 64, device="cuda", dtype=torch.bfloat16), pages, sequences)
    with pytest.raises(ValueError, match="scale"):
        ops.cache_attention(rows, pages, sequences, scale=0.0)
    with pytest.raises(ValueError, match="negative"):
        ops.cache_read(pages, sequences, -1)
    with pytest.raises(ValueError, match="aligned"):
        odd = torch.zeros(3 * 2 * 64 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(3, 2, 64)
        ops.cache_attention(odd, pages, sequences)
    assert ops.cache_attention(rows[:0], pages, Sequences(starts_of([0]), lengths, table)).shape == (0, 128)
    ops.cache_write(rows[:0], rows[:0], pages, Sequences(starts_of([0]), lengths, table))
