"""The 4-bit K/V cache: rows written and read back (bitwise) and attention of
new tokens over its pages against fp64."""

import pytest
import torch

from pir2_b200 import _lib, ops
from pir2_b200.kv_cache import KVPages, Sequences
from int4_reference import make_pool4, quantise4, values4
from ragged_reference import attend, starts_of, tolerance

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def new_rows(rows, hk, d, seed, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, 2 * hk + 1, d, generator=g, device="cuda")
    x *= torch.exp(spread * torch.randn(rows, 1, 1, generator=g, device="cuda"))
    x = x.to(torch.bfloat16)
    return x[:, 1 : hk + 1], x[:, hk + 1 :]


def queries(rows, hq, d, seed):
    q, _ = new_rows(rows, hq, d, seed)
    return q.div_(q.float().abs().amax(-1, keepdim=True)).mul_(3)


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


@pytest.mark.parametrize("hk,d,page", [(8, 128, 64), (1, 64, 16), (3, 128, 32), (5, 64, 128), (40, 128, 16)])
@pytest.mark.parametrize("new,past", [([1], [0]), ([1, 1, 1], [15, 16, 127]), ([0, 37, 200, 1], [5, 0, 60, 300])])
def test_write_and_read_back_bitwise(hk, d, page, new, past):
    total = [n + p for n, p in zip(new, past)]
    pool, table, rows = make_pool4(total, hk, d, page, seed=sum(total), poison=False)
    before = [t.clone() for t in pool]
    k, v = new_rows(sum(new), hk, d, seed=9)
    k[0, 0] = 0                                # a row of zeros: scale 1, factors 0
    v[0, 0, 32:] = 0                           # and groups of zeros
    k[-1, -1, 3:] *= 2.0**-14                  # groups whose factors are small or 0
    starts = starts_of(new)
    pages = KVPages(*pool)
    ops.cache_write(k, v, pages, Sequences(starts, ints(total), table))
    back_k, back_v = ops.cache_read(pages, Sequences(starts_of(total), ints(total), table), sum(total))
    assert _lib.device_status() == 0
    for which, x, back in ((0, k, back_k), (1, v, back_v)):
        codes, scale, factor = quantise4(x)
        at, expected = 0, []
        for b, (n, t) in enumerate(zip(new, total)):
            for i in range(n):
                p = t - n + i
                slot = int(table[b, p // page]), slice(None), p % page
                before[which][slot] = codes[at + i]
                before[2 + which][slot] = scale[at + i]
                before[4 + which].view(torch.uint8)[slot] = factor.view(torch.uint8)[at + i]
            at += n
            expected += [rows[b][which][: t - n], values4(codes[at - n : at], scale[at - n : at], factor[at - n : at])]
        assert torch.equal(pool[which], before[which])
        assert torch.equal(pool[2 + which], before[2 + which])
        assert torch.equal(pool[4 + which].view(torch.uint8), before[4 + which].view(torch.uint8))
        assert torch.equal(back, torch.cat(expected).to(torch.bfloat16))


def test_write_of_every_magnitude():
    """Rows from bf16's smallest numbers to its largest, and borders of codes."""
    rows = 254
    x = (torch.arange(128, device="cuda").float() + 128)[None, :] * torch.ones(rows, 1, device="cuda")
    x = x * torch.where(torch.arange(128, device="cuda") % 3 == 0, -1.0, 1.0)
    x = torch.ldexp(x.double(), (torch.arange(rows, device="cuda") - 133)[:, None]).to(torch.bfloat16)[:, None].contiguous()
    assert torch.isfinite(x).all() and x[0].abs().max() > 0
    x[::2, :, 64:] /= 37                       # other factors
    pool, table, _ = make_pool4([rows], 1, 128, 64, seed=1, poison=False)
    ops.cache_write(x, -x, KVPages(*pool), Sequences(starts_of([rows]), ints([rows]), table))
    ids, p = table[0].long()[torch.arange(rows, device="cuda") // 64], torch.arange(rows, device="cuda") % 64
    for which, y in ((0, x), (1, -x)):
        codes, scale, factor = quantise4(y)
        assert torch.equal(pool[2 + which][ids, :, p], scale)
        assert torch.equal(pool[4 + which].view(torch.uint8)[ids, :, p], factor.view(torch.uint8))
        assert torch.equal(pool[which][ids, :, p], codes)


def test_write_of_values_that_are_not_finite():
    pool, table, _ = make_pool4([4], 2, 128, 16, seed=3, poison=False)
    k, v = (x.clone() for x in new_rows(4, 2, 128, seed=4))
    k[0, 0, 3], k[1, 1, 7], v[2, 0, 9], v[3], k[3, 1, 5], k[3, 1, 6] = (
        float("nan"), float("inf"), -float("inf"), float("inf"), float("nan"), float("inf"))
    pages = KVPages(*pool)
    ops.cache_write(k, v, pages, Sequences(starts_of([4]), ints([4]), table))
    page = int(table[0, 0])
    for which, x in ((0, k), (1, v)):
        codes, scale, factor = quantise4(x)
        assert torch.equal(pool[which][page, :, :4].transpose(0, 1), codes)
        assert torch.equal(pool[4 + which].view(torch.uint8)[page, :, :4].transpose(0, 1), factor.view(torch.uint8))
        assert torch.equal(torch.nan_to_num(pool[2 + which][page, :, :4].T, nan=-1.0), torch.nan_to_num(scale, nan=-1.0))
        assert torch.isnan(scale).sum() == (2 if x is k else 0)
    # A reader of a row with a NaN sees it, the others do not.
    q = queries(1, 4, 128, seed=4)
    for length, spoiled in ((1, [True, False]), (4, [True, True])):
        out = ops.cache_attention(q, pages, Sequences(starts_of([1]), ints([length]), table)).view(2, 2, 128)
        for h in range(2):
            assert torch.isnan(out[h]).all() if spoiled[h] else torch.isfinite(out[h]).all()


def test_pools_of_all_layers_in_one_allocation():
    """Pages of one layer lie apart; a large stride puts them past 2^31 bytes."""
    pages, hk, size, d = 6, 2, 64, 128
    apart = 450_000_000 // 16 * 16
    total = [300, 40]
    shape, strides = (pages, hk, size, d // 2), (apart, size * d // 2, d // 2, 1)
    store = torch.zeros(2 * hk * size * d + 5 * apart, device="cuda", dtype=torch.uint8)
    k, v = store.as_strided(shape, strides), store.as_strided(shape, strides, hk * size * d // 2)
    scales = [torch.ones(pages, 3, hk, size, device="cuda")[:, i] for i in (0, 2)]
    factors = [torch.zeros(pages, 3, hk, size, d // 32, device="cuda").to(torch.float8_e4m3fn)[:, i] for i in (0, 2)]
    cache = KVPages(k, v, *scales, *factors)
    table = ints([[5, 0, 4, 1, 3], [2, -1, -1, -1, -1]])
    xk, xv = new_rows(sum(total), hk, d, seed=5, spread=0.5)
    ops.cache_write(xk, xv, cache, Sequences(starts_of(total), ints(total), table))
    back = ops.cache_read(cache, Sequences(starts_of(total), ints(total), table), sum(total))
    held = [values4(*quantise4(x)) for x in (xk, xv)]
    for want, got in zip(held, back):
        assert torch.equal(got, want.to(torch.bfloat16))
    q = queries(5, 4, d, seed=6)
    out = ops.cache_attention(q, cache, Sequences(starts_of([3, 2]), ints(total), table))
    check(out, q, [(held[0][:300], held[1][:300]), (held[0][300:], held[1][300:])], [3, 2], total)


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


@pytest.mark.parametrize("heads", [(16, 8, 128), (8, 1, 128), (6, 2, 64), (4, 4, 64), (24, 1, 128)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("new,total", CHUNKS, ids=lambda x: "-".join(map(str, x)))
def test_attention_over_pages(heads, new, total):
    hq, hk, d = heads
    for page in (16, 128) if len(new) > 2 else (32, 64):
        pool, table, rows = make_pool4(total, hk, d, page, seed=hq + page)
        q = queries(sum(new), hq, d, seed=page)
        out = ops.cache_attention(q, KVPages(*pool), Sequences(starts_of(new), ints(total), table))
        assert out.shape == (sum(new), hq * d)
        check(out, q, rows, new, total)


@pytest.mark.parametrize("new", [1, 6, 40, 300])
def test_attention_over_a_long_cache(new):
    total = [9001, 20011]
    pool, table, rows = make_pool4(total, 2, 128, 64, seed=11)
    q = queries(2 * new, 4, 128, seed=12)
    sequences = Sequences(starts_of([new, new]), ints(total), table)
    out = ops.cache_attention(q, KVPages(*pool), sequences)
    check(out, q, rows, [new, new], total)
    assert torch.equal(out, ops.cache_attention(q, KVPages(*pool), sequences))


@pytest.mark.parametrize("heads", [(2, 1, 128), (9, 3, 64)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("new", [[1, 1, 0, 1, 1], [1, 2, 0, 3, 4]], ids=["one", "few"])
def test_few_sequences_one_of_them_long(heads, new):
    hq, hk, d = heads
    total = [29990, 0, 5, 300, 4003]
    pool, table, rows = make_pool4(total, hk, d, 32, seed=hq)
    q = queries(sum(new), hq, d, seed=31)
    sequences = Sequences(starts_of(new), ints(total), table)
    out = ops.cache_attention(q, KVPages(*pool), sequences)
    check(out, q, rows, new, total)
    assert torch.equal(out, ops.cache_attention(q, KVPages(*pool), sequences))


@pytest.mark.parametrize("batch", [41, 128, 129])
@pytest.mark.parametrize("new", [1, 37, 70])
def test_many_sequences_of_uneven_lengths(batch, new):
    fresh = [0 if b % 11 == 5 else 1 + (b * 7) % new if new > 1 else 1 for b in range(batch)]
    fresh[2] = 3 * new
    total = [(n * 5 + b * 17) % 90 for b, n in enumerate(fresh)]
    total[1], total[batch // 2], total[batch - 1] = 1500, 1101, 700
    pool, table, rows = make_pool4(total, 16, 64, 64, seed=batch)
    q = queries(sum(fresh), 16, 64, seed=new)
    out = ops.cache_attention(q, KVPages(*pool), Sequences(starts_of(fresh), ints(total), table))
    check(out, q, rows, fresh, total)


@pytest.mark.parametrize("new", [1, 50])
def test_large_and_small_values_and_queries(new):
    """Scales over 2^-60 to 2^60, factors to the largest E4M3 number."""
    total, hk, d = [300], 2, 128
    pool, table, _ = make_pool4(total, hk, d, 64, seed=21)
    for which, power in ((0, 40), (1, 60)):
        pool[4 + which].view(torch.uint8)[:, :, ::3] = 0x7E        # 448
        pool[2 + which][:] = 2.0**power if which else 2.0**-power
    rows = [values4(pool[w], pool[2 + w], pool[4 + w])[table[0].long()].permute(0, 2, 1, 3).reshape(-1, hk, d)[:300] for w in (0, 1)]
    q = (queries(new, 4, d, seed=5).float() * 2.0**32).to(torch.bfloat16)
    out = ops.cache_attention(q, KVPages(*pool), Sequences(starts_of([new]), ints(total), table))
    check(out, q, [tuple(rows)], [new], total)


def test_replayed_graph_another_stream_and_strided_rows():
    new, total = [1, 2], [70, 333]
    pool, table, rows = make_pool4(total, 2, 128, 16, seed=8)
    pages = KVPages(*pool)
    lengths, starts = ints([60, 300]), starts_of(new)
    sequences = Sequences(starts, lengths, table)
    wide = queries(3, 11, 128, seed=9)
    q = wide[:, 2:10]
    store = torch.full((3, 1104), 5.0, device="cuda", dtype=torch.bfloat16)
    out = store[:, 40:1064]
    ops.cache_attention(q, pages, sequences, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_attention(q, pages, sequences, out=out)
    lengths.copy_(ints(total))
    out.fill_(7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    side.synchronize()
    check(out, q, rows, new, total)
    assert (store[:, :40] == 5).all() and (store[:, 1064:] == 5).all()


def test_bad_pages_are_reported():
    pool, table, _ = make_pool4([40], 1, 64, 16, seed=2)
    table[0, 1] = 99
    k, v = new_rows(40, 1, 64, seed=1)
    pages, sequences = KVPages(*pool), Sequences(starts_of([40]), ints([40]), table)
    ops.cache_write(k, v, pages, sequences)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    back, _ = ops.cache_read(pages, sequences, 40)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE
    assert (back[16:32] == 0).all()
    ops.cache_attention(queries(40, 1, 64, seed=3), pages, sequences)
    assert _lib.device_status() == _lib.STATUS_BAD_PAGE


def test_pools_that_the_handle_refuses():
    def make(**changes):
        fields = dict(k=torch.uint8, v=torch.uint8, factor=torch.float8_e4m3fn, shape=(2, 1, 16, 32), groups=2, with_factor=True)
        fields.update(changes)
        code = [torch.zeros(fields["shape"], dtype=fields[x], device="cuda") for x in "kv"]
        scale = [torch.ones(2, 1, 16, device="cuda") for _ in "kv"]
        factor = [torch.zeros(2, 1, 16, fields["groups"], device="cuda").to(fields["factor"]) for _ in "kv"]
        return KVPages(*code, *scale, *(factor if fields["with_factor"] else ()))

    assert make().head_dim == 64 and make(shape=(2, 1, 16, 64), groups=4).head_dim == 128
    for changes in ({"v": torch.int8}, {"factor": torch.float32}, {"shape": (2, 1, 16, 48)}, {"groups": 4}, {"with_factor": False},
                    {"k": torch.int8, "v": torch.int8, "shape": (2, 1, 16, 64)}):
        with pytest.raises(ValueError, match="KVPages"):
            make(**changes)
