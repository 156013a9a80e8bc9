"""Causal grouped-query attention over packed prompts, against fp64."""

import pytest
import torch

from pir2_b200 import _lib, ops
from ragged_reference import attend, starts_of, tolerance

pytestmark = pytest.mark.gpu


def merged(rows, hq, hk, d, seed, gain=1.0):
    """q, k, v as views of merged projection rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, hq + 2 * hk, d, generator=g, device="cuda")
    x[:, :hq] *= gain
    x = x.to(torch.bfloat16)
    return x[:, :hq], x[:, hq : hq + hk], x[:, hq + hk :]


def check(out, q, k, v, lengths, first=0, scale=None):
    hq, d = q.shape[1], q.shape[2]
    scale = d**-0.5 if scale is None else scale
    at = first
    for n in lengths:
        mine = slice(at, at + n)
        want, mass, spoiled = attend(q[mine], k[mine], v[mine], scale)
        got = out[mine].view(n, hq, d).double()
        far = ((got - want).abs() > tolerance(want, mass)) | ~torch.isfinite(got)
        assert not (far & ~spoiled).any(), f"{int((far & ~spoiled).sum())} values of a prompt of {n} rows"
        assert not torch.isfinite(got[spoiled]).any()
        at += n
    assert _lib.device_status() == 0


LENGTHS = [[1], [2, 1, 0, 3], [0, 127, 128, 129], [64, 65, 0, 200, 1], [544], [300, 17, 513, 0], [1025]]
HEADS = [(16, 8, 128), (4, 4, 64), (6, 2, 64), (8, 1, 128), (3, 1, 128), (5, 5, 64)]


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
def test_prompts_of_different_lengths(lengths, heads):
    hq, hk, d = heads
    q, k, v = merged(sum(lengths), hq, hk, d, seed=len(lengths) + hq)
    out = ops.prompt_attention(q, k, v, starts_of(lengths))
    assert out.shape == (sum(lengths), hq * d) and out.dtype == torch.bfloat16
    check(out, q, k, v, lengths)


def test_long_prompt_and_many_short_ones():
    q, k, v = merged(5001, 2, 1, 128, seed=1)
    check(ops.prompt_attention(q, k, v, starts_of([5001])), q, k, v, [5001])
    lengths = [(7 * i) % 23 for i in range(300)]
    q, k, v = merged(sum(lengths), 4, 2, 64, seed=2)
    check(ops.prompt_attention(q, k, v, starts_of(lengths)), q, k, v, lengths)


@pytest.mark.parametrize("d", [64, 128])
def test_heads_first_storage_and_strided_output(d):
    lengths = [70, 200]
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (
        torch.randn(h, 270, d, generator=g, device="cuda").to(torch.bfloat16).transpose(0, 1) for h in (4, 2, 2)
    )
    rows = torch.full((270, 4 * d + 24), 7.0, device="cuda", dtype=torch.bfloat16)
    out = ops.prompt_attention(q, k, v, starts_of(lengths), out=rows[:, 8 : 8 + 4 * d])
    check(out, q, k, v, lengths)
    assert (rows[:, :8] == 7).all() and (rows[:, 8 + 4 * d :] == 7).all()


def test_scale_and_sharp_scores():
    """Scores of thousands: the largest takes all the weight."""
    lengths = [190, 333]
    q, k, v = merged(523, 4, 2, 128, seed=4, gain=300.0)
    check(ops.prompt_attention(q, k, v, starts_of(lengths), scale=0.25), q, k, v, lengths, scale=0.25)
    # Scores that grow along the keys: the running maximum moves in every tile.
    k = k.clone()
    k.copy_(q[:, ::2] * 0 + torch.arange(523, device="cuda")[:, None, None] * 0.01)
    q = q * 0 + 1
    check(ops.prompt_attention(q, k, v, starts_of(lengths), scale=0.5), q, k, v, lengths, scale=0.5)


def test_rows_of_no_prompt_are_left_alone():
    q, k, v = merged(300, 4, 2, 128, seed=5)
    out = torch.full((300, 512), 3.0, device="cuda", dtype=torch.bfloat16)
    ops.prompt_attention(q, k, v, starts_of([100, 140], first=20), out=out)
    check(out, q, k, v, [100, 140], first=20)
    assert (out[:20] == 3).all() and (out[260:] == 3).all()


@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["k", "v"])
def test_hidden_rows_do_not_reach_others(what, where):
    """A value that is not finite spoils the rows that see it, in its column
    (v) or whole (k), and no others: not earlier rows of its prompt, not the
    neighbouring prompts."""
    lengths = [130, 150, 140]
    q, k, v = (x.clone() for x in merged(420, 4, 2, 128, seed=6))
    if where == "v":
        v[210, 1, 5] = what
    else:
        k[210, 1] = what
    out = ops.prompt_attention(q, k, v, starts_of(lengths))
    got = out.view(420, 4, 128)
    for rows, seen in ((slice(0, 210), False), (slice(210, 280), True), (slice(280, 420), False)):
        hit = ~torch.isfinite(got[rows])
        if not seen:
            assert not hit.any()
        elif where == "v":
            assert hit[:, 2:, 5].all() and not hit[:, 2:, :5].any() and not hit[:, 2:, 6:].any() and not hit[:, :2].any()
    fine = q.clone(), k.clone(), v.clone()
    fine[1][210, 1], fine[2][210, 1, 5] = 0, 0
    calm = ops.prompt_attention(*fine, starts_of(lengths)).view(420, 4, 128)
    assert torch.equal(got[:210], calm[:210]) and torch.equal(got[280:], calm[280:])


def test_repeatable_on_another_stream_and_in_a_graph():
    lengths = [544, 13, 700]
    q, k, v = merged(sum(lengths), 16, 8, 128, seed=7)
    starts = starts_of(lengths)
    first = ops.prompt_attention(q, k, v, starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = ops.prompt_attention(q, k, v, starts)
    side.synchronize()
    assert torch.equal(first, second)
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(q, k, v, starts, out=out)
    # New lengths and values in the same buffers.
    lengths = [200, 900, 157]
    starts.copy_(starts_of(lengths))
    q.copy_(torch.randn(q.shape, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    check(out, q, k, v, lengths)


def test_refusals():
    q, k, v = merged(16, 4, 2, 128, seed=8)
    starts = starts_of([16])
    cases = [
        ((q.float(), k, v, starts), "bf16"),
        ((q, k[:8], v, starts), "must be"),
        ((q, k, v[..., :64], starts), "must be"),
        ((q[:, :3], k, v, starts), "multiple of hk"),
        ((q[..., :32], k[..., :32], v[..., :32], starts), "head_dim 64 or 128"),
        ((q, k, v, starts.long()), "int32"),
        ((q, k, v, starts[:1]), "int32"),
        ((q.cpu(), k, v, starts), "CUDA"),
        ((q, k, v, starts.cpu()), "one device"),
    ]
    for args, match in cases:
        with pytest.raises(ValueError, match=match):
            ops.prompt_attention(*args)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            ops.prompt_attention(q, k, v, starts, scale=scale)
    odd = torch.zeros(16 * 8 * 128 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(16, 8, 128)
    with pytest.raises(ValueError, match="aligned"):
        ops.prompt_attention(odd[:, :4], k, v, starts)
    with pytest.raises(ValueError, match="out must be"):
        ops.prompt_attention(q, k, v, starts, out=torch.empty(16, 100, device="cuda", dtype=torch.bfloat16))
    assert ops.prompt_attention(q[:0], k[:0], v[:0], starts_of([0])).shape == (0, 512)
