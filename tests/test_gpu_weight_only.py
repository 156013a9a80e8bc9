"""Products of a few bf16 rows with 4-bit weights in groups, against fp64."""

import pytest
import torch

from pir2_b200 import _lib, ops
from pir2_b200.weight_only import WeightOnlyLinear, quantize_groups
from int4_reference import pack, unpack

pytestmark = pytest.mark.gpu


def weights(n, k, group, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-8, 8, (n, k), generator=g, device="cuda").to(torch.int8)
    scales = (torch.rand(n, k // group, generator=g, device="cuda") + 0.1).to(torch.bfloat16)
    scales *= torch.exp2(torch.randint(-6, 7, (n, 1), generator=g, device="cuda").float()).to(torch.bfloat16)
    return pack(codes), scales


def rows(m, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(m, k, generator=g, device="cuda") * torch.exp(torch.randn(k, generator=g, device="cuda"))).to(torch.bfloat16)


def dense(packed, scales):
    group = 2 * packed.shape[1] // scales.shape[1]
    return unpack(packed).double() * scales.double().repeat_interleave(group, dim=1)


def check(out, x, packed, scales, bias=None):
    """A sum of products in fp32 adds less than 2^-15 of the sum of their
    magnitudes (a tensor-core step of 16 products loses 2^-22 of it at most, a
    warp takes less than 2^7 of them in turn); bf16's rounding is half a step."""
    w = dense(packed, scales)
    want, mass = x.double() @ w.T, x.double().abs() @ w.abs().T
    if bias is not None:
        want, mass = want + bias.double(), mass + bias.double().abs()
    far = ~((out.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-14 * mass)
    assert not far.any(), f"{int(far.sum())} values"
    assert _lib.device_status() == 0


@pytest.fixture(params=[0, 1, 2], ids=["chosen", "direct", "rows kept"])
def plan(request):
    """Both ways of running the same product."""
    previous = _lib.set_w4_mode(request.param)
    yield request.param
    _lib.set_w4_mode(previous)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 130])
@pytest.mark.parametrize("n,pieces", [(16, 1), (1, 3), (777, 9), (4096, 16), (33, 40)])
def test_products(group, m, n, pieces, plan):
    k = group * pieces
    packed, scales = weights(n, k, group, seed=n + m)
    x = rows(m, k, seed=k)
    bias = rows(1, n, seed=1)[0] if m % 2 else None
    out = ops.gemm_w4a16(x, packed, scales, bias)
    assert out.shape == (m, n)
    check(out, x, packed, scales, bias)
    assert torch.equal(out, ops.gemm_w4a16(x, packed, scales, bias))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize(
    "m,n,k", [(1, 2048, 6144), (8, 2050, 8192), (4, 20011, 2048), (32, 12288, 2048), (3, 40, 65536), (50, 1001, 8192), (12, 8001, 2304)]
)
def test_large_products(group, m, n, k, plan):
    packed, scales = weights(n, k, group, seed=2)
    x = rows(m, k, seed=3)
    check(ops.gemm_w4a16(x, packed, scales), x, packed, scales)


@pytest.mark.parametrize("m", [1, 20])
def test_every_code_and_strides(m):
    """One nonzero row element at a time gives a weight back; rows and outputs
    apart, memory between them left alone."""
    k, n, group = 128, 24, 64
    packed, scales = weights(n, k, group, seed=5)
    w = dense(packed, scales)
    wide = torch.zeros(128, k + 40, device="cuda", dtype=torch.bfloat16)
    wide[torch.arange(128), torch.arange(128) + 8] = 2.0
    store = torch.full((128, n + 3), 9.0, device="cuda", dtype=torch.bfloat16)
    for at in range(0, 128, m):
        x, out = wide[at : at + m, 8 : 8 + k], store[at : at + m, 1 : 1 + n]
        ops.gemm_w4a16(x, packed, scales, out=out)
    assert torch.equal(store[:, 1 : 1 + n], (2.0 * w.T).to(torch.bfloat16))
    assert (store[:, 0] == 9).all() and (store[:, n + 1 :] == 9).all()


@pytest.mark.parametrize("m", [6, 12])
def test_rows_that_are_not_finite_stay_alone(m, plan):
    packed, scales = weights(100, 256, 32, seed=6)
    x = rows(m, 256, seed=7)
    x[3, 200], x[5, 8] = float("nan"), -float("inf")
    x[4, 77] = 2.0**120                                      # finite, and so are its products
    x[1] *= 2.0**-110
    out = ops.gemm_w4a16(x, packed, scales)
    assert torch.isnan(out[3]).all()
    # An infinity gives infinities, and NaN where the weight is 0.
    w = dense(packed, scales)[:, 8]
    assert torch.equal(torch.isnan(out[5]), w == 0)
    assert torch.equal(out[5][w != 0], torch.where(w[w != 0] > 0, -float("inf"), float("inf")).to(torch.bfloat16))
    keep = [i for i in range(m) if i not in (3, 5)]
    check(out[keep], x[keep], packed, scales)


@pytest.mark.parametrize("m", [5, 12, 40])
def test_rows_of_any_range(m, plan):
    """Small values count beside large ones where the codes of those are 0."""
    g = torch.Generator(device="cuda").manual_seed(m)
    packed, scales = weights(200, 512, 64, seed=12)
    x = torch.randn(m, 512, generator=g, device="cuda")
    x = torch.ldexp(x, torch.randint(-50, 51, x.shape, generator=g, device="cuda")).to(torch.bfloat16)
    x[1] = 0
    x[1, 7], x[1, 300] = 2.0**90, 2.0**-30
    codes = unpack(packed)
    codes[:, 7] = 0
    packed = pack(codes)
    check(ops.gemm_w4a16(x, packed, scales), x, packed, scales)


@pytest.mark.parametrize("m", [4, 40])
def test_two_streams_at_once(m):
    """Each call has rows and a workspace of its own."""
    sets = [weights(6400, 1024, 64, seed=s) for s in (30, 31)]
    xs = [rows(m, 1024, seed=s) for s in (32, 33)]
    wants = [ops.gemm_w4a16(x, *w) for x, w in zip(xs, sets)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    outs = [[], []]
    for _ in range(30):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(ops.gemm_w4a16(xs[i], *sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for mine, want in zip(outs, wants) for out in mine)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("m", [5, 20])
def test_another_stream_and_a_replayed_graph_with_new_weights(m, plan):
    packed, scales = weights(300, 512, 128, seed=8)
    other, other_scales = weights(300, 512, 128, seed=9)
    x = rows(m, 512, seed=10)
    out = torch.empty(m, 300, device="cuda", dtype=torch.bfloat16)
    ops.gemm_w4a16(x, packed, scales, out=out)
    want = ops.gemm_w4a16(x, other, other_scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gemm_w4a16(x, packed, scales, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        packed.copy_(other)
        scales.copy_(other_scales)
        graph.replay()
    side.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("m", [2, 30])
def test_weights_written_right_before_the_call(m, plan):
    """Nothing of the weights is read before the launches ahead of the call end."""
    x = rows(m, 2048, seed=11)
    sets = [weights(4096, 2048, 128, seed=s) for s in (20, 21)]
    wants = [ops.gemm_w4a16(x, *s) for s in sets]
    packed, scales = (t.clone() for t in sets[0])
    outs = []
    for i in range(40):
        packed.copy_(sets[i % 2][0])
        scales.copy_(sets[i % 2][1])
        outs.append(ops.gemm_w4a16(x, packed, scales))
    assert all(torch.equal(out, wants[i % 2]) for i, out in enumerate(outs))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_linear_of_several_linears(group):
    torch.manual_seed(3)
    layers = [torch.nn.Linear(256, n, bias=b).cuda().to(torch.bfloat16) for n, b in ((48, True), (7, False), (130, True))]
    with torch.no_grad():
        layers[0].weight[5, :group] = 0
    merged = WeightOnlyLinear.from_linear(*layers, group=group)
    x = rows(6, 256, seed=4).view(2, 3, 256)
    out = merged(x)
    assert out.shape == (2, 3, 185) and (merged.in_features, merged.out_features, merged.group) == (256, 185, group)
    w = dense(merged.packed_weight, merged.weight_scale)
    bias = torch.cat([layers[0].bias, torch.zeros(7, device="cuda", dtype=torch.bfloat16), layers[2].bias]).detach()
    check(out.view(6, 185), x.view(6, 256), merged.packed_weight, merged.weight_scale, bias)
    assert torch.equal(merged.bias, bias)
    # Half a step of a group's scale (max / 7, rounded by 2^-9 of itself, which a
    # code of 7 multiplies and which may cut the largest weight).
    full = torch.cat([layer.weight for layer in layers]).detach().double()
    most = full.unflatten(1, (-1, group)).abs().amax(-1).repeat_interleave(group, dim=1)
    assert ((w - full).abs() <= most * (0.5 / 7 + 2.0**-8)).all()
    assert torch.equal(out[0, 0], merged(x[0, 0]))


def test_refusals():
    packed, scales = weights(32, 256, 64, seed=1)
    x = rows(2, 256, seed=2)
    for args, message in (
        ((x.float(), packed, scales), "bf16"),
        ((x[:, :128], packed, scales), "packed"),
        ((x, packed.to(torch.int8), scales), "packed"),
        ((x, packed, scales.float()), "scales"),
        ((x, packed, scales[:16]), "scales"),
        ((x, packed, scales[:, :3].contiguous()), "group"),
        ((x, packed, scales[:, :1].contiguous()), "group"),
        ((x, packed, scales, scales[0]), "bias"),
        ((x.cpu(), packed, scales), "CUDA"),
        ((x, packed.cpu(), scales), "device"),
        ((torch.cat([x, x], 1)[:, 4:260], packed, scales), "aligned"),
    ):
        with pytest.raises(ValueError, match=message):
            ops.gemm_w4a16(*args)
    with pytest.raises(ValueError, match="mode"):
        _lib.set_w4_mode(3)
    with pytest.raises(ValueError, match="out"):
        ops.gemm_w4a16(x, packed, scales, out=torch.empty(2, 31, device="cuda", dtype=torch.bfloat16))
    assert ops.gemm_w4a16(x[:0], packed, scales).shape == (0, 32)
    with pytest.raises(ValueError, match="group"):
        quantize_groups(torch.zeros(4, 96, device="cuda"), 64)
    with pytest.raises(ValueError, match="finite"):
        quantize_groups(torch.full((4, 64), float("inf"), device="cuda"), 64)
    with pytest.raises(ValueError, match="feature"):
        WeightOnlyLinear(packed, scales)(x[:, :128])
    with pytest.raises(ValueError, match="BF16"):
        WeightOnlyLinear.from_linear(torch.nn.Linear(64, 4).cuda(), group=64)
