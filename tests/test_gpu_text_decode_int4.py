"""The packed text decoder with what a decoded token runs in 4 bits: the cache,
norm + rotation + cache write in one launch, and the projections' weights."""

import pytest
import torch

from pir2_b200 import _lib, harness
from pir2_b200.text_decode import PackedTextDecoder, TextCache
from pir2_b200.transformer import TransformerINT
from pir2_b200.weight_only import TextProjections
from test_gpu_text_decode import far, plain, small_policy

pytestmark = pytest.mark.gpu

CALLS = [[70, 0, 33, 200], [1, 1, 1, 1], [0, 150, 17, 1], [1, 1, 1, 1], [65, 1, 0, 0]]
# As in the decoder's other tests: ten bf16 roundings of the hidden state per
# layer, and what the cache's codes add to keys and values.  4-bit codes: half a
# step is a 14th of a group's largest value, about a sixth of a typical one's
# (32 normal values have a largest of 2.1), uniform: 0.1 of the values in the
# mean; as int8's 1/127 of 2.7 / sqrt(3) = 0.012 goes with a bound of 0.04 over
# bf16's 0.03, 0.1 goes with 0.03 + 0.1.
BOUNDS = {torch.bfloat16: 0.03, torch.int8: 0.04, torch.float8_e4m3fn: 0.08, torch.uint8: 0.13}


def run(backbone, decoder, rows, calls=CALLS):
    got, at = [[] for _ in rows], [0] * len(rows)
    for new in calls:
        hidden = torch.cat([rows[b][at[b] : at[b] + n] for b, n in enumerate(new)])
        for b, part in enumerate(decoder.run(hidden, new).split(new)):
            got[b].append(part)
            at[b] += new[b]
    assert all("forward" not in m.__dict__ for layer in backbone.layers for m in (layer.self_attn, layer.mlp))
    assert _lib.device_status() == 0
    return [torch.cat(g) for g in got]


def inputs(seed, width=512, calls=CALLS):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(sum(c[b] for c in calls), width, generator=g, device="cuda").to(torch.bfloat16) for b in range(len(calls[0]))]


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("dtype", list(BOUNDS), ids=["bf16", "int8", "e4m3", "int4"])
@torch.inference_mode()
def test_caches_and_the_single_launch(dtype, append):
    backbone, rows = small_policy().backbone, inputs(5)
    cache = TextCache(2, 24, 2, 128, batch=4, max_tokens=300, page_size=32, dtype=dtype)
    got = run(backbone, PackedTextDecoder(backbone, cache, append=append), rows)
    for b in range(4):
        assert far(got[b], plain(backbone, rows[b])) < BOUNDS[dtype]


class Rounded(torch.nn.Module):
    """A Linear whose weights are what a WeightOnlyLinear's codes stand for."""

    def __init__(self, linear):
        super().__init__()
        from int4_reference import unpack

        w = unpack(linear.packed_weight).float().unflatten(1, (-1, linear.group)) * linear.weight_scale.float()[..., None]
        self.w = w.flatten(1)

    def forward(self, x):
        return (x.float() @ self.w.T).to(torch.bfloat16)


@pytest.mark.parametrize("group", [32, 128])
@torch.inference_mode()
def test_weights_in_4_bits_are_used_for_few_rows(group):
    """The layers of short calls equal the same layers with the weights that the
    codes stand for; long calls keep the layers' own."""
    policy = small_policy()
    backbone, rows = policy.backbone, inputs(6)
    narrow = TextProjections(backbone, group=group, rows=8)
    make = lambda **more: PackedTextDecoder(  # noqa: E731
        backbone, TextCache(2, 24, 2, 128, batch=4, max_tokens=300, page_size=32, dtype=torch.bfloat16), append=True, **more)
    got = run(backbone, make(weight_only=narrow), rows)
    # The same calls with the short ones through the rounded layers.
    twin = harness.Backbone(backbone.config).to("cuda", torch.bfloat16).eval()
    twin.load_state_dict(backbone.state_dict())
    decoder, own = make(), [(layer.self_attn, layer.mlp) for layer in twin.layers]
    decoder.backbone, decoder.attentions = twin, [a for a, _ in own]
    want, at = [[] for _ in rows], [0] * 4
    for new in CALLS:
        if sum(new) <= 8:
            for i, layer in enumerate(twin.layers):
                merged = [Rounded(x) for x in (narrow.qkv[i], narrow.o[i], narrow.gate_up[i], narrow.down[i])]
                widths = [512, 256, 256]
                for name, part in zip(("q_proj", "k_proj", "v_proj"), merged[0].w.split(widths)):
                    getattr(layer.self_attn, name).weight.copy_(part)
                layer.self_attn.o_proj.weight.copy_(merged[1].w)
                for name, part in zip(("gate_proj", "up_proj"), merged[2].w.split(1024)):
                    getattr(layer.mlp, name).weight.copy_(part)
                layer.mlp.down_proj.weight.copy_(merged[3].w)
        else:
            twin.load_state_dict(backbone.state_dict())
        hidden = torch.cat([rows[b][at[b] : at[b] + n] for b, n in enumerate(new)])
        for b, part in enumerate(decoder.run(hidden, new).split(new)):
            want[b].append(part)
            at[b] += new[b]
    for b in range(4):
        # Both round their hidden state some ten times a layer; the twin's weights
        # are rounded to bf16 once more (2^-9 each).
        assert far(got[b], torch.cat(want[b])) < BOUNDS[torch.bfloat16]
    # It is not the plain layers' result: 4-bit weights are off by some 0.1.
    assert far(got[0], run(backbone, make(), rows)[0]) > 0


@torch.inference_mode()
def test_everything_together_decodes_each_robot_as_alone():
    backbone = small_policy().backbone
    lengths = [37, 120, 64]
    rows = [torch.randn(n, 512, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").to(torch.bfloat16) for n in lengths]
    narrow = TextProjections(backbone, rows=8)   # below every prompt, alone or together

    def decode(some):
        cache = TextCache(2, 16, 2, 128, batch=len(some), max_tokens=200, dtype=torch.uint8)
        decoder = PackedTextDecoder(backbone, cache, append=True, weight_only=narrow)
        out = decoder.run(torch.cat(some), [len(r) for r in some])
        last = torch.stack([part[-1] for part in out.split([len(r) for r in some])])
        return decoder.decode(last, 6)

    together = decode(rows)
    assert together.shape == (3, 6) and _lib.device_status() == 0
    for b in range(3):
        assert torch.equal(together[b : b + 1], decode([rows[b]]))


@torch.inference_mode()
def test_installed_projections_stay():
    """While a precision is installed, a decoder with 4-bit weights runs it."""
    policy = small_policy()
    names = {
        f"backbone.layers.{i}.{part}"
        for i in range(2)
        for part in ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj",
                     "mlp.up_proj", "mlp.down_proj")
    }
    controller = TransformerINT(policy, names, native=False, expanded=True)
    narrow = TextProjections(policy.backbone)
    hidden = inputs(9, calls=[[3, 2]])

    def once(**more):
        cache = TextCache(2, 8, 2, 128, batch=2, max_tokens=64, dtype=torch.bfloat16)
        return PackedTextDecoder(policy.backbone, cache, controller=controller, **more).run(torch.cat(hidden), [3, 2])

    try:
        controller.set("w8a8")
        assert torch.equal(once(weight_only=narrow), once())
        controller.set("bf16")
        assert not torch.equal(once(weight_only=narrow), once())
    finally:
        controller.close()


def test_refusals():
    policy = small_policy()
    cache = TextCache(2, 4, 2, 128, batch=1, max_tokens=64, dtype=torch.uint8)
    assert cache.layers[0].dtype == torch.uint8 and cache.layers[0].head_dim == 128
    short = TextProjections(policy.backbone)
    short.qkv = short.qkv[:1]
    with pytest.raises(ValueError, match="layers"):
        PackedTextDecoder(policy.backbone, cache, weight_only=short)
    policy.backbone.layers[0].mlp.config.hidden_act = "gelu"
    with pytest.raises(ValueError, match="SiLU"):
        TextProjections(policy.backbone)
