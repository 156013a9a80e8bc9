"""Short calls of a decoder with 4-bit weights whose backbone has changed since
they were packed: the backbone as it is answers, in every call length alike."""

import pytest
import torch

from pir2_b200 import _lib
from pir2_b200.fusion import SwiGLUFusion
from pir2_b200.text_decode import PackedTextDecoder, TextCache
from pir2_b200.transformer import TransformerINT
from pir2_b200.weight_only import TextProjections
from test_gpu_text_decode import small_policy

pytestmark = pytest.mark.gpu


def once(backbone, new=(3, 2), steps=2, **more):
    """(the rows of a short call, tokens decoded after it)."""
    cache = TextCache(2, 8, 2, 128, batch=2, max_tokens=64, dtype=torch.bfloat16)
    decoder = PackedTextDecoder(backbone, cache, append=True, **more)
    hidden = torch.randn(sum(new), 512, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    out = decoder.run(hidden, list(new))
    last = torch.stack([part[-1] for part in out.split(list(new))])
    tokens = decoder.decode(last, steps)
    assert _lib.device_status() == 0
    return torch.cat([out.flatten().float(), tokens.flatten().float()])


def gained(mlp, gain):
    """An MLP's forward with its result times `gain`, in its place."""
    plain = mlp.forward
    mlp.forward = lambda x: plain(x) * gain


@pytest.mark.parametrize("change", ["mlp", "swapped", "hook", "written", "data", "loaded"])
def test_changed_backbones_answer_themselves(change):
    backbone = small_policy().backbone
    packed = TextProjections(backbone)
    assert not torch.equal(once(backbone, weight_only=packed), once(backbone))
    layer, handle = backbone.layers[1], None
    if change == "mlp":
        gained(layer.mlp, 0.5)
    elif change == "swapped":
        linear = layer.self_attn.o_proj
        layer.self_attn.o_proj = torch.nn.Sequential(linear, torch.nn.Hardtanh(-0.1, 0.1))
    elif change == "hook":
        handle = layer.mlp.up_proj.register_forward_hook(lambda module, args, out: out * 0.5)
    elif change == "written":
        with torch.no_grad():
            layer.self_attn.v_proj.weight.mul_(2)
    elif change == "data":
        layer.mlp.down_proj.weight.data = layer.mlp.down_proj.weight.data * 2
    else:
        backbone.load_state_dict({name: 0.9 * w for name, w in backbone.state_dict().items()})
    assert torch.equal(once(backbone, weight_only=packed), once(backbone))
    if handle is not None:
        handle.remove()
        assert not torch.equal(once(backbone, weight_only=packed), once(backbone))
    if change in ("written", "data", "loaded"):
        assert not torch.equal(once(backbone, weight_only=TextProjections(backbone)), once(backbone))


def test_embeddings_written_to():
    """The output layer is the embeddings' own again; the layers keep their 4 bits."""
    backbone = small_policy().backbone
    packed = TextProjections(backbone)
    asked, vocabulary = [], packed.vocabulary
    packed.vocabulary = lambda x: asked.append(x.shape[0]) or vocabulary(x)
    first = once(backbone, weight_only=packed)
    assert asked == [2, 2]
    with torch.no_grad():
        backbone.embed_tokens.weight.mul_(1.5)
    again = once(backbone, weight_only=packed)
    assert asked == [2, 2] and torch.equal(first[: 5 * 512], again[: 5 * 512])


def test_an_installed_swiglu_stays():
    """A fusion that replaces the MLP's forward alone (its controller's
    projections are back to bf16) is not put aside by short calls."""
    policy = small_policy()
    names = {f"backbone.layers.{i}.mlp.{part}" for i in range(2) for part in ("gate_proj", "up_proj", "down_proj")}
    controller = TransformerINT(policy, names, native=False, expanded=True)
    packed = TextProjections(policy.backbone)
    fusion = SwiGLUFusion(policy, controller)
    try:
        fusion.set()
        assert all("forward" in layer.mlp.__dict__ for layer in policy.backbone.layers)
        assert torch.equal(once(policy.backbone, weight_only=packed), once(policy.backbone))
    finally:
        fusion.close()
        controller.close()
    assert not torch.equal(once(policy.backbone, weight_only=packed), once(policy.backbone))
