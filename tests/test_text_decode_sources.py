"""When a decoder's short calls take the 4-bit projections: only while the layers
hold what was packed.  On the CPU, with the packing of a Linear replaced."""

import threading

import pytest
import torch

from pir2_b200 import harness, weight_only
from pir2_b200.text_decode import _ROUTES, PackedTextDecoder


class Cache:
    def __init__(self, layers):
        self.layers, self.batch = [None] * layers, 2


@pytest.fixture
def made(monkeypatch):
    monkeypatch.setattr(weight_only.WeightOnlyLinear, "from_linear", classmethod(lambda cls, *linears, group: linears))
    config = harness.VLMConfig(hidden=128, layers=2, heads=1, kv_heads=1, intermediate=256, vocab=64)
    backbone = harness.Backbone(config).eval()
    projections = weight_only.TextProjections(backbone, rows=8)
    return backbone, projections, PackedTextDecoder(backbone, Cache(2), weight_only=projections)


LINEARS = ["self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj",
           "mlp.down_proj"]


def test_rows(made):
    _, _, decoder = made
    assert decoder._narrow(1) and decoder._narrow(8) and not decoder._narrow(9)


@pytest.mark.parametrize("layer", [0, 1])
@pytest.mark.parametrize("name", LINEARS)
def test_linears_that_are_not_those_packed(made, layer, name):
    backbone, _, decoder = made
    owner, part = backbone.layers[layer].get_submodule(name.split(".")[0]), name.split(".")[1]
    linear = getattr(owner, part)
    setattr(owner, part, torch.nn.Linear(linear.in_features, linear.out_features, bias=False))
    assert not decoder._narrow(1)
    setattr(owner, part, linear)
    assert decoder._narrow(1)
    # Another weight, the same one written to, its memory replaced, a bias that was not there.
    weight = linear.weight
    linear.weight = torch.nn.Parameter(weight.detach().clone())
    assert not decoder._narrow(1)
    linear.weight = weight
    assert decoder._narrow(1)
    linear.bias = torch.nn.Parameter(torch.zeros(linear.out_features))
    assert not decoder._narrow(1)
    linear.bias = None
    assert decoder._narrow(1)
    data = weight.data
    weight.data = data.clone()
    assert not decoder._narrow(1)
    weight.data = data
    assert decoder._narrow(1)
    for hook in (linear.register_forward_hook, linear.register_forward_pre_hook):
        handle = hook(lambda *args: None)
        assert not decoder._narrow(1)
        handle.remove()
        assert decoder._narrow(1)
    linear.forward = lambda x: x
    assert not decoder._narrow(1)
    del linear.forward
    assert decoder._narrow(1)
    with torch.no_grad():
        weight.mul_(2)
    assert not decoder._narrow(1)


@pytest.mark.parametrize("name", ["mlp", "self_attn", "input_layernorm", "post_attention_layernorm"])
def test_modules_that_are_not_those_packed(made, name):
    backbone, _, decoder = made
    layer = backbone.layers[1]
    own = getattr(layer, name)
    if name != "self_attn":              # which a decoder replaces in every call
        own.forward = lambda x: x
        assert not decoder._narrow(1)
        del own.forward
        assert decoder._narrow(1)
    if name in ("mlp", "self_attn"):
        setattr(layer, name, type(own)(backbone.config))
        assert not decoder._narrow(1)
        setattr(layer, name, own)
        assert decoder._narrow(1)
    backbone.layers[1] = harness.Qwen3VLTextDecoderLayer(backbone.config)
    assert not decoder._narrow(1)
    backbone.layers[1] = layer
    layer.forward = lambda h, cos, sin: h
    assert not decoder._narrow(1)


def test_weights_loaded_later(made):
    backbone, _, decoder = made
    backbone.load_state_dict(backbone.state_dict())
    assert not decoder._narrow(1)


def test_a_call_of_another_thread_installs_nothing(made):
    """The forwards that a running call puts into the modules are not installed
    ones; a forward that was there before it is."""
    backbone, _, decoder = made
    mlps = [layer.mlp for layer in backbone.layers]

    def meanwhile():
        seen, inside, leave = [], threading.Event(), threading.Event()

        def other():
            with _ROUTES.routed(mlps, [lambda x: x] * 2):
                inside.set()
                leave.wait(20)

        thread = threading.Thread(target=other)
        thread.start()
        assert inside.wait(20)
        assert all("forward" in mlp.__dict__ for mlp in mlps)
        seen = decoder._narrow(1)
        leave.set()
        thread.join()
        return seen

    assert meanwhile()
    mlps[1].forward = lambda x: x
    assert not meanwhile()


def test_vocabulary(made):
    backbone, projections, decoder = made
    asked = []
    projections.vocabulary = lambda x: asked.append(x.shape[0]) or x @ backbone.embed_tokens.weight.detach().T
    decoder._run = lambda hidden, new, narrow: hidden
    last = torch.randn(2, 128)
    decoder.decode(last, 2)
    assert asked == [2, 2]
    projections.rows = 1
    decoder.decode(last, 1)
    projections.rows = 8
    # Installed projections: the whole step as installed.
    backbone.layers[0].mlp.forward = lambda x: x
    decoder.decode(last, 1)
    del backbone.layers[0].mlp.forward
    with torch.no_grad():
        backbone.embed_tokens.weight.add_(1)
    assert decoder._narrow(2)            # the layers are those packed
    decoder.decode(last, 1)
    assert asked == [2, 2]


def test_projections_of_another_backbone(made):
    backbone, projections, _ = made
    other = harness.Backbone(backbone.config)
    with pytest.raises(ValueError, match="backbone's layers"):
        PackedTextDecoder(other, Cache(2), weight_only=projections)


def test_weights_without_versions(made):
    """Inference tensors count no versions: what replaces them is seen."""
    backbone, _, _ = made
    with torch.inference_mode():
        other = harness.Backbone(backbone.config)
        decoder = PackedTextDecoder(other, Cache(2), weight_only=weight_only.TextProjections(other, rows=8))
        assert decoder._narrow(1)
        other.layers[0].mlp.up_proj.weight = torch.nn.Parameter(other.layers[0].mlp.up_proj.weight.clone())
        assert not decoder._narrow(1)


def test_weights_that_are_no_parameters(monkeypatch):
    """A buffer in a weight's place is followed too; a weight that is computed
    anew each time never equals the one packed."""
    monkeypatch.setattr(weight_only.WeightOnlyLinear, "from_linear", classmethod(lambda cls, *linears, group: linears))
    backbone = harness.Backbone(harness.VLMConfig(hidden=128, layers=1, heads=1, kv_heads=1, intermediate=256, vocab=64))
    linear = backbone.layers[0].mlp.down_proj
    value = linear.weight.detach().clone()
    del linear.weight
    linear.register_buffer("weight", value)
    decoder = PackedTextDecoder(backbone, Cache(1), weight_only=weight_only.TextProjections(backbone))
    assert decoder._narrow(1)
    linear.weight = value.clone()
    assert not decoder._narrow(1)
    linear.weight = value
    assert decoder._narrow(1)
    value.add_(1)
    assert not decoder._narrow(1)
    torch.nn.utils.parametrize.register_parametrization(backbone.layers[0].mlp.up_proj, "weight", torch.nn.Tanh())
    decoder = PackedTextDecoder(backbone, Cache(1), weight_only=weight_only.TextProjections(backbone))
    assert not decoder._narrow(1)


@pytest.mark.parametrize("narrow", [True, False])
def test_rows_that_are_not_one_per_sequence(made, narrow):
    _, projections, decoder = made
    projections.vocabulary = lambda x: torch.zeros(x.shape[0], 64)
    projections.rows = 8 if narrow else 0
    with pytest.raises(ValueError, match="rows"):
        decoder.decode(torch.randn(1, 128), 1)


def test_rows_at_which_4_bit_weights_stop_by_themselves(made):
    """Above these the layers' own Linears are faster, and exact."""
    backbone, _, _ = made
    decoder = PackedTextDecoder(backbone, Cache(2), weight_only=weight_only.TextProjections(backbone))
    assert decoder._narrow(32) and not decoder._narrow(33)
