"""The packed text decoder follows the precision that is installed in the
layers at the time of a call."""

import pytest
import torch

from pir2_b200.text_decode import PackedTextDecoder, TextCache
from pir2_b200.transformer import TransformerINT
from test_gpu_text_decode import far, plain, small_policy

pytestmark = pytest.mark.gpu

MODES = ["bf16", "w8a8", "w4a4", "w8a8", "bf16"]


def controlled(policy):
    names = {
        f"backbone.layers.{i}.{part}"
        for i in range(2)
        for part in ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj",
                     "mlp.up_proj", "mlp.down_proj")
    }
    return TransformerINT(policy, names, native=False, expanded=True)


@pytest.mark.parametrize("bits", [None, 8, 4])
@torch.inference_mode()
def test_projections_are_those_installed(bits):
    """q, k and v of a call are, bit for bit, what the layers' own projections
    give in every mode, and after the controller has closed."""
    policy = small_policy()
    controller = controlled(policy)
    decoder = PackedTextDecoder(
        policy.backbone, TextCache(2, 8, 2, 128, batch=1, max_tokens=128), controller=controller, bits=bits
    )
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, 33, 512, generator=g, device="cuda").to(torch.bfloat16)
    results = {}
    try:
        for mode in [*MODES, "closed"]:
            controller.close() if mode == "closed" else controller.set(mode)
            for attn in decoder.attentions:
                got = decoder._project(attn, x)
                controller.clear_projection_cache()
                want = torch.cat((attn.q_proj(x), attn.k_proj(x), attn.v_proj(x)), dim=-1)
                assert torch.equal(got, want), mode
            results[mode] = got
    finally:
        controller.close()
    assert torch.equal(results["bf16"], results["closed"])
    assert not torch.equal(results["bf16"], results["w8a8"]) and not torch.equal(results["w4a4"], results["w8a8"])


@torch.inference_mode()
def test_one_decoder_through_all_modes():
    """Against the same layers run prompt by prompt in the same mode; the bf16
    attention's bound, twice it for W4A4, whose codes are 18 times as coarse."""
    policy = small_policy()
    controller = controlled(policy)
    g = torch.Generator(device="cuda").manual_seed(6)
    lengths = [90, 41]
    hidden = torch.randn(131, 512, generator=g, device="cuda").to(torch.bfloat16)
    cache = TextCache(2, 8, 2, 128, batch=2, max_tokens=128, dtype=torch.bfloat16)
    decoder = PackedTextDecoder(policy.backbone, cache, controller=controller)
    try:
        for mode in MODES:
            controller.set(mode)
            out = decoder.run(hidden, lengths)
            for part, rows in zip(out.split(lengths), hidden.split(lengths)):
                assert far(part, plain(policy.backbone, rows)) < (0.1 if mode == "w4a4" else 0.05), mode
            for b in range(2):
                cache.release(b)
    finally:
        controller.close()
