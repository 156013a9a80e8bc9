"""The packed text decoder (prompts of different lengths, a paged cache, new
tokens behind them) against the same layers run prompt by prompt."""

import pytest
import torch

from pir2_b200 import harness
from pir2_b200.text_decode import PackedTextDecoder, TextCache
from pir2_b200.transformer import TransformerINT

pytestmark = pytest.mark.gpu


def small_policy():
    vlm = harness.VLMConfig(hidden=512, layers=2, heads=4, kv_heads=2, intermediate=1024, vocab=1000)
    dit = harness.DiTConfig(hidden=256, layers=2, heads=4, head_dim=64, ff=512, context=512)
    return harness.build_policy("cuda", vlm=vlm, dit=dit, seed=3)


def plain(backbone, rows):
    """The layers on one prompt alone (torch attention)."""
    h = rows[None]
    cos, sin = backbone.rope(h.shape[1], h.device, h.dtype)
    for layer in backbone.layers:
        h = layer(h, cos, sin)
    return h[0]


def far(got, want):
    return ((got.double() - want.double()).norm() / want.double().norm()).item()


# A layer rounds its hidden state to bf16 (2^-9 of it) some ten times in either
# path; 8-bit rows add 1/254 (int8: half a step of the row's largest value, 3.5
# times the others for 128 normal values) or 1/32 (E4M3's half step, 2^-4 / 2)
# to keys and values, which the average over keys and the residual shrink.
BOUNDS = {torch.bfloat16: 0.03, torch.int8: 0.04, torch.float8_e4m3fn: 0.08}


@pytest.mark.parametrize("dtype", list(BOUNDS), ids=["bf16", "int8", "e4m3"])
@torch.inference_mode()
def test_prompts_chunks_and_tokens_match_whole_prompts(dtype):
    backbone = small_policy().backbone
    g = torch.Generator(device="cuda").manual_seed(5)
    calls = [[70, 0, 33, 200], [1, 1, 1, 1], [0, 150, 17, 1], [1, 1, 1, 1], [65, 1, 0, 0]]
    total = [sum(c[b] for c in calls) for b in range(4)]
    rows = [torch.randn(n, 512, generator=g, device="cuda").to(torch.bfloat16) for n in total]
    cache = TextCache(2, 24, 2, 128, batch=4, max_tokens=300, page_size=32, dtype=dtype)
    decoder = PackedTextDecoder(backbone, cache)
    got, at = [[] for _ in range(4)], [0] * 4
    for new in calls:
        hidden = torch.cat([rows[b][at[b] : at[b] + n] for b, n in enumerate(new)])
        out = decoder.run(hidden, new)
        for b, part in enumerate(out.split(new)):
            got[b].append(part)
            at[b] += new[b]
    for b in range(4):
        assert far(torch.cat(got[b]), plain(backbone, rows[b])) < BOUNDS[dtype]
    assert all("forward" not in layer.self_attn.__dict__ for layer in backbone.layers)


@torch.inference_mode()
def test_quantized_projections_and_the_grouped_gemm():
    """W8A8 projections through TransformerINT: the packed run equals the same
    quantized layers run prompt by prompt (bf16 attention bound)."""
    policy = small_policy()
    names = {
        f"backbone.layers.{i}.{part}"
        for i in range(2)
        for part in ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj",
                     "mlp.up_proj", "mlp.down_proj")
    }
    controller = TransformerINT(policy, names, native=False, expanded=True)
    try:
        controller.set("w8a8")
        g = torch.Generator(device="cuda").manual_seed(6)
        lengths = [90, 41]
        hidden = torch.randn(131, 512, generator=g, device="cuda").to(torch.bfloat16)
        cache = TextCache(2, 8, 2, 128, batch=2, max_tokens=128, dtype=torch.bfloat16)
        decoder = PackedTextDecoder(policy.backbone, cache, controller=controller)
        out = decoder.run(hidden, lengths)
        for part, rows in zip(out.split(lengths), hidden.split(lengths)):
            assert far(part, plain(policy.backbone, rows)) < 0.05
    finally:
        controller.close()


@torch.inference_mode()
def test_greedy_decoding_of_a_batch_equals_one_robot_alone():
    backbone = small_policy().backbone
    g = torch.Generator(device="cuda").manual_seed(7)
    lengths = [37, 120, 64]
    rows = [torch.randn(n, 512, generator=g, device="cuda").to(torch.bfloat16) for n in lengths]

    def decode(some):
        cache = TextCache(2, 16, 2, 128, batch=len(some), max_tokens=200, dtype=torch.int8)
        decoder = PackedTextDecoder(backbone, cache)
        out = decoder.run(torch.cat(some), [len(r) for r in some])
        last = torch.stack([part[-1] for part in out.split([len(r) for r in some])])
        return decoder.decode(last, 6)

    together = decode(rows)
    for b in range(3):
        # The same kernels on the same sequence: batch mates change nothing.
        assert torch.equal(together[b : b + 1], decode([rows[b]]))


def test_cache_pages_are_dealt_and_returned():
    cache = TextCache(1, 6, 1, 64, batch=2, max_tokens=128, page_size=32, dtype=torch.int8)
    cache.extend([33, 64])
    assert [len(h) for h in cache.held] == [2, 2] and len(cache.free) == 2
    with pytest.raises(ValueError, match="free"):
        cache.extend([60, 64])
    with pytest.raises(ValueError, match="max_tokens"):
        cache.extend([96, 0])
    with pytest.raises(ValueError, match="per sequence"):
        cache.extend([1])
    assert cache.tokens == [33, 64] and len(cache.free) == 2
    cache.release(0)
    cache.extend([0, 64])
    assert len(cache.held[1]) == 4 and cache.lengths.tolist() == [0, 128] and cache.starts.tolist() == [0, 0, 64]
    held = set(cache.held[1])
    assert len(held) == 4 and set(cache.table[1, :4].tolist()) == held


def test_refusals():
    backbone = small_policy().backbone
    with pytest.raises(ValueError, match="per layer"):
        PackedTextDecoder(backbone, TextCache(1, 4, 2, 128, batch=1, max_tokens=64))
    decoder = PackedTextDecoder(backbone, TextCache(2, 4, 2, 128, batch=1, max_tokens=64))
    with pytest.raises(ValueError, match="rows"):
        decoder.run(torch.zeros(3, 512, device="cuda", dtype=torch.bfloat16), [2])
    assert decoder.run(torch.zeros(0, 512, device="cuda", dtype=torch.bfloat16), [0]).shape == (0, 512)
