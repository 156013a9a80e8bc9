"""The packed text decoder inside an installed session, with the fused
producers, residuals and SwiGLU of its layers."""

from types import SimpleNamespace

import pytest
import torch

from pir2_b200.config import OptimizationConfig
from pir2_b200.session import GrootOptimizations
from pir2_b200.text_decode import PackedTextDecoder, TextCache
from test_gpu_text_decode import far, plain, small_policy

pytestmark = pytest.mark.gpu

# As in the decoder's other tests: the bf16 attention's bound beside quantized
# projections (whose codes may move by one), twice it for 4-bit codes.
BOUNDS = {"w8a8": 0.05, "w4a4": 0.1}


@pytest.mark.parametrize("precision", list(BOUNDS))
@pytest.mark.parametrize("with_controller", [True, False], ids=["grouped", "single"])
@torch.inference_mode()
def test_prompts_and_chunks_under_the_session_fusions(precision, with_controller):
    policy = small_policy()
    config = OptimizationConfig(
        precision=precision, fusion=True, scope="all", group_conditioning=True, norm_modulation_quant=True,
        residual_norm_quant=True,
    )
    g = torch.Generator(device="cuda").manual_seed(8)
    calls = [[70, 33], [1, 40], [1, 1]]
    rows = [torch.randn(sum(c[b] for c in calls), 512, generator=g, device="cuda").to(torch.bfloat16) for b in range(2)]
    with GrootOptimizations(SimpleNamespace(model=policy), config) as session:
        assert session.residual is not None and session.pointwise is not None
        cache = TextCache(2, 12, 2, 128, batch=2, max_tokens=128, page_size=32, dtype=torch.bfloat16)
        decoder = PackedTextDecoder(
            policy.backbone, cache, controller=session.controller if with_controller else None
        )
        forwards = [attn.__dict__.get("forward") for attn in decoder.attentions]
        got, at = [[], []], [0, 0]
        for new in calls:
            hidden = torch.cat([rows[b][at[b] : at[b] + n] for b, n in enumerate(new)])
            for b, part in enumerate(decoder.run(hidden, new).split(new)):
                got[b].append(part)
                at[b] += new[b]
        for b in range(2):
            assert far(torch.cat(got[b]), plain(policy.backbone, rows[b])) < BOUNDS[precision]
        assert [attn.__dict__.get("forward") for attn in decoder.attentions] == forwards
