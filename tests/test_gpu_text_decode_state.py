"""What a packed decoder leaves behind: a failed call changes nothing."""

import pytest
import torch

from pir2_b200.text_decode import PackedTextDecoder, TextCache
from test_gpu_text_decode import small_policy

pytestmark = pytest.mark.gpu


def state(cache):
    return list(cache.tokens), [list(h) for h in cache.held], list(cache.free)


@torch.inference_mode()
def test_a_layer_that_raises_leaves_the_cache_as_it_was():
    backbone = small_policy().backbone
    g = torch.Generator(device="cuda").manual_seed(1)
    calls = [([40, 7], False), ([30, 90], True), ([1, 1], False), ([30, 90], True), ([30, 90], False)]
    rows = [torch.randn(sum(new), 512, generator=g, device="cuda").to(torch.bfloat16) for new, _ in calls]

    def results(with_failures):
        cache = TextCache(2, 12, 2, 128, batch=2, max_tokens=160, page_size=32, dtype=torch.int8)
        decoder = PackedTextDecoder(backbone, cache)
        norm, out = backbone.layers[1].input_layernorm, []
        for (new, fails), hidden in zip(calls, rows):
            if not fails:
                out.append(decoder.run(hidden, new))
            elif with_failures:
                def broken(x):
                    raise RuntimeError("out of memory")

                before = state(cache)
                norm.forward = broken
                try:
                    with pytest.raises(RuntimeError, match="out of memory"):
                        decoder.run(hidden, new)
                finally:
                    del norm.forward
                assert state(cache) == before
                assert all("forward" not in attn.__dict__ for attn in decoder.attentions)
        return out

    for got, want in zip(results(True), results(False)):
        assert torch.equal(got, want)


def test_rewind():
    cache = TextCache(1, 8, 1, 64, batch=2, max_tokens=128, page_size=32, dtype=torch.int8)
    cache.extend([33, 64])
    before = state(cache)
    cache.extend([60, 1])
    cache.rewind([33, 64])
    assert state(cache) == before
    cache.rewind([32, 0])
    assert [len(h) for h in cache.held] == [1, 0] and len(cache.free) == 7 and cache.tokens == [32, 0]
    for tokens in ([33, 0], [-1, 0], [32]):
        with pytest.raises(ValueError, match="rewind"):
            cache.rewind(tokens)
