"""Packed decoders of several threads over one backbone, on the CPU: the
attention operators are replaced by functions that mark whose they are."""

import threading
from types import SimpleNamespace

import pytest
import torch

from pir2_b200.text_decode import PackedTextDecoder


class Attention(torch.nn.Module):
    head_dim = 128

    def forward(self, x, cos, sin):
        return x + 1000.0


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.self_attn = Attention()

    def forward(self, h, cos, sin):
        return self.self_attn(h, cos, sin)


class Cache:
    def __init__(self, layers):
        self.layers, self.tokens = [None] * layers, [0]

    def extend(self, new):
        self.tokens = [t + n for t, n in zip(self.tokens, new)]


class Marked(PackedTextDecoder):
    """Adds `mark` in every layer, after all threads have come to it."""

    def __init__(self, backbone, mark, together):
        super().__init__(backbone, Cache(len(backbone.layers)))
        self.mark, self.together = mark, together

    def _attend(self, *args):
        self.together.wait(timeout=20)
        return args[-3] + self.mark


@pytest.mark.parametrize("own", [False, True])
def test_each_thread_gets_its_own_attention(own):
    config = SimpleNamespace(rope_theta=1e4, head_dim=128)
    backbone = SimpleNamespace(layers=torch.nn.ModuleList(Layer() for _ in range(3)), config=config)
    attentions = [layer.self_attn for layer in backbone.layers]
    if own:                              # an instance forward, as fusions install them
        for attn in attentions:
            attn.forward = lambda x, cos, sin: x + 2000.0
    before = [attn.__dict__.get("forward") for attn in attentions]
    step = 2000.0 if own else 1000.0
    together = threading.Barrier(3)
    decoders = [Marked(backbone, mark, together) for mark in (1.0, 10.0)]
    hidden, results, errors = torch.zeros(2, 4), {}, []

    def decoded(decoder):
        try:
            results[decoder.mark] = decoder.run(hidden, [2])
        except BaseException as error:
            together.abort()
            errors.append(error)

    threads = [threading.Thread(target=decoded, args=(decoder,)) for decoder in decoders]
    for t in threads:
        t.start()
    plain = []
    try:
        for layer in backbone.layers:    # a plain call beside them, layer by layer
            together.wait(timeout=20)
            plain.append(layer(hidden, None, None))
    except threading.BrokenBarrierError:
        pass
    for t in threads:
        t.join()
    assert not errors
    assert torch.equal(results[1.0], hidden + 3) and torch.equal(results[10.0], hidden + 30)
    assert all(torch.equal(y, hidden + step) for y in plain)
    assert all(attn.__dict__.get("forward") is f for attn, f in zip(attentions, before))


def test_forwards_come_back_after_an_exception():
    config = SimpleNamespace(rope_theta=1e4, head_dim=128)
    backbone = SimpleNamespace(layers=torch.nn.ModuleList([Layer()]), config=config)

    class Broken(PackedTextDecoder):
        def _attend(self, *args):
            raise RuntimeError("no attention")

    cache = Cache(1)
    cache.rewind = lambda tokens: setattr(cache, "tokens", list(tokens))
    with pytest.raises(RuntimeError, match="no attention"):
        Broken(backbone, cache).run(torch.zeros(2, 4), [2])
    assert "forward" not in backbone.layers[0].self_attn.__dict__ and cache.tokens == [0]
