"""Linears whose weights are held in 4 bits and whose activations stay bf16, for
decoding a few rows at a time.

The reference's int4 format (coexecution/kernels/ampere_ada/integer.py:222-238)
has one scale per output channel and quantises activations to 4 bits as well,
which suits many rows; a decoded token's Linears are bound by reading weights,
so here the weights alone are narrow, with a bf16 scale for every group of 32, 64
or 128 of a channel's weights.
"""

from functools import partial

import torch
import torch.nn.functional as F

from . import ops

GROUPS = (32, 64, 128)

# Rows up to which a backbone's 4-bit projections take its calls.  Graph replays on
# one B200, us, the layers' own bf16 Linears (q|k|v three, gate|up two of them)
# against the 4-bit ones in groups of 128:
#   rows                         1            8            16           32           48           64
#   q|k|v     2048 -> 4096       23.1  3.2    20.4  3.7    19.1  5.5    17.6  7.2    16.3 10.3    16.3 10.9
#   o         2048 -> 2048       8.4   2.1    7.1   2.3    5.6   3.4    5.6   4.5    5.7   6.5    5.7   7.5
#   gate|up   2048 -> 12288      13.9  7.0    13.6  7.4    14.7 10.0    15.1 13.0    14.7 23.7    14.1 25.5
#   down      6144 -> 2048       16.8  4.1    16.1  4.8    10.4  6.4    10.4 10.0    10.4 15.4    10.6 18.4
#   output    2048 -> 151936     101  35      103  35      105  70      106 101      105 203      106 221
# (In groups of 32 down takes 12.9 at 32 rows and the output layer 106.)  The device
# is busy for 1.91 ms a token of 16 such layers in bf16 and 1.14 in 4 bits for one
# sequence, 2.13 and 1.96 for 32, 2.16 and 2.59 for 64.
NARROW_ROWS = 32


def quantize_groups(weight, group):
    """(packed uint8 [n, k / 2], scales bf16 [n, k / group]) of weights [n, k]:
    scale = bf16(max|w| / 7) of a group (1 for zeros), code = w / scale rounded
    to nearest even and clamped to -7..7, the even k in the low bits."""
    if group not in GROUPS or weight.ndim != 2 or weight.shape[1] % group or not weight.shape[1]:
        raise ValueError(f"quantize_groups: group must be one of {GROUPS} and divide the weights' columns")
    w = weight.detach().float()
    if not torch.isfinite(w).all():
        raise ValueError("Weights must be finite")
    w = w.unflatten(1, (-1, group))
    most = w.abs().amax(-1)
    scales = (most / torch.full_like(most, 7)).to(torch.bfloat16)   # by a number: a product with its reciprocal
    scales = torch.where(scales == 0, torch.ones_like(scales), scales)
    codes = torch.round(w / scales.float()[..., None]).clamp(-7, 7).flatten(1).to(torch.int8)
    u = codes.view(torch.uint8) & 15
    return u[:, 0::2] | (u[:, 1::2] << 4), scales


class WeightOnlyLinear(torch.nn.Module):
    """y = x W^T + b with W in 4 bits and groups of `group` weights per scale."""

    def __init__(self, packed, scales, bias=None):
        super().__init__()
        self.register_buffer("packed_weight", packed)
        self.register_buffer("weight_scale", scales)
        self.register_buffer("bias", bias)
        self.out_features, self.in_features = packed.shape[0], 2 * packed.shape[1]
        self.group = self.in_features // scales.shape[1]

    @classmethod
    def from_linear(cls, *linears, group=128):
        """Of one Linear, or of several with the same input side by side (their
        outputs concatenated)."""
        weights = [linear.weight for linear in linears]
        if not weights or any(not w.is_cuda or w.dtype != torch.bfloat16 or w.shape[1] != weights[0].shape[1] for w in weights):
            raise ValueError("WeightOnlyLinear requires CUDA BF16 weights of one input width")
        packed, scales = zip(*(quantize_groups(w, group) for w in weights))
        biases = [linear.bias for linear in linears]
        bias = None
        if any(b is not None for b in biases):
            bias = torch.cat([w.new_zeros(w.shape[0]) if b is None else b.detach().to(torch.bfloat16) for w, b in zip(weights, biases)])
        return cls(torch.cat(packed), torch.cat(scales), bias)

    def forward(self, x):
        if x.shape[-1] != self.in_features:
            raise ValueError("Wrong input feature count")
        rows = x.reshape(-1, self.in_features)
        return ops.gemm_w4a16(rows, self.packed_weight, self.weight_scale, self.bias).view(*x.shape[:-1], self.out_features)


def _mark(tensor):
    """What changes when a tensor's memory is replaced or written to.  (Inference
    tensors count no versions.)"""
    return None if tensor is None else (tensor.data_ptr(), None if tensor.is_inference() else tensor._version)


class TextProjections:
    """A text backbone's projections in 4 bits, beside its own, for decoding:
    q|k|v and gate|up of a layer merged, o and down, and the output layer over the
    input embeddings.  `PackedTextDecoder` takes them where a call has at most
    `rows` new rows; longer ones (prompts, camera views) keep the layers' own.

    They stand for the weights at the time of packing.  A backbone whose Linears or
    weights are others since (`holds`), or whose embeddings are
    (`holds_vocabulary`), runs its own until it is packed again.  Weights that
    are written to through `.data` or as inference tensors do not show it."""

    def __init__(self, backbone, *, group=128, rows=NARROW_ROWS):
        def of(*linears):
            return WeightOnlyLinear.from_linear(*linears, group=group)

        self.rows = rows
        self.layers = list(backbone.layers)
        self.sources = []       # (owner, name, module, its class, [(how to get a weight or bias, it, its mark)])
        self.qkv, self.o, self.gate_up, self.down = [], [], [], []
        for layer in backbone.layers:
            attn, mlp = layer.self_attn, layer.mlp
            if mlp.config.hidden_act != "silu":
                raise ValueError("TextProjections needs SiLU text layers")
            self.qkv.append(of(attn.q_proj, attn.k_proj, attn.v_proj))
            self.o.append(of(attn.o_proj))
            self.gate_up.append(of(mlp.gate_proj, mlp.up_proj))
            self.down.append(of(mlp.down_proj))
            self.sources += [(layer, name, module, type(module), None) for name, module in (("self_attn", attn), ("mlp", mlp))]
            for owner, name in [(attn, part + "_proj") for part in "qkvo"] + [(mlp, name) for name, _ in mlp.named_children()]:
                module = getattr(owner, name)
                held = []
                for part in ("weight", "bias"):
                    tensor = getattr(module, part, None)
                    get = partial(module._parameters.get if tensor is module._parameters.get(part) else partial(getattr, module), part, None)
                    held.append((get, tensor, _mark(tensor)))
                self.sources.append((owner, name, module, type(module), held))
        self.embedding = backbone.embed_tokens.weight
        self.vocabulary = WeightOnlyLinear(*quantize_groups(self.embedding, group))
        self.embedding_mark = _mark(self.embedding)

    def holds(self, backbone):
        """Whether the backbone's projections are those that were packed, with
        nothing installed in them."""
        if len(backbone.layers) != len(self.layers) or any(a is not b for a, b in zip(backbone.layers, self.layers)):
            return False
        for owner, name, module, kind, held in self.sources:
            if owner._modules.get(name) is not module or type(module) is not kind:
                return False
            if held is None:    # self_attn, mlp: their hooks run, their own forwards are the caller's matter
                continue
            if "forward" in module.__dict__ or module._forward_hooks or module._forward_pre_hooks:
                return False
            for get, was, mark in held:
                if get() is not was or (was is not None and _mark(was) != mark):
                    return False
        return True

    def holds_vocabulary(self, backbone):
        """The same of the embeddings."""
        weight = backbone.embed_tokens.weight
        return weight is self.embedding and _mark(weight) == self.embedding_mark

    def feed(self, index, x):
        """Layer `index`'s SwiGLU."""
        gate, up = self.gate_up[index](x).chunk(2, dim=-1)
        return self.down[index](F.silu(gate) * up)
