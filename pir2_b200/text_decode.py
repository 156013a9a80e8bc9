"""The VLM text decoder over packed prompts and a paged K/V cache.

piR2 runs the decoder once per observation, one prompt length per batch
(coexecution/optimization/groot/vlm.py:312-313).  `PackedTextDecoder` runs the
same layers for several robots at once: prompts of different lengths lie one
after the other in one row of tokens, each layer's keys and values enter a
paged cache as they are computed, and later calls give each sequence more
tokens, one or many (a new camera view, a decoded word).  The projections stay
whatever is installed in the layers: bf16 Linears, or the quantized ones and
their grouped q|k|v GEMM when a TransformerINT controller is passed.

`TextCache` owns the pools of all layers and deals pages to sequences on the
host; a batch's index tensors are rewritten in place by every `extend`.
"""

import threading
from contextlib import contextmanager
from functools import partial

import torch

from . import ops
from .kv_cache import FACTOR_GROUP, KVPages, Sequences, rotary_table
from .transformer import _MODE_BITS


class TextCache:
    """Pools of `layers` layers in one allocation ([pages, layers, 2, kv_heads,
    page_size, head_dim]; dtype uint8: two 4-bit codes to a byte) and the pages of up to `batch` sequences of at most
    `max_tokens` tokens."""

    def __init__(self, layers, pages, kv_heads, head_dim, *, batch, max_tokens, page_size=64, dtype=torch.int8, device="cuda"):
        packed = dtype == torch.uint8
        shape = (pages, layers, 2, kv_heads, page_size, head_dim // 2 if packed else head_dim)
        self.codes = torch.zeros(shape, dtype=dtype, device=device)
        self.scales = None if dtype == torch.bfloat16 else torch.ones(shape[:-1], dtype=torch.float32, device=device)
        groups = (*shape[:-1], head_dim // FACTOR_GROUP)
        self.factors = torch.zeros(groups, dtype=torch.float8_e4m3fn, device=device) if packed else None
        self.layers = [
            KVPages(*(t[:, i, which] for t in (self.codes, self.scales, self.factors) if t is not None for which in (0, 1)))
            for i in range(layers)
        ]
        self.page_size, self.batch = page_size, batch
        self.free = list(range(pages - 1, -1, -1))
        self.held = [[] for _ in range(batch)]      # pages of each sequence
        self.tokens = [0] * batch
        self.table_host = torch.zeros(batch, max(1, -(-max_tokens // page_size)), dtype=torch.int32)
        self.table = self.table_host.to(device)
        self.starts = torch.zeros(batch + 1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.sequences = Sequences(self.starts, self.lengths, self.table)

    def extend(self, new):
        """Makes room for new[b] more tokens of sequence b and describes that
        batch in `sequences`.  Nothing changes when the pages do not suffice."""
        if len(new) != self.batch or any(n < 0 for n in new):
            raise ValueError("extend: one count of new tokens, at least 0, per sequence")
        wanted = [-(-(t + n) // self.page_size) - len(h) for t, n, h in zip(self.tokens, new, self.held)]
        if any(-(-(t + n) // self.page_size) > self.table.shape[1] for t, n in zip(self.tokens, new)):
            raise ValueError("extend: a sequence would pass max_tokens")
        if sum(wanted) > len(self.free):
            raise ValueError(f"extend: {sum(wanted)} pages wanted, {len(self.free)} free")
        starts = [0]
        for b, n in enumerate(new):
            for _ in range(wanted[b]):
                self.table_host[b, len(self.held[b])] = self.free[-1]
                self.held[b].append(self.free.pop())
            self.tokens[b] += n
            starts.append(starts[-1] + n)
        if sum(wanted):
            self.table.copy_(self.table_host)
        self.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        self.lengths.copy_(torch.tensor(self.tokens, dtype=torch.int32))
        return self.sequences

    def rewind(self, tokens):
        """Back to `tokens` of each sequence, at most those it has: the later
        ones are forgotten and their pages free."""
        if len(tokens) != self.batch or any(not 0 <= n <= t for n, t in zip(tokens, self.tokens)):
            raise ValueError("rewind: one count per sequence, at most its tokens")
        for b in range(self.batch - 1, -1, -1):
            while len(self.held[b]) > -(-tokens[b] // self.page_size):
                self.free.append(self.held[b].pop())
            self.tokens[b] = tokens[b]

    def release(self, b):
        """Sequence b ends: its pages are free again."""
        self.free.extend(reversed(self.held[b]))
        self.held[b], self.tokens[b] = [], 0


class _Routes:
    """Which forward of an attention module a thread calls.  The layers call
    their attention themselves, so a run puts its own forward in the place of the
    module's; a backbone may be shared by decoders and plain calls of several
    threads, each of which must get its own."""

    def __init__(self):
        self.lock = threading.Lock()
        self.modules = {}       # id -> (its own instance attribute or None, {thread: forward})

    @staticmethod
    def _by_thread(mine, plain):
        return lambda *args, **kwargs: mine.get(threading.get_ident(), plain)(*args, **kwargs)

    def installed(self, module):
        """The module's own instance attribute, whichever runs there are."""
        with self.lock:
            routed = self.modules.get(id(module))
            return module.__dict__.get("forward") if routed is None else routed[0]

    @contextmanager
    def routed(self, modules, forwards):
        """In this thread, and within the block, module i's forward is
        forwards[i]."""
        thread = threading.get_ident()
        with self.lock:
            for module, forward in zip(modules, forwards):
                if id(module) not in self.modules:
                    own, mine = module.__dict__.get("forward"), {}
                    module.forward = self._by_thread(mine, module.forward)
                    self.modules[id(module)] = own, mine
                self.modules[id(module)][1][thread] = forward
        try:
            yield
        finally:
            with self.lock:
                for module in modules:
                    own, mine = self.modules[id(module)]
                    del mine[thread]
                    if mine:
                        continue
                    del self.modules[id(module)]
                    if own is None:
                        module.__dict__.pop("forward", None)
                    else:
                        module.forward = own


_ROUTES = _Routes()


class PackedTextDecoder:
    """Runs a text backbone's layers (Qwen3-VL attention: q/k norm, RoPE,
    grouped heads of 128) on packed rows over a TextCache.  With a TransformerINT
    `controller`, q, k and v are one grouped GEMM of the precision that it has
    installed at the time of a call (only of `bits`, if given).

    `append`: norm, rotation and cache write of a layer are one launch
    (`ops.cache_append`), in fp32 with one rounding, where the layers' own
    arithmetic rounds each step to bf16: results differ in the last bits.
    `weight_only` (weight_only.TextProjections, packed from this backbone): the
    projections, SwiGLU and output layer of calls with few rows, in 4-bit weights.
    While anything is installed in a layer's projections, MLP, norms or the layer
    itself (quantised projections, fusions, hooks), or their weights are not those
    that were packed, all layers and the output layer run as they are; the output
    layer alone does while the embeddings are not those that were packed."""

    def __init__(self, backbone, cache, *, controller=None, bits=None, append=False, weight_only=None):
        self.backbone, self.cache, self.controller = backbone, cache, controller
        self.append, self.weight_only = append, weight_only
        self.attentions = [layer.self_attn for layer in backbone.layers]
        if len(self.attentions) != len(cache.layers):
            raise ValueError("the cache must have one pool per layer")
        if any(attn.head_dim != 128 for attn in self.attentions):
            raise ValueError("PackedTextDecoder needs heads of 128")
        self.groups = {}          # (bits, attention) -> its q|k|v group
        if controller is not None:
            names = {id(site[0]): name for name, site in controller.sites.items()}
            for precision in (8, 4) if bits is None else (bits,):
                grouped = {members[0]: group for members, group in controller.grouped[precision] if len(members) == 3}
                for attn in self.attentions:
                    group = grouped.get(names.get(id(attn.q_proj)))
                    if group is not None:
                        self.groups[precision, id(attn)] = group
        if weight_only is not None and len(weight_only.qkv) != len(self.attentions):
            raise ValueError("weight_only must have the backbone's layers")
        if weight_only is not None and any(a is not b for a, b in zip(weight_only.layers, backbone.layers)):
            raise ValueError("weight_only must be packed from the backbone's layers")
        self.rope = self.turns = None

    def _narrow(self, rows):
        """Whether the 4-bit projections take a call of so many rows."""
        if self.weight_only is None or rows > self.weight_only.rows or not self.weight_only.holds(self.backbone):
            return False
        return not any(
            "forward" in module.__dict__ for layer in self.backbone.layers
            for module in (layer, layer.input_layernorm, layer.post_attention_layernorm)
        ) and all(_ROUTES.installed(layer.mlp) is None for layer in self.backbone.layers)

    def _project(self, attn, x):
        mode = None if self.controller is None else self.controller.mode
        group = self.groups.get((_MODE_BITS.get(mode), id(attn)))
        if group is not None:
            return group.linear(x)
        return torch.cat((attn.q_proj(x), attn.k_proj(x), attn.v_proj(x)), dim=-1)

    def _attend(self, index, prompts, narrow, x, cos, sin):
        attn, pages, sequences = self.attentions[index], self.cache.layers[index], self.cache.sequences
        rows = x.shape[1]
        qkv = self.weight_only.qkv[index](x) if narrow else self._project(attn, x)
        if self.append:
            qkv = qkv.reshape(rows, -1, attn.head_dim)
            v = qkv[:, attn.heads + attn.kv_heads :]
            k = v.new_empty((rows, attn.kv_heads, attn.head_dim)) if prompts else None
            q = ops.cache_append(qkv, pages, sequences, *self.turns, q_weight=attn.q_norm.weight, k_weight=attn.k_norm.weight,
                                 eps=attn.q_norm.variance_epsilon, k_out=k)
        else:
            q, k, v = ops.qk_norm_rope(
                qkv.reshape(rows, qkv.shape[-1]), attn.q_norm.weight, attn.k_norm.weight, cos, sin, tokens=rows,
                hq=attn.heads, hk=attn.kv_heads, eps=attn.q_norm.variance_epsilon,
            )
            q, k, v = (z[0].transpose(0, 1) for z in (q, k, v))        # [rows, heads, 128] views
            ops.cache_write(k, v, pages, sequences)
        if prompts:
            y = ops.prompt_attention(q, k, v, sequences.starts)
        else:
            y = ops.cache_attention(q, pages, sequences)
        y = y.view(1, rows, y.shape[1])
        return self.weight_only.o[index](y) if narrow else attn.o_proj(y)

    def _rope(self, positions, device, dtype):
        longest = max(positions) + 1
        if self.rope is None or self.rope[0].shape[0] < longest:
            # Grown by doubling: angles of a position do not depend on the rest.
            size = max(longest, 2 * (0 if self.rope is None else self.rope[0].shape[0]))
            c = self.backbone.config
            inv = 1.0 / (c.rope_theta ** (torch.arange(0, c.head_dim, 2, device=device, dtype=torch.float32) / c.head_dim))
            angles = torch.outer(torch.arange(size, device=device, dtype=torch.float32), inv)
            angles = torch.cat((angles, angles), dim=-1)
            self.rope = angles.cos().to(dtype), angles.sin().to(dtype)
        at = torch.tensor(positions, dtype=torch.int64).to(device)
        return self.rope[0][at], self.rope[1][at]

    def _turns(self, longest, device):
        if self.turns is None or self.turns[0].shape[0] < longest:
            size = max(longest, 2 * (0 if self.turns is None else self.turns[0].shape[0]))
            c = self.backbone.config
            self.turns = rotary_table(size, c.head_dim, c.rope_theta, device=device)

    @torch.inference_mode()
    def run(self, hidden, new):
        """hidden: [rows, hidden] embeddings of the sequences' next tokens, one
        sequence after the other, new[b] of them for sequence b.  Returns the
        last layer's [rows, hidden].  Where a layer raises, the cache is as it
        was before the call."""
        return self._run(hidden, new, self._narrow(hidden.shape[0]))

    def _run(self, hidden, new, narrow):
        if hidden.ndim != 2 or hidden.shape[0] != sum(new):
            raise ValueError("run: hidden must hold the new tokens' rows")
        past = list(self.cache.tokens)
        try:
            self.cache.extend(new)
            return self._layers(hidden, past, new, narrow) if hidden.shape[0] else hidden
        except BaseException:
            self.cache.rewind(past)      # rows that no layer may have written
            raise

    def _layers(self, hidden, past, new, narrow):
        prompts = all(p == 0 for p, n in zip(past, new) if n)   # every sequence of the batch starts with this call
        if self.append:
            cos = sin = None                                     # positions are looked up on the device
            self._turns(max(p + n for p, n in zip(past, new)), hidden.device)
        else:
            positions = [p + i for p, n in zip(past, new) for i in range(n)]
            cos, sin = self._rope(positions, hidden.device, hidden.dtype)
        modules = list(self.attentions)
        forwards = [partial(self._attend, index, prompts, narrow) for index in range(len(self.attentions))]
        if narrow:
            modules += [layer.mlp for layer in self.backbone.layers]
            forwards += [partial(self.weight_only.feed, index) for index in range(len(self.attentions))]
        h = hidden[None]
        with _ROUTES.routed(modules, forwards):
            for layer in self.backbone.layers:
                h = layer(h, cos, sin)
        return h[0]

    @torch.inference_mode()
    def decode(self, last_hidden, steps):
        """Greedy decoding with the input embeddings as the output layer:
        last_hidden [batch, hidden] is each sequence's newest row; returns token
        ids [batch, steps]."""
        embed = self.backbone.embed_tokens.weight
        tokens = []
        for _ in range(steps):
            narrow = self._narrow(last_hidden.shape[0])      # of the whole step
            packed = narrow and self.weight_only.holds_vocabulary(self.backbone)
            logits = self.weight_only.vocabulary(last_hidden) if packed else last_hidden @ embed.T
            ids = logits.argmax(-1)
            tokens.append(ids)
            last_hidden = self._run(embed[ids], [1] * self.cache.batch, narrow)
        return torch.stack(tokens, dim=1)
