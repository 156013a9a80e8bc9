"""Cases of the prompt-attention and paged K/V-cache operators.

Three operators of a text decoder that serves several robots at once:

* prompt: causal grouped-query attention over a batch of prompts of different
  lengths whose token rows lie one after the other (no padding rows);
* cache: writing the new tokens' keys and values into a paged cache (int8 or
  E4M3 codes with one fp32 scale per token and head, or bf16) and reading a
  sequence's rows back as bf16;
* chunk: attention of the new tokens of each sequence (one token, or a chunk)
  over its pages of that cache.

`run` computes them from elementary torch operations in fp32, or, with `own`
set, by the calls that a program makes of `pir2_b200.ops`.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
FORMATS = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
CODE_BYTES = {"bf16": 2, "int8": 1, "e4m3": 1}
# symmetric-row-v1: scale = max|v| * f32(1 / L), 1 for a row of zeros.
LIMIT = {"int8": 127.0, "e4m3": 448.0}
RECIPROCAL = {form: float(1.0 / torch.tensor(limit)) for form, limit in LIMIT.items()}


def listed():
    return [
        # Instruction texts alone, a few words each: launch latency.
        {"name": "prompt_instruction", "op": "prompt", "batch": 3, "lo": 1, "hi": 40, "heads": 16, "kv_heads": 8,
         "head_dim": 128, "mix": 1},
        # One robot's observation: two camera views of 256 tokens and 32 of text.
        {"name": "prompt_observation", "op": "prompt", "batch": 1, "lo": 544, "hi": 544, "heads": 16, "kv_heads": 8,
         "head_dim": 128, "mix": 2},
        # 64 robots with one to three views and instructions of their own.
        {"name": "prompt_fleet", "op": "prompt", "batch": 64, "lo": 280, "hi": 816, "heads": 16, "kv_heads": 8,
         "head_dim": 128, "mix": 3},
        # A long context of many frames: bound by the matrix products.
        {"name": "prompt_long", "op": "prompt", "batch": 1, "lo": 8192, "hi": 8192, "heads": 16, "kv_heads": 8,
         "head_dim": 128, "mix": 4},
        # Heads of 64 in groups of three, lengths down to none.
        {"name": "prompt_narrow_heads", "op": "prompt", "batch": 12, "lo": 0, "hi": 701, "heads": 12, "kv_heads": 4,
         "head_dim": 64, "mix": 5},
        # One decoding step of eight robots: one row each is written.
        {"name": "cache_step_int8", "op": "cache", "batch": 8, "new_lo": 1, "new_hi": 1, "past_lo": 544, "past_hi": 700,
         "kv_heads": 8, "head_dim": 128, "page": 64, "format": "int8", "mix": 6},
        # The prompts of 64 robots enter an empty cache.
        {"name": "cache_fleet_int8", "op": "cache", "batch": 64, "new_lo": 280, "new_hi": 816, "past_lo": 0,
         "past_hi": 0, "kv_heads": 8, "head_dim": 128, "page": 64, "format": "int8", "mix": 7},
        # Uneven chunks behind uneven histories, small pages, narrow heads.
        {"name": "cache_episode_e4m3", "op": "cache", "batch": 5, "new_lo": 0, "new_hi": 301, "past_lo": 0,
         "past_hi": 1501, "kv_heads": 4, "head_dim": 64, "page": 16, "format": "e4m3", "mix": 8},
        # One robot answers in text, token by token: latency.
        {"name": "chunk_robot_step_int8", "op": "chunk", "batch": 1, "new_lo": 1, "new_hi": 1, "past_lo": 577,
         "past_hi": 577, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "format": "int8", "mix": 9},
        # 64 robots answer, each with a history of its own.
        {"name": "chunk_fleet_step_int8", "op": "chunk", "batch": 64, "new_lo": 1, "new_hi": 1, "past_lo": 500,
         "past_hi": 4001, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "format": "int8", "mix": 10},
        # Four long episodes kept in bf16: few rows over a long axis.
        {"name": "chunk_episode_step_bf16", "op": "chunk", "batch": 4, "new_lo": 1, "new_hi": 1, "past_lo": 29000,
         "past_hi": 32700, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 128, "format": "bf16", "mix": 11},
        # A new camera view of 16 robots joins what they have seen so far.
        {"name": "chunk_view_e4m3", "op": "chunk", "batch": 16, "new_lo": 250, "new_hi": 288, "past_lo": 544,
         "past_hi": 2100, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 32, "format": "e4m3", "mix": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1))))))))


def draw(rng):
    op = rng.choice(["prompt", "cache", "chunk"])
    heads, kv_heads, head_dim = rng.choice(
        [(16, 8, 128), (16, 8, 128), (32, 8, 128), (16, 16, 128), (8, 1, 128), (12, 4, 64), (16, 2, 64), (5, 5, 64)]
    )
    mix = rng.randrange(1 << 20)
    batch = _spread(rng, 1, 64)
    if op == "prompt":
        # At most the listed long prompt's score matrix, and 40000 rows.
        top = min(8192, int(math.sqrt(16 * 8192 * 8192 / (heads * batch))), 40000 // batch)
        hi = _spread(rng, 1, top)
        return {"op": op, "batch": batch, "lo": rng.choice([0, 1, hi // 3, hi]) if batch > 1 else hi, "hi": hi,
                "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "mix": mix}
    form = rng.choice(["int8", "int8", "e4m3", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "cache":
        room = min(4096, 35000 * 8 // (batch * kv_heads))
        new = _spread(rng, 1, min(1024, room))
        past = rng.choice([0, _spread(rng, 1, max(1, room - new))])
        return {"op": op, "batch": batch, "new_lo": rng.choice([0, new]) if batch > 1 else new, "new_hi": new,
                "past_lo": past // 2, "past_hi": past, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
                "format": form, "mix": mix}
    new = rng.choice([1, 1, _spread(rng, 2, 17), _spread(rng, 18, 512)])
    room = min(32000, 120000 * 8 // (batch * max(kv_heads, 4)), int(1e9 / (batch * heads * new)) - new)
    past = _spread(rng, 1, max(1, room))
    return {"op": op, "batch": batch, "new_lo": rng.choice([1, new]), "new_hi": new, "past_lo": past // 2,
            "past_hi": past, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "format": form,
            "mix": mix}


def _lengths(case):
    """(new tokens, tokens after them) of each sequence; the first has the most."""
    rng = random.Random(case["mix"])
    if case["op"] == "prompt":
        new = [case["hi"]] + [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"] - 1)]
        return new, new
    new = [case["new_hi"]] + [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"] - 1)]
    past = [case["past_hi"]] + [rng.randint(case["past_lo"], case["past_hi"]) for _ in range(case["batch"] - 1)]
    return new, [n + p for n, p in zip(new, past)]


def _starts(lengths):
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    return torch.tensor(starts, dtype=torch.int32, device=DEVICE)


def _quantise(x, form):
    """fp32 rows [..., D] -> codes and fp32 scales [...], symmetric-row-v1."""
    if form == "bf16":
        return x.to(torch.bfloat16), None
    most = x.abs().amax(-1)
    scale = torch.where(most == 0, torch.ones_like(most), most * RECIPROCAL[form])
    y = (x / scale[..., None]).clamp(-LIMIT[form], LIMIT[form])
    return (torch.round(y).to(torch.int8) if form == "int8" else y.to(torch.float8_e4m3fn)), scale


def _values(codes, scale):
    return codes.float() if scale is None else codes.float() * scale[..., None]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    new, total = _lengths(case)
    rows = sum(new)
    hk, d = case["kv_heads"], case["head_dim"]
    hq = case.get("heads", 0)
    # Keys keep a gain per channel from their norm's weight: a few are large.
    gain = torch.exp(0.5 * normal(hk, d)) if hq else torch.exp(normal(hk, d))
    # The merged projection's rows: q, k and v are strided views of them.
    qkv = normal(rows, hq + 2 * hk, d)
    qkv[:, hq : hq + hk] *= gain
    qkv = qkv.to(torch.bfloat16)
    state = {
        "op": case["op"],
        "q": qkv[:, :hq],
        "k": qkv[:, hq : hq + hk],
        "v": qkv[:, hq + hk :],
        "starts": _starts(new),
        "longest": max(new),
        "rows": rows,
    }
    if case["op"] == "prompt":
        return state
    page = case["page"]
    counts = [-(-n // page) for n in total]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((case["batch"], max(counts)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at : at + n]
        at += n
    kc, ks = _quantise(normal(pages, hk, page, d) * gain[None, :, None], case["format"])
    vc, vs = _quantise(normal(pages, hk, page, d), case["format"])
    state.update(
        form=case["format"], page=page, k_pages=kc, v_pages=vc, k_scale=ks, v_scale=vs, table=table,
        lengths=torch.tensor(total, dtype=torch.int32, device=DEVICE), reads=_starts(total), read_rows=sum(total),
    )
    if own:
        # The handles that a serving program keeps: checked pointers and sizes of its pool and of a batch.
        from pir2_b200 import kv_cache

        state["pages"] = kv_cache.KVPages(kc, vc, ks, vs)
        state["batch"] = kv_cache.Sequences(state["starts"], state["lengths"], table)
        state["whole"] = kv_cache.Sequences(state["reads"], state["lengths"], table)
    return state


def _rows_of(starts, rows):
    """Sequence and place in it of each packed row."""
    r = torch.arange(rows, device=starts.device)
    seq = (r[:, None] >= starts[1:]).sum(1)
    return seq, r - starts[seq]


def _padded(x, starts, longest):
    """Packed rows [T, ...] -> [B, longest, ...]."""
    at = starts[:-1, None].long() + torch.arange(longest, device=starts.device)
    return x[at.clamp(max=x.shape[0] - 1)]


def _attend(q, k, v, seen):
    """q [B, N, Hq, D], k and v [B, L, Hk, D], seen [B, N, L] -> [B, N, Hq, D], fp32."""
    b, n, hq, d = q.shape
    hk = k.shape[2]
    q = q.view(b, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, hq // hk * n, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)).view(b, hq, n, -1)
    s *= d**-0.5
    s.masked_fill_(~seen[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s -= torch.where(top == -math.inf, torch.zeros_like(top), top)
    s.exp_()
    total = s.sum(-1)
    y = torch.matmul(s.view(b, hk, hq // hk * n, -1), v.permute(0, 2, 1, 3)).view(b, hq, n, d)
    y /= torch.where(total == 0, torch.ones_like(total), total)[..., None]
    return y.permute(0, 2, 1, 3)


def _plain_prompt(s):
    starts, longest = s["starts"], s["longest"]
    q, k, v = (_padded(s[x].float(), starts, longest) for x in "qkv")
    at = torch.arange(longest, device=starts.device)
    n = starts[1:] - starts[:-1]
    seen = (at[None, :] <= at[:, None])[None] & (at < n[:, None])[:, None]
    v = torch.where((at < n[:, None])[..., None, None], v, torch.zeros_like(v))
    y = _attend(q, k, v, seen)
    seq, place = _rows_of(starts, s["rows"])
    return y[seq, place].reshape(s["rows"], -1).to(torch.bfloat16)


def _slots(s, starts, rows, first):
    """Page and place in it of each packed row; `first`: its sequence's first position."""
    seq, place = _rows_of(starts, rows)
    at = first[seq] + place
    return s["table"][seq, at // s["page"]].long(), at % s["page"]


def _plain_cache(s):
    n = s["starts"][1:] - s["starts"][:-1]
    page, place = _slots(s, s["starts"], s["rows"], s["lengths"] - n)
    back_page, back_place = _slots(s, s["reads"], s["read_rows"], torch.zeros_like(s["lengths"]))

    def through(x, pages, scales):
        codes, scale = _quantise(x.float(), s["form"])
        raw = torch.uint8 if s["form"] == "e4m3" else pages.dtype
        pages.view(raw)[page, :, place] = codes.view(raw)
        if scale is not None:
            scales[page, :, place] = scale
        back = pages.view(raw)[back_page, :, back_place].view(pages.dtype)
        return _values(back, None if scale is None else scales[back_page, :, back_place]).to(torch.bfloat16)

    k = through(s["k"], s["k_pages"], s["k_scale"])
    v = through(s["v"], s["v_pages"], s["v_scale"])
    return _cache_outputs(s, k, v)


def _cache_outputs(s, k, v):
    out = {"k": k, "v": v}
    if s["form"] == "bf16":
        out.update(k_pages=s["k_pages"], v_pages=s["v_pages"])
    else:
        out.update(k_scale=s["k_scale"], v_scale=s["v_scale"])
    return out


def _plain_chunk(s):
    lengths, longest = s["lengths"], s["longest"]
    table = s["table"].clamp(min=0).long()
    width = table.shape[1] * s["page"]
    at = torch.arange(width, device=table.device)
    inside = at < lengths[:, None]

    def rows_of(pages, scales):
        raw = torch.uint8 if s["form"] == "e4m3" else pages.dtype
        x = _values(pages.view(raw)[table].view(pages.dtype), None if scales is None else scales[table])
        return x.permute(0, 1, 3, 2, 4).reshape(table.shape[0], width, x.shape[2], x.shape[4])

    k = rows_of(s["k_pages"], s["k_scale"])
    v = rows_of(s["v_pages"], s["v_scale"])
    v = torch.where(inside[..., None, None], v, torch.zeros_like(v))
    n = s["starts"][1:] - s["starts"][:-1]
    last = (lengths - n)[:, None] + torch.arange(longest, device=table.device)
    y = _attend(_padded(s["q"].float(), s["starts"], longest), k, v, (at <= last[..., None]) & inside[:, None])
    seq, place = _rows_of(s["starts"], s["rows"])
    return y[seq, place].reshape(s["rows"], -1).to(torch.bfloat16)


def run(state):
    s = state
    if not own:
        return {"prompt": _plain_prompt, "cache": _plain_cache, "chunk": _plain_chunk}[s["op"]](s)
    from pir2_b200 import ops

    if s["op"] == "prompt":
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["starts"])
    if s["op"] == "cache":
        ops.cache_write(s["k"], s["v"], s["pages"], s["batch"])
        k, v = ops.cache_read(s["pages"], s["whole"], s["read_rows"])
        return _cache_outputs(s, k, v)
    return ops.cache_attention(s["q"], s["pages"], s["batch"])


def work(case):
    new, total = _lengths(case)
    hk, d, hq = case["kv_heads"], case["head_dim"], case.get("heads", 0)
    rows, keys = sum(new), sum(total)
    # Row i of a sequence's n new ones sees the first total - n + i + 1 keys.
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    if case["op"] == "prompt":
        return {"bytes": 2 * rows * d * (2 * hq + 2 * hk) + 4 * (case["batch"] + 1), "flops": 4 * hq * d * pairs}
    per_key = 2 * hk * (d * CODE_BYTES[case["format"]] + (0 if case["format"] == "bf16" else 4))
    table = 4 * sum(-(-t // case["page"]) for t in total) + 4 * (2 * case["batch"] + 1)
    if case["op"] == "cache":
        moved = 2 * 2 * hk * d * rows + per_key * rows + per_key * (keys - rows) + 2 * 2 * hk * d * keys
        return {"bytes": moved + table, "flops": 2 * hk * d * (4 * rows + keys)}
    return {"bytes": 4 * rows * hq * d + per_key * keys + table, "flops": 4 * hq * d * pairs}


def exact(case, seed):
    """The same outputs in fp64, sequence by sequence, from the definitions."""
    s = prepare(case, seed)
    new, total = _lengths(case)
    starts = s["starts"].tolist()
    if case["op"] == "cache":
        return _exact_cache(case, s, new, total, starts)
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(sum(new), hq, d, dtype=torch.float64, device=DEVICE)
    for b, (n, t) in enumerate(zip(new, total)):
        mine = slice(starts[b], starts[b] + n)
        for h in range(hk if n else 0):
            if case["op"] == "prompt":
                k, v = s["k"][mine, h].double(), s["v"][mine, h].double()
            else:
                held = s["table"][b, : -(-t // case["page"])].tolist()
                k = torch.cat([_exact_page(s["k_pages"], s["k_scale"], p, h) for p in held])[:t]
                v = torch.cat([_exact_page(s["v_pages"], s["v_scale"], p, h) for p in held])[:t]
            hidden = torch.ones(n, t, dtype=torch.bool, device=DEVICE).triu(t - n + 1)
            for i in range(h * hq // hk, (h + 1) * hq // hk):
                score = (s["q"][mine, i].double() @ k.T) / math.sqrt(d)
                score[hidden] = -math.inf
                p = torch.softmax(score, dim=1)
                out[mine, i] = p @ v
    return out.view(sum(new), hq * d)


def _exact_page(pages, scales, p, h):
    values = pages[p, h].double()
    return values if scales is None else values * scales[p, h, :, None].double()


def _exact_cache(case, s, new, total, starts):
    form, page = case["format"], case["page"]
    out, back = {}, {"k": [], "v": []}
    pages = {x: s[x + "_pages"].double() for x in "kv"}
    scales = {x: None if form == "bf16" else s[x + "_scale"].double() for x in "kv"}
    for x in "kv":
        for b, (n, t) in enumerate(zip(new, total)):
            rows = s[x][starts[b] : starts[b] + n].double()
            at = torch.arange(t - n, t, device=DEVICE)
            into, place = s["table"][b].long()[at // page] if n else at, at % page
            if n and form != "bf16":
                # The scale is an fp32 number: the row's largest magnitude times the fp32 reciprocal of the limit.
                most = rows.abs().amax(-1)
                scale = (most * RECIPROCAL[form]).float().double()
                scale[most == 0] = 1.0
                rows = rows / scale[..., None]
                if form == "int8":
                    rows = rows.round().clamp(-127, 127)
                else:
                    # E4M3: steps of 2^(e-3) from 2^e on, e at least -6.
                    e = torch.floor(torch.log2(rows.abs().clamp(min=2.0**-6)))
                    rows = (torch.round(rows * 2.0 ** (3 - e)) * 2.0 ** (e - 3)).clamp(-448, 448)
                scales[x][into, :, place] = scale
            if n:
                pages[x][into, :, place] = rows
        for b, t in enumerate(total):
            at = torch.arange(t, device=DEVICE)
            if t:
                of, place = s["table"][b].long()[at // page], at % page
                value = pages[x][of, :, place]
                back[x].append(value if form == "bf16" else value * scales[x][of, :, place][..., None])
        out[x] = torch.cat(back[x])
        out[x + ("_pages" if form == "bf16" else "_scale")] = pages[x] if form == "bf16" else scales[x]
    return out
