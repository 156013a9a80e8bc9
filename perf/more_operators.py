"""Cases of the operators that a text decoder runs for every new token.

* attend4: attention of the new tokens of each sequence over pages that hold
  keys and values in 4 bits: codes of -7..7, two to a byte, an E4M3 factor for
  every 32 of them and a power of two for every row;
* append: per-head norm of q and k, their rotation by the token's position, and
  k and v into the pages of their sequences, in any of the cache's formats;
* weights4: products of a few bf16 rows with weights held in 4 bits, one bf16
  scale for every group of 32, 64 or 128 of an output channel's weights.

`run` computes them from elementary torch operations, or, with `own` set, by
the calls that a program makes of `pir2_b200.ops`.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
FORMATS = ("bf16", "int8", "e4m3", "int4")
# symmetric-row-v1: scale = max|v| * f32(1 / L), 1 for a row of zeros.
LIMIT = {"int8": 127.0, "e4m3": 448.0}
RECIPROCAL = {form: float(1.0 / torch.tensor(limit)) for form, limit in LIMIT.items()}
GROUP = 32          # values of a cached row that share a factor
EPS = 1e-6


def listed():
    return [
        # One robot answers in text, token by token: latency.
        {"name": "attend4_robot_step", "op": "attend4", "batch": 1, "new_lo": 1, "new_hi": 1, "past_lo": 577,
         "past_hi": 577, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "mix": 1},
        # 64 robots answer, each with a history of its own.
        {"name": "attend4_fleet_step", "op": "attend4", "batch": 64, "new_lo": 1, "new_hi": 1, "past_lo": 500,
         "past_hi": 4001, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "mix": 2},
        # Four long episodes: few rows over a long axis.
        {"name": "attend4_episode_step", "op": "attend4", "batch": 4, "new_lo": 1, "new_hi": 1, "past_lo": 29000,
         "past_hi": 32700, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 128, "mix": 3},
        # Narrow heads in groups of three, small pages, a few words each, some with no history.
        {"name": "attend4_narrow_heads", "op": "attend4", "batch": 5, "new_lo": 0, "new_hi": 3, "past_lo": 0,
         "past_hi": 1501, "heads": 12, "kv_heads": 4, "head_dim": 64, "page": 16, "mix": 4},
        # A new camera view of 16 robots joins what they have seen so far.
        {"name": "attend4_view", "op": "attend4", "batch": 16, "new_lo": 250, "new_hi": 288, "past_lo": 544,
         "past_hi": 2100, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 32, "mix": 5},
        # Eight robots decode the first words of an answer: one row each is kept.
        {"name": "append_step_int4", "op": "append", "batch": 8, "new_lo": 1, "new_hi": 1, "past_lo": 20,
         "past_hi": 60, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "format": "int4", "norm": True, "mix": 6},
        # The prompts of 64 robots enter an empty cache.
        {"name": "append_fleet_int4", "op": "append", "batch": 64, "new_lo": 280, "new_hi": 816, "past_lo": 0,
         "past_hi": 0, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "format": "int4", "norm": True, "mix": 7},
        # Uneven chunks behind uneven histories, small pages, narrow heads, a model without head norms.
        {"name": "append_episode_e4m3", "op": "append", "batch": 5, "new_lo": 0, "new_hi": 301, "past_lo": 0,
         "past_hi": 1501, "heads": 12, "kv_heads": 4, "head_dim": 64, "page": 16, "format": "e4m3", "norm": False,
         "mix": 8},
        # The text layers' q|k|v projection of one new token: latency.
        {"name": "weights4_qkv_token", "op": "weights4", "rows": 1, "k": 2048, "n": 4096, "group": 128, "bias": False},
        # Their down projection for eight robots, with a bias.
        {"name": "weights4_down_robots", "op": "weights4", "rows": 8, "k": 6144, "n": 2048, "group": 64, "bias": True},
        # Their gate|up projection for 32 robots, fine groups.
        {"name": "weights4_gate_up_fleet", "op": "weights4", "rows": 32, "k": 2048, "n": 12288, "group": 32, "bias": False},
        # The output layer over the whole vocabulary for four robots.
        {"name": "weights4_vocabulary", "op": "weights4", "rows": 4, "k": 2048, "n": 151936, "group": 128, "bias": False},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1))))))))


def draw(rng):
    op = rng.choice(["attend4", "append", "weights4"])
    mix = rng.randrange(1 << 20)
    if op == "weights4":
        group = rng.choice([32, 64, 128, 128])
        k = group * _spread(rng, max(1, 128 // group), 8192 // group)
        rows = _spread(rng, 1, 64)
        # At most the vocabulary's weights, and the fleet's products.
        n = _spread(rng, 9, min(151936 * 2048 // k, 2 * 151936 * 2048 // (k * rows)))
        return {"op": op, "rows": rows, "k": k, "n": n, "group": group, "bias": rng.random() < 0.5, "mix": mix}
    heads, kv_heads, head_dim = rng.choice(
        [(16, 8, 128), (16, 8, 128), (32, 8, 128), (16, 16, 128), (8, 1, 128), (12, 4, 64), (16, 2, 64), (5, 5, 64)]
    )
    batch = _spread(rng, 1, 64)
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        room = min(4096, 35000 * 16 // (batch * max(kv_heads, heads // 2)))
        new = rng.choice([1, _spread(rng, 1, min(1024, room))])
        past = rng.choice([0, _spread(rng, 1, max(1, room - new))])
        return {"op": op, "batch": batch, "new_lo": rng.choice([0, new]) if batch > 1 else new, "new_hi": new,
                "past_lo": past // 2, "past_hi": past, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "page": page, "format": rng.choice(["int4", "int4", "int8", "e4m3", "bf16"]),
                "norm": rng.random() < 0.7, "mix": mix}
    new = rng.choice([1, 1, _spread(rng, 2, 17), _spread(rng, 18, 512)])
    room = min(32000, 120000 * 8 // (batch * max(kv_heads, 4)), int(1e8 / (batch * heads * new)) - new)
    past = _spread(rng, 1, max(1, room))
    return {"op": op, "batch": batch, "new_lo": rng.choice([1, new]), "new_hi": new, "past_lo": past // 2,
            "past_hi": past, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "mix": mix}


def _lengths(case):
    """(new tokens, tokens after them) of each sequence; the first has the most."""
    rng = random.Random(case["mix"])
    new = [case["new_hi"]] + [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"] - 1)]
    past = [case["past_hi"]] + [rng.randint(case["past_lo"], case["past_hi"]) for _ in range(case["batch"] - 1)]
    return new, [n + p for n, p in zip(new, past)]


def _starts(lengths):
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    return torch.tensor(starts, dtype=torch.int32, device=DEVICE)


def _pack4(codes):
    """int8 codes of -8..7 -> two to a byte, the even one in the low bits."""
    u = codes.to(torch.uint8) & 15
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _unpack4(packed):
    both = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)
    return (both ^ 8).to(torch.int8) - 8


def _quantise(x, form):
    """Rows [..., D] of bf16 values in fp32 -> (codes, fp32 scale of a row, factors of its groups)."""
    if form == "bf16":
        return x.to(torch.bfloat16), None, None
    most = x.abs().amax(-1)
    if form == "int4":
        # Each step is exact up to its rounding: scales are powers of two, and
        # quotients of numbers of 8 and of 4 bits lie off a border or on it.
        power = ((most.view(torch.int32) >> 23) - 10).clamp(min=1)
        scale = torch.where(most == 0, torch.ones_like(most), (power << 23).view(torch.float32))
        y = (x / scale[..., None]).unflatten(-1, (-1, GROUP))
        # (By a tensor: a division by a number is one product with its reciprocal.)
        factor = (y.abs().amax(-1) / torch.full_like(most, 7.0)[..., None]).to(torch.float8_e4m3fn)
        f = factor.float()[..., None]
        codes = torch.round(y / torch.where(f == 0, torch.ones_like(f), f)).clamp(-7, 7)
        codes = torch.where(f == 0, torch.zeros_like(codes), codes)
        return _pack4(codes.flatten(-2).to(torch.int8)), scale, factor
    scale = torch.where(most == 0, torch.ones_like(most), most * RECIPROCAL[form])
    y = (x / scale[..., None]).clamp(-LIMIT[form], LIMIT[form])
    return (torch.round(y).to(torch.int8) if form == "int8" else y.to(torch.float8_e4m3fn)), scale, None


def _values(codes, scale, factor):
    if scale is None:
        return codes.float()
    if factor is not None:
        codes = (_unpack4(codes).float().unflatten(-1, (-1, GROUP)) * factor.float()[..., None]).flatten(-2)
    return codes.float() * scale[..., None]


def _raw(x):
    """fp8 tensors as bytes: torch indexes those."""
    return x.view(torch.uint8) if x is not None and x.dtype == torch.float8_e4m3fn else x


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    if case["op"] == "weights4":
        return _prepare_weights(case, normal)
    new, total = _lengths(case)
    rows, page, batch = sum(new), case["page"], case["batch"]
    hk, d, hq = case["kv_heads"], case["head_dim"], case["heads"]
    form = case.get("format", "int4")
    # Keys keep a gain per channel from their norm's weight: a few are large.
    gain = torch.exp(0.5 * normal(hk, d))
    counts = [-(-n // page) for n in total]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((batch, max(counts)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at : at + n]
        at += n
    held = [_quantise((normal(pages, hk, page, d) * y).to(torch.bfloat16).float(), form) for y in (gain[None, :, None], 1.0)]
    # The merged projection's rows: q, k and v are strided views of them.
    qkv = normal(rows, hq + 2 * hk, d).to(torch.bfloat16)
    state = {"op": case["op"], "form": form, "page": page, "qkv": qkv, "heads": hq, "kv_heads": hk, "table": table,
             "starts": _starts(new), "lengths": torch.tensor(total, dtype=torch.int32, device=DEVICE), "rows": rows,
             "longest": max(new), "reads": _starts(total), "read_rows": sum(total)}
    for x, (codes, scale, factor) in zip("kv", held):
        state.update({x + "_pages": codes, x + "_scale": scale, x + "_factor": factor})
    if case["op"] == "append":
        # The rotation's table, as a decoder makes it once: angles in 64 bits.
        turns = torch.outer(torch.arange(max(total), device=DEVICE, dtype=torch.float64),
                            1e6 ** (-torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d))
        state.update(cos=turns.cos().float(), sin=turns.sin().float())
        weights = [torch.exp(0.3 * normal(d)).to(torch.bfloat16) for _ in range(2)]
        state.update(q_weight=weights[0] if case["norm"] else None, k_weight=weights[1] if case["norm"] else None)
    if own:
        # The handles that a serving program keeps: checked pointers and sizes of its pool and of a batch.
        from pir2_b200 import kv_cache

        state["pages"] = kv_cache.KVPages(
            *(state[x + y] for y in ("_pages", "_scale", "_factor") for x in "kv" if state[x + y] is not None)
        )
        state["batch"] = kv_cache.Sequences(state["starts"], state["lengths"], table)
        state["whole"] = kv_cache.Sequences(state["reads"], state["lengths"], table)
    return state


def _prepare_weights(case, normal):
    m, k, n, group = case["rows"], case["k"], case["n"], case["group"]
    # Weights as a model has them, rounded to the nearest code of their group.
    w = (normal(n, k) * 0.02).unflatten(-1, (-1, group))
    scale = (w.abs().amax(-1) / 7.0).to(torch.bfloat16)
    codes = torch.round(w / scale.float()[..., None]).clamp(-7, 7).to(torch.int8).flatten(-2)
    # Rows as they leave a norm: a few channels are large.
    x = (normal(m, k) * torch.exp(0.5 * normal(k))).to(torch.bfloat16)
    bias = (normal(n) * 0.1).to(torch.bfloat16) if case["bias"] else None
    return {"op": "weights4", "x": x, "packed": _pack4(codes), "scales": scale, "group": group, "bias": bias}


def _plain_weights(s):
    w = _unpack4(s["packed"]).float().unflatten(-1, (-1, s["group"]))
    y = torch.matmul(s["x"].float(), (w * s["scales"].float()[..., None]).flatten(-2).T)
    return (y if s["bias"] is None else y + s["bias"].float()).to(torch.bfloat16)


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


def _plain_attend(s):
    lengths, longest = s["lengths"], s["longest"]
    table = s["table"].clamp(min=0).long()
    width = table.shape[1] * s["page"]
    at = torch.arange(width, device=table.device)
    inside = at < lengths[:, None]

    def rows_of(x):
        y = _values(s[x + "_pages"][table], s[x + "_scale"][table], _raw(s[x + "_factor"])[table].view(torch.float8_e4m3fn))
        return y.permute(0, 1, 3, 2, 4).reshape(table.shape[0], width, y.shape[2], y.shape[4])

    k, v = rows_of("k"), rows_of("v")
    v = torch.where(inside[..., None, None], v, torch.zeros_like(v))
    n = s["starts"][1:] - s["starts"][:-1]
    last = (lengths - n)[:, None] + torch.arange(longest, device=table.device)
    q = _padded(s["qkv"][:, : s["heads"]].float(), s["starts"], longest)
    y = _attend(q, k, v, (at <= last[..., None]) & inside[:, None])
    seq, place = _rows_of(s["starts"], s["rows"])
    return y[seq, place].reshape(s["rows"], -1).to(torch.bfloat16)


def _halves(x):
    a, b = x.chunk(2, -1)
    return a + b


def _normed(x, weight):
    """x / sqrt(mean x^2 + eps) * weight over heads of 64 or 128.  The order of
    the sum is fixed, so that a value next to a border of its code falls on the
    same side wherever it is computed."""
    if weight is None:
        return x
    y = _halves(x * x).unflatten(-1, (-1, 4))
    y = _halves(_halves(_halves((y[..., 0] + y[..., 2]) + (y[..., 1] + y[..., 3]))))
    y = _halves(y) if y.shape[-1] == 2 else y
    return x * (1.0 / torch.sqrt(y / x.shape[-1] + EPS)) * weight.float()


def _turned(x, cos, sin):
    """Rotates the pairs (i, i + D / 2) of [rows, heads, D] by their row's angles."""
    a, b = x.chunk(2, -1)
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _slots(s, starts, rows, first):
    """Page, place in it and position of each packed row; `first`: its sequence's first position."""
    seq, place = _rows_of(starts, rows)
    at = first[seq] + place
    return s["table"][seq, at // s["page"]].long(), at % s["page"], at


def _plain_append(s):
    hq, hk = s["heads"], s["kv_heads"]
    n = s["starts"][1:] - s["starts"][:-1]
    page, place, at = _slots(s, s["starts"], s["rows"], s["lengths"] - n)
    back_page, back_place, _ = _slots(s, s["reads"], s["read_rows"], torch.zeros_like(s["lengths"]))
    x, cos, sin = s["qkv"].float(), s["cos"][at], s["sin"][at]
    q = _turned(_normed(x[:, :hq], s["q_weight"]), cos, sin).to(torch.bfloat16)
    # What is kept is the row as bf16 holds it, in every format.
    k = _turned(_normed(x[:, hq : hq + hk], s["k_weight"]), cos, sin).to(torch.bfloat16)

    def through(x, rows):
        held = [_raw(s[x + y]) for y in ("_pages", "_scale", "_factor")]
        for into, y in zip(held, _quantise(rows.float(), s["form"])):
            if into is not None:
                into[page, :, place] = _raw(y)
        if s["form"] == "bf16":
            return None
        read = [None if y is None else y[back_page, :, back_place] for y in held]
        codes = read[0].view(s[x + "_pages"].dtype)
        factor = None if read[2] is None else read[2].view(torch.float8_e4m3fn)
        return _values(codes, read[1], factor).to(torch.bfloat16)

    return _append_outputs(s, q, through("k", k), through("v", s["qkv"][:, hq + hk :]))


def _append_outputs(s, q, k, v):
    if s["form"] == "bf16":
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    out = {"q": q, "k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if s["form"] == "int4":
        out.update(k_factor=s["k_factor"], v_factor=s["v_factor"])
    return out


def run(state):
    s = state
    if not own:
        return {"attend4": _plain_attend, "append": _plain_append, "weights4": _plain_weights}[s["op"]](s)
    from pir2_b200 import ops

    if s["op"] == "weights4":
        return ops.gemm_w4a16(s["x"], s["packed"], s["scales"], s["bias"])
    if s["op"] == "attend4":
        return ops.cache_attention(s["qkv"][:, : s["heads"]], s["pages"], s["batch"])
    q = ops.cache_append(s["qkv"], s["pages"], s["batch"], s["cos"], s["sin"], q_weight=s["q_weight"],
                         k_weight=s["k_weight"], eps=EPS)
    if s["form"] == "bf16":
        return _append_outputs(s, q, None, None)
    return _append_outputs(s, q, *ops.cache_read(s["pages"], s["whole"], s["read_rows"]))


def work(case):
    if case["op"] == "weights4":
        m, k, n = case["rows"], case["k"], case["n"]
        moved = n * k // 2 + 2 * n * (k // case["group"]) + 2 * m * (k + n) + (2 * n if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * m * n * k}
    new, total = _lengths(case)
    hk, d, hq = case["kv_heads"], case["head_dim"], case["heads"]
    rows, keys = sum(new), sum(total)
    form = case.get("format", "int4")
    row_bytes = {"bf16": 2 * d, "int8": d + 4, "e4m3": d + 4, "int4": d // 2 + d // GROUP + 4}[form]
    per_key = 2 * hk * row_bytes
    table = 4 * sum(-(-t // case["page"]) for t in total) + 4 * (2 * case["batch"] + 1)
    if case["op"] == "append":
        moved = 2 * rows * d * (2 * hq + 2 * hk) + per_key * rows + 4 * d * max(total)
        if form != "bf16":
            moved += per_key * (keys - rows) + 2 * 2 * hk * d * keys
        return {"bytes": moved + table, "flops": d * rows * (8 * (hq + hk) + 4 * 2 * hk) + 2 * hk * d * keys}
    # Row i of a sequence's n new ones sees the first total - n + i + 1 keys.
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    return {"bytes": 4 * rows * hq * d + per_key * keys + table, "flops": 4 * hq * d * pairs}


def exact(case, seed):
    """The same outputs in fp64 from the definitions."""
    s = prepare(case, seed)
    if case["op"] == "weights4":
        low, high = s["packed"].to(torch.int16) % 16, s["packed"].to(torch.int16) // 16
        codes = torch.stack((low, high), dim=2).reshape(case["n"], case["k"])
        codes = torch.where(codes > 7, codes - 16, codes)
        w = codes.double().view(case["n"], -1, case["group"])
        w *= s["scales"].double()[:, :, None]
        y = s["x"].double() @ w.view(case["n"], -1).T
        return y if s["bias"] is None else y + s["bias"].double()
    new, total = _lengths(case)
    starts = s["starts"].tolist()
    if case["op"] == "append":
        return _exact_append(case, s, new, total, starts)
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(sum(new), hq, d, dtype=torch.float64, device=DEVICE)
    pools = [_exact_pool(s, x) for x in "kv"]
    for b, (n, t) in enumerate(zip(new, total)):
        mine = slice(starts[b], starts[b] + n)
        held = s["table"][b, : -(-t // case["page"])].long()
        for h in range(hk if n else 0):
            k, v = (pool[held, h].reshape(-1, d)[:t] for pool in pools)
            hidden = torch.ones(n, t, dtype=torch.bool, device=DEVICE).triu(t - n + 1)
            for i in range(h * hq // hk, (h + 1) * hq // hk):
                score = (s["qkv"][mine, i].double() @ k.T) / math.sqrt(d)
                score[hidden] = -math.inf
                out[mine, i] = torch.softmax(score, dim=1) @ v
    return out.view(sum(new), hq * d)


def _exact_pool(s, x):
    """What a pool's codes stand for, fp64 [pages, heads, page, D]."""
    codes, scale, factor = (s[x + y] for y in ("_pages", "_scale", "_factor"))
    if s["form"] == "int4":
        wide = codes.to(torch.int16)
        values = torch.stack((wide % 16, wide // 16), dim=-1).flatten(-2)
        values = torch.where(values > 7, values - 16, values).double()
        values = values * factor.double().repeat_interleave(GROUP, dim=-1)
    else:
        values = codes.double()
    return values if scale is None else values * scale.double()[..., None]


def _power(e):
    """2^e in fp64, e whole."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_e4m3(y):
    """The nearest E4M3 number: steps of 2^(e-3) from 2^e on, e at least -6, at most 448."""
    e = torch.frexp(y.abs().clamp(min=2.0**-6)).exponent - 1
    return (torch.round(y * _power(3 - e)) * _power(e - 3)).clamp(-448, 448)


def _exact_rows(rows, form):
    """(what a row's codes stand for without its scale, scale, factors)."""
    most = rows.abs().amax(-1)
    if form == "int4":
        scale = _power((torch.frexp(most).exponent - 11).clamp(min=-126))
        scale[most == 0] = 1.0
        y = rows / scale[..., None]
        f = _exact_e4m3(y.view(*y.shape[:-1], -1, GROUP).abs().amax(-1) / 7)
        wide = f.repeat_interleave(GROUP, dim=-1)
        codes = (y / wide).round().clamp(-7, 7)
        codes[wide == 0] = 0
        return codes * wide, scale, f
    # The scale is an fp32 number: the row's largest magnitude times the fp32 reciprocal of the limit.
    scale = (most * RECIPROCAL[form]).float().double()
    scale[most == 0] = 1.0
    y = rows / scale[..., None]
    return (y.round().clamp(-127, 127) if form == "int8" else _exact_e4m3(y)), scale, None


def _exact_append(case, s, new, total, starts):
    form, page, hq, hk = case["format"], case["page"], case["heads"], case["kv_heads"]
    x = s["qkv"].double()
    at = torch.cat([torch.arange(t - n, t, device=DEVICE) for n, t in zip(new, total)])
    angle = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None]

    def turned(x, weight):
        if weight is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.double()
        half = x.shape[-1] // 2
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * angle
        return torch.cat((z.real, z.imag), dim=-1)

    out = {"q": turned(x[:, :hq], s["q_weight"])}
    rows = {"k": turned(x[:, hq : hq + hk], s["k_weight"]), "v": x[:, hq + hk :]}
    for name in "kv":
        if form == "bf16":
            pool = s[name + "_pages"].double()
            codes = rows[name]
        else:
            pool = _exact_pool(s, name)
            # A cached row is that of bf16 numbers.
            codes, scale, factor = _exact_rows(rows[name].to(torch.bfloat16).double(), form)
            scales = s[name + "_scale"].double()
            factors = None if factor is None else s[name + "_factor"].double()
        back = []
        for b, (n, t) in enumerate(zip(new, total)):
            p = torch.arange(t - n, t, device=DEVICE)
            into, place, mine = s["table"][b].long()[p // page], p % page, slice(starts[b], starts[b] + n)
            pool[into, :, place] = codes[mine] if form == "bf16" else codes[mine] * scale[mine][..., None]
            if form != "bf16":
                scales[into, :, place] = scale[mine]
            if form == "int4":
                factors[into, :, place] = factor[mine]
            p = torch.arange(t, device=DEVICE)
            back.append(pool[s["table"][b].long()[p // page], :, p % page])
        if form == "bf16":
            out[name + "_pages"] = pool
        else:
            out[name], out[name + "_scale"] = torch.cat(back), scales
        if form == "int4":
            out[name + "_factor"] = factors
    return out
