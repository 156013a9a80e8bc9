"""Plain fp64 forms of the ragged-batch operators, sequence by sequence, for
their tests."""

import torch

INT8_LIMIT, E4M3_LIMIT = 127.0, 448.0


def starts_of(lengths, device="cuda", first=0):
    total = [first]
    for n in lengths:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device=device)


def attend(q, k, v, scale):
    """q [n, hq, D], k and v [L, hk, D] (any float type): fp64 output [n, hq,
    D] and sum_j p_j |v_j| / sum_j p_j, row i seeing keys 0 .. L - n + i.
    Each row is summed over the keys that it sees and no others."""
    n, hq, d = q.shape
    length, hk = k.shape[0], k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    kk = k.repeat_interleave(hq // hk, dim=1)
    vv = v.repeat_interleave(hq // hk, dim=1)
    score = torch.einsum("ihd,jhd->hij", q, torch.nan_to_num(kk, nan=0.0, posinf=0.0, neginf=0.0)) * scale
    bad = (~torch.isfinite(kk)).any(-1).T[:, None, :]
    seen = (torch.arange(length, device=q.device)[None, :] <= (torch.arange(n, device=q.device) + length - n)[:, None])[None]
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True) if length else torch.zeros(hq, n, 1, dtype=torch.float64, device=q.device)
    p = torch.where(seen, torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top)), torch.zeros_like(score))
    total = p.sum(-1, keepdim=True)
    w = p / torch.where(total == 0, torch.ones_like(total), total)
    finite = torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)
    out = torch.einsum("hij,jhd->ihd", w, finite)
    mass = torch.einsum("hij,jhd->ihd", w, finite.abs())
    # Rows that see a key or value that is not finite are not compared.
    spoiled = (seen & bad).any(-1).T[..., None] | torch.einsum(
        "hij,jhd->ihd", seen.double().expand(hq, n, length).contiguous(), (~torch.isfinite(vv)).double()
    ).bool()
    return out, mass, spoiled


def tolerance(out, mass):
    """Each weight is rounded to bf16 (half a unit in the last place, 2^-8 of
    it) and so may be the sum that divides them: 2^-7 of sum_j w_j |v_j|; the
    output is rounded to bf16 once more.  fp32 products and sums of at most
    2^16 terms and exp2 add less than 2^-12."""
    return (2.0**-7 + 2.0**-12) * mass + 2.0**-8 * out.abs() + 1e-30


def quantise(x, dtype):
    """symmetric-row-v1 per row of the last dimension, in fp32 as defined:
    (codes, scale).  A row with a NaN: codes of 0, the NaN as its scale."""
    x = x.float()
    if dtype == torch.bfloat16:
        return x.to(torch.bfloat16), None
    limit = INT8_LIMIT if dtype == torch.int8 else E4M3_LIMIT
    most = torch.where(torch.isinf(x), torch.zeros_like(x), x.abs()).amax(-1)
    scale = torch.where(most == 0, torch.ones_like(most), most * float(1.0 / torch.tensor(limit)))
    y = torch.nan_to_num(x / scale[..., None], nan=0.0).clamp(-limit, limit)
    if dtype == torch.int8:
        return torch.round(y).to(torch.int8), scale
    return y.to(torch.float8_e4m3fn), scale


def values(codes, scale):
    return codes.float() if scale is None else codes.float() * scale[..., None]


def make_pool(total, hk, d, page, dtype, seed, *, poison=True, spare=3):
    """Pages for sequences of `total` tokens, in a random order, holding random
    rows: (k, v, k_scale, v_scale, table, rows) with rows[b] the (k, v) values
    [total_b, hk, d] in fp32.  With `poison`, everything that no sequence owns
    (unused pages, the rest of last pages) is NaN where the format has one."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    counts = [-(-t // page) for t in total]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    width = max(max(counts), 1)
    table = torch.full((len(total), width), -7, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at : at + n]
        at += n
    raw = [torch.randn(pages, hk, page, d, generator=g, device="cuda") for _ in range(2)]
    raw[0] *= torch.exp(0.5 * torch.randn(hk, 1, d, generator=g, device="cuda"))
    (kc, ks), (vc, vs) = (quantise(x, dtype) for x in raw)
    owned = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    rows = []
    for b, t in enumerate(total):
        ids = table[b, : counts[b]].long()
        for i in range(counts[b]):
            owned[ids[i], : min(page, t - i * page)] = True
        rows.append(tuple(
            values(c[ids] if dtype != torch.float8_e4m3fn else c.view(torch.uint8)[ids].view(dtype), None if s is None else s[ids])
            .permute(0, 2, 1, 3).reshape(counts[b] * page, hk, d)[:t]
            for c, s in ((kc, ks), (vc, vs))
        ))
    if poison:
        lost = ~owned[:, None, :].expand(pages, hk, page)
        for c, s in ((kc, ks), (vc, vs)):
            if dtype == torch.bfloat16:
                c[lost] = float("nan")
            else:
                s[lost] = float("nan")
                if dtype == torch.float8_e4m3fn:
                    c.view(torch.uint8)[lost] = 0x7F
    return kc, vc, ks, vs, table, rows
