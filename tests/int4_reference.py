"""Plain forms of the 4-bit cache format, for its tests."""

import torch

GROUP = 32


def pack(codes):
    """Codes of -8..7 -> bytes, the even one in the low bits."""
    u = codes.to(torch.int16) & 15
    return (u[..., 0::2] | (u[..., 1::2] << 4)).to(torch.uint8)


def unpack(packed):
    p = packed.to(torch.int16)
    u = torch.stack((p & 15, p >> 4), dim=-1).flatten(-2)
    return torch.where(u > 7, u - 16, u)


def quantise4(x):
    """Rows [..., D] of bf16 values -> (bytes [..., D / 2], fp32 scale [...],
    E4M3 factors [..., D / 32]), in fp64 from the definition."""
    x = x.double()
    lost = torch.isnan(x).any(-1)
    most = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    x = torch.where(torch.isinf(x), torch.sign(x) * most[..., None], x)
    x = torch.where(lost[..., None], torch.zeros_like(x), x)
    power = (torch.frexp(most).exponent.long() - 11).clamp(min=-126)
    scale = torch.where(most == 0, torch.ones_like(most), ((power + 1023) << 52).view(torch.float64))
    y = (x / scale[..., None]).unflatten(-1, (-1, GROUP))
    factor = (y.abs().amax(-1) / torch.full_like(most, 7.0)[..., None]).float().to(torch.float8_e4m3fn)
    f = factor.double()[..., None]
    codes = torch.round(y / torch.where(f == 0, torch.ones_like(f), f)).clamp(-7, 7)
    codes = torch.where(f == 0, torch.zeros_like(codes), codes).flatten(-2)
    scale = torch.where(lost, torch.full_like(scale, float("nan")), scale)
    return pack(codes), scale.float(), factor


def values4(packed, scale, factor):
    """fp64 values of the codes."""
    v = unpack(packed).double().unflatten(-1, (-1, GROUP)) * factor.double()[..., None]
    return v.flatten(-2) * scale.double()[..., None]


def make_pool4(total, hk, d, page, seed, *, poison=True, spare=3):
    """As ragged_reference.make_pool: (k, v, k_scale, v_scale, k_factor,
    v_factor), table, rows [(k, v) values of each sequence].  With `poison`,
    what no sequence owns is any code, a NaN factor and a NaN scale."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    counts = [-(-t // page) for t in total]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(total), max(max(counts), 1)), -7, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at : at + n]
        at += n
    raw = [torch.randn(pages, hk, page, d, generator=g, device="cuda") for _ in range(2)]
    raw[0] *= torch.exp(0.5 * torch.randn(hk, 1, d, generator=g, device="cuda"))
    (kc, ks, kf), (vc, vs, vf) = (quantise4(x.to(torch.bfloat16)) for x in raw)
    owned = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    whole = [values4(c, s, f) for c, s, f in ((kc, ks, kf), (vc, vs, vf))]
    rows = []
    for b, t in enumerate(total):
        ids = table[b, : counts[b]].long()
        for i in range(counts[b]):
            owned[ids[i], : min(page, t - i * page)] = True
        rows.append(tuple(w[ids].permute(0, 2, 1, 3).reshape(counts[b] * page, hk, d)[:t] for w in whole))
    if poison:
        lost = ~owned[:, None, :].expand(pages, hk, page)
        for c, s, f in ((kc, ks, kf), (vc, vs, vf)):
            c[lost] = torch.randint(0, 256, c[lost].shape, generator=g, device="cuda", dtype=torch.uint8)
            s[lost] = float("nan")
            f.view(torch.uint8)[lost] = 0x7F
    return (kc, vc, ks, vs, kf, vf), table, rows
