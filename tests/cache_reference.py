"""The 4-bit cache and attention over it in 64 bits, written from the definition (no code of the operators)."""
import math

import torch


def bf16_beside(x, up):
    """The nearest bf16 number not below (up) or not above x, as f64; x f64."""
    r = x.to(torch.bfloat16)
    other = torch.nextafter(r, torch.full_like(r, math.inf if up else -math.inf))
    return torch.where((r.double() < x) if up else (r.double() > x), other, r).double()


def quantized(x):
    """(codes, step, least) of rows [..., dim], f64; the 32-bit steps of the definition are rounded as it says."""
    x = x.double()
    least = bf16_beside(x.amin(-1, keepdim=True), False)
    step = bf16_beside(((x.amax(-1, keepdim=True) - least).float().double() / 15).float().double(), True).clamp_min(2.0 ** -100)
    code = ((x - least).float().double() * (1 / step).float().double()).float().double().round().clamp(0, 15)
    bad = ~(torch.isfinite(least) & torch.isfinite(step) & torch.isfinite(x.amax(-1, keepdim=True)))
    nan = torch.full_like(least, math.nan)
    return torch.where(bad, torch.zeros_like(code), code), torch.where(bad, nan, step), torch.where(bad, nan, least)


def rows_of(codes, scale):
    """(codes, step, least) f64 of a cache's bytes and pairs."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    return c, scale[..., :1].double(), scale[..., 1:].double()


def gathered(cache, table, length, page):
    """(codes, step, least) of the keys and of the values at positions 0 .. length - 1: [length, heads, ...] each, and which
    positions have a page."""
    out = []
    pos = torch.arange(length, device=table.device)
    slot = pos // page
    ok = slot < table.numel()
    name = table.long()[slot.clamp_max(max(0, table.numel() - 1))] if table.numel() else torch.full_like(pos, -1)
    ok &= (name >= 0) & (name < cache[0].shape[0])
    name = torch.where(ok, name, torch.zeros_like(name))
    for i in (0, 2):
        out.append(rows_of(cache[i][name, :, pos % page], cache[i + 1][name, :, pos % page]))
    return out[0], out[1], ok


def attention(q, cache, table, lengths, starts, scale, out):
    """(y, bound) f64 like q: what attention gives, and how far a correct kernel may be off; rows of no sequence are out's.

    The bound counts, beside the output's own rounding: p times step rounded to f16 (half a step, 2^-11, of each term, all of one
    sign), f32 sums (a rounding of 2^-23, or a cut of as much, per addition; 16 tokens an addition), and scores that are off by
    delta (sums of dim products and a few more roundings), which moves p by a factor of 1 +- 2 delta."""
    tokens, heads, dim = q.shape
    page, kv = cache[0].shape[2], cache[0].shape[1]
    per = heads // kv
    y, bound = out.double().clone(), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    half = torch.finfo(q.dtype).eps / 2
    for b in range(table.shape[0]):
        beg, end = (b, b + 1) if starts is None else (int(starts[b]), int(starts[b + 1]))
        n, length = end - beg, int(lengths[b])
        if n <= 0:
            continue
        have = max(0, min(length, table.shape[1] * page))
        (kc, ks, kl), (vc, vs, vl), ok = gathered(cache, table[b], have, page)
        last = torch.arange(length - n, length, device=q.device)
        seen = (torch.arange(have, device=q.device)[None] <= last[:, None]) & ok[None]     # [n, have]
        for h in range(kv):
            x = q[beg:end, h * per:(h + 1) * per].double()
            # a row that is not seen may hold anything: its place is taken by zeros
            some = seen.any(0)[:, None]
            step, least, codes = (torch.where(some, v[:, h], torch.zeros_like(v[:, h])) for v in (ks, kl, kc))
            z = torch.einsum("npd,jd->npj", x, codes * step + least) * scale
            z = z.masked_fill(~seen[:, None], -math.inf)
            size = torch.einsum("npd,jd->npj", x.abs(), codes * step.abs() + least.abs()) * abs(scale)
            delta = ((dim + 16) * 2.0 ** -23 * size).masked_fill(~seen[:, None], 0).amax(-1, keepdim=True) if have else torch.zeros(n, per, 1, dtype=torch.float64, device=q.device)
            top = z.amax(-1, keepdim=True) if have else torch.zeros(n, per, 1, dtype=torch.float64, device=q.device)
            p = torch.where(seen[:, None], torch.exp(z - top), torch.zeros_like(z))
            p = torch.where(p.sum(-1, keepdim=True) == 0, torch.zeros_like(p), p / p.sum(-1, keepdim=True))
            step, least, codes = (torch.where(some, v[:, h], torch.zeros_like(v[:, h])) for v in (vs, vl, vc))
            got = torch.einsum("npj,jd->npd", p, codes * step + least)
            grain = torch.einsum("npj,jd->npd", p, codes * step)
            full = torch.einsum("npj,jd->npd", p, codes * step + least.abs())
            y[beg:end, h * per:(h + 1) * per] = got
            adds = have / 16 + 64
            bound[beg:end, h * per:(h + 1) * per] = (half * 1.01 * got.abs() + 2.0 ** -11 * grain + (adds * 2.0 ** -22 + 2.5 * delta) * full)
    smallest = 2.0 ** -24 if q.dtype == torch.float16 else 2.0 ** -126
    return y, bound + smallest
