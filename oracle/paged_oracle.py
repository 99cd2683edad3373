"""Norm and rotation of heads, the paged cache and attention over it, in float64 (test infrastructure): the definitions, one token at a time where that is
plainest.  Works on torch tensors of any device."""
import math

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def rotate(x, positions, frequencies=None, layout="half", magnitude=1.0, weight=None, eps=1e-6):
    """x [..., d] float64, positions broadcastable to x[..., 0]; differentiable."""
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    if frequencies is None:
        return x
    n = frequencies.numel()
    angle = positions.double()[..., None] * frequencies
    cos, sin = angle.cos() * magnitude, angle.sin() * magnitude
    one = torch.arange(n) if layout == "half" else 2 * torch.arange(n)
    two = one + n if layout == "half" else one + 1
    a, b = x[..., one], x[..., two]
    out = x.clone()
    out[..., one] = a * cos - b * sin
    out[..., two] = b * cos + a * sin
    return out


def to_4bit(x):
    """(values, bytes of the powers of two) of float64 x [..., d]: of every 32 the smallest power of two with which the largest is at most 6, the nearest
    e2m1 values, ties to the even code.  By comparison with every value there is."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    top = g.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, 126)
    for k in range(125, -128, -1):
        e = torch.where(top <= 6 * 2.0 ** k, torch.full_like(e, k), e)
    y = (g.abs() / torch.exp2(e)).clamp(max=6)
    table = E2M1.to(x)
    far = (y[..., None] - table).abs()
    near = far == far.amin(-1, keepdim=True)                   # one value, or the two that y lies between
    even = torch.arange(8, device=x.device) % 2 == 0
    code = torch.where(near & (even | (near.sum(-1, keepdim=True) == 1)), torch.arange(8, device=x.device), -1).amax(-1)
    v = table[code] * torch.exp2(e) * torch.where(g < 0, -1.0, 1.0)
    v = torch.where(torch.isnan(top), torch.nan, v)
    byte = torch.where(torch.isnan(top), 255, e + 127).squeeze(-1).to(torch.uint8)
    return v.reshape(x.shape), byte


def held_values(pages, scales=None):
    """float64 values of a cache's pages [pages, page_size, H, d]."""
    if scales is None:
        return pages.double()
    table = torch.cat((E2M1, -E2M1)).double().to(pages.device)
    x = table[torch.stack((pages & 15, pages >> 4), -1).long().flatten(-2)]
    f = torch.exp2(scales.double() - 127)
    f = torch.where(scales == 255, torch.full_like(f, math.nan), f)
    return (x.reshape(*x.shape[:-1], -1, 32) * f[..., None]).reshape(x.shape)


def context(values, table, b, length, page_size):
    """[length, H, d] of sequence b."""
    at = torch.arange(length, device=values.device)
    return values[table[b].long()[at // page_size], at % page_size]


def attend(q, ks, vs, lengths, new_lengths, scale=None, window=None):
    """q [B, T, Hq, d] float64, ks[b] and vs[b] [length, Hkv, d]; (o, lse, sum of p |v|)."""
    B, T, Hq, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    o = torch.zeros_like(q)
    size = torch.zeros_like(q)
    lse = q.new_full((B, Hq, T), -math.inf)
    for b in range(B):
        G = Hq // ks[b].shape[1]
        for t in range(min(new_lengths[b], T)):
            end = lengths[b] - new_lengths[b] + t + 1
            lo = 0 if window is None else max(0, end - 1 - window)
            if end <= lo:
                continue
            k, v = (x[lo:end].repeat_interleave(G, 1) for x in (ks[b], vs[b]))
            logits = torch.einsum("hd,lhd->hl", q[b, t], k) * scale
            p = torch.softmax(logits, -1)
            o[b, t], size[b, t] = torch.einsum("hl,lhd->hd", p, v), torch.einsum("hl,lhd->hd", p, v.abs())
            lse[b, :, t] = torch.logsumexp(logits, -1)
    return o, lse, size
