"""The 4-bit cache and attention over it, from their definitions, in 64 bits on the CPU (the steps that the definition takes in 32 bits
are taken so). Shares no code with the package."""
import math

import torch

FIFTEENTH = 0.06666667014360428         # the 32-bit number next to 1/15


def width(hd):
    return 32 * -(-hd // 32) + 8


def rotate(x, positions, inv_freq):
    """x [T, heads, hd] -> float64, rotated by the angles position * inv_freq in 32 bits."""
    x = x.double()
    if inv_freq is None:
        return x
    t = (positions.float()[:, None] * inv_freq[None]).double()[:, None]
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()), dim=-1)


def quantise(x):
    """float32 [..., hd] -> (codes int [..., hd], scale, minimum float32 [...])."""
    lo, hi = x.amin(-1), x.amax(-1)
    s = (hi * FIFTEENTH - lo * FIFTEENTH).bfloat16().float()
    m = lo.bfloat16().float()
    n = torch.where((s != 0)[..., None], torch.round((x - m[..., None]) / s[..., None]).clamp(0, 15), torch.zeros_like(x)).nan_to_num(0.0)
    bad = ~torch.isfinite(x).all(-1)
    s, m = (torch.where(bad, torch.full_like(t, float("nan")), t) for t in (s, m))
    return torch.where(bad[..., None], torch.zeros_like(n), n).int(), s, m


def values(n, s, m):
    return m.double()[..., None] + s.double()[..., None] * n.double()


def _offsets(hd, which, off):
    """Byte, inside the group of eight tokens, of every number of token `off`'s key (0) or value (1), and the shift of its code."""
    C = -(-hd // 32)
    d = torch.arange(hd)
    return (which * C + d // 32) * 128 + (off % 8) * 16 + (d % 32) // 2, 4 * (d % 2)


def write(cache, page, head, off, which, n, s, m):
    """Put one vector's codes, scale and minimum into the bytes of a cache (uint8 [pages, heads, page size, W], CPU)."""
    hd, W = n.numel(), cache.shape[3]
    group = cache[page, head].reshape(-1)[(off // 8) * 8 * W:][:8 * W]
    at, shift = _offsets(hd, which, off)
    C = -(-hd // 32)
    mine = torch.arange(C)[:, None] * 128 + which * C * 128 + (off % 8) * 16 + torch.arange(16)[None]
    group[mine.reshape(-1)] = 0
    for i in range(hd):
        group[at[i]] |= int(n[i]) << int(shift[i])
    p = 256 * C + 8 * (off % 8) + 4 * which
    group[p:p + 4] = torch.stack((s, m)).bfloat16().view(torch.uint8)


def read(cache, page, head, off, which, hd):
    """float64 [hd]: the vector that the bytes stand for."""
    W = cache.shape[3]
    group = cache[page, head].reshape(-1)[(off // 8) * 8 * W:][:8 * W]
    at, shift = _offsets(hd, which, off)
    n = group[at].int() >> shift & 15
    p = 256 * (-(-hd // 32)) + 8 * (off % 8) + 4 * which
    s, m = group[p:p + 4].clone().view(torch.bfloat16).double()
    return m + s * n.double()


def pack(k, v, page_size):
    """k, v float32 [L, heads, hd] with L a multiple of page_size -> (cache uint8 [L / page_size, heads, page_size, W], keys, values
    float64 [L, heads, hd] that it holds): the same bytes that `write` makes, all at once."""
    L, G, hd = k.shape
    C, W = -(-hd // 32), width(hd)
    parts, held, par = [], [], []
    for x in (k, v):
        n, s, m = quantise(x)
        held.append(values(n, s, m))
        n = torch.nn.functional.pad(n, (0, 32 * C - hd))
        b = (n[..., 0::2] | n[..., 1::2] << 4).to(torch.uint8)                      # [L, G, 16 C]
        parts.append(b.view(L // 8, 8, G, C, 16).permute(0, 2, 3, 1, 4).reshape(L // 8, G, C * 128))
        par += [s, m]
    par = torch.stack(par, dim=-1).bfloat16().view(torch.uint8).view(L // 8, 8, G, 8).transpose(1, 2).reshape(L // 8, G, 64)
    groups = torch.cat(parts + [par], dim=-1)                                       # [L / 8, G, 8 W]
    cache = groups.view(L // page_size, page_size // 8, G, 8 * W).transpose(1, 2).reshape(L // page_size, G, page_size, W)
    return cache.contiguous(), held[0], held[1]


def attend(q, k, v, positions, scale, window=0):
    """q [rows, H, hd], k, v float64 [L, G, hd] of one request, positions [rows] -> (out float64 [rows, H, hd], the largest |score| terms:
    sum |q_d k_d| * scale of the visible keys, the rows' softmax-weighted sum of |v|)."""
    rows, H, hd = q.shape
    G = k.shape[1]
    q = q.double().view(rows, G, H // G, hd)
    s = torch.einsum("ngud,lgd->nglu", q, k) * scale
    j = torch.arange(k.shape[0])
    seen = j[None] <= positions[:, None]
    if window:
        seen &= j[None] > positions[:, None] - window
    s = s.masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.softmax(s, dim=2).masked_fill(~seen.any(1)[:, None, None, None], 0.0)
    out = torch.einsum("nglu,lgd->ngud", p, v.masked_fill(~seen.any(0)[:, None, None], 0.0))
    size = (torch.einsum("ngud,lgd->nglu", q.abs(), k.abs()) * abs(scale)).masked_fill(~seen[:, None, :, None], 0.0).amax(2)
    mag = torch.einsum("nglu,lgd->ngud", p, v.abs().masked_fill(~seen.any(0)[:, None, None], 0.0))
    return out.reshape(rows, H, hd), size.reshape(rows, H, 1), mag.reshape(rows, H, hd)
