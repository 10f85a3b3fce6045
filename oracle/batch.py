"""The operators around a batch's attention in float64 (torch, any device): NVFP4 rows with the roundings
to E4M3 and E2M1 by the formats' tables, products with the sums of magnitudes their error bounds need,
residual norm, beam selection."""

from __future__ import annotations

import torch

EPS = 1e-6
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]


def _nearest(v, grid):
    """Indices of the nearest of an ascending grid's values for v >= 0, ties to the even index."""
    grid = torch.tensor(grid, dtype=torch.float64, device=v.device)
    middle = (grid[1:] + grid[:-1]) / 2
    low = torch.bucketize(v, middle)              # ties go down ..
    high = torch.bucketize(v, middle, right=True)  # .. or up
    return torch.where(low % 2 == 0, low, high)


def rms(x, w):
    x = x.double()
    return x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()


def quantize(x, pieces):
    """x [m, k] of bf16 values: E2M1 codes uint8 [pieces, m, k], E4M3 bytes uint8 [pieces, m, k / 16] and
    the factors f64 [m] (NaN for a row that is not finite, 0 for one of zeros)."""
    x = x.double()
    m, k = x.shape
    top = x.abs().amax(1)
    live = (top > 0) & torch.isfinite(top)
    g = torch.ones_like(top)
    g[live] = 2.0 ** 126
    while (over := live & (top * g > 2688)).any():
        g[over] /= 2
    y = torch.where(live[:, None], x * g[:, None], 0.0).view(m, k // 16, 16)
    codes, scales = [], []
    for _ in range(pieces):
        at = _nearest(y.abs().amax(2) / 6, E4M3)
        s = torch.tensor(E4M3, dtype=torch.float64, device=x.device)[at][..., None]
        c = torch.where(s > 0, _nearest((y / s.clamp(min=2.0 ** -9)).abs(), E2M1), 0)
        value = torch.tensor(E2M1, dtype=torch.float64, device=x.device)[c] * torch.sign(y)
        codes.append((c + 8 * ((y < 0) & (c > 0))).view(m, k).byte())
        scales.append(at.byte())
        y = y - value * s
    factor = torch.where(live, 1 / g, torch.where(torch.isfinite(x).all(1), 0.0, torch.nan))
    return torch.stack(codes), torch.stack(scales), factor


def values(codes, scales):
    """c * s of codes [..., k] (0..15) and E4M3 bytes [..., k / 16], without any factor."""
    table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=codes.device)
    return table[codes.long()] * torch.tensor(E4M3, dtype=torch.float64, device=codes.device)[scales.long()].repeat_interleave(16, -1)


def pack(codes):
    return (codes[..., 0::2] | codes[..., 1::2] << 4).contiguous()


def unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def scale_at(row, block, cols):
    """Byte of a scale within its matrix's scale blocks."""
    return ((row // 128) * -(-cols // 64) + block // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + block % 4


def scale_blocks(scales, fill=0):
    """[rows, cols / 16] in the order of the scale blocks."""
    rows, nb = scales.shape
    out = torch.full((-(-rows // 128) * -(-nb // 4) * 512,), fill, dtype=torch.uint8, device=scales.device)
    r = torch.arange(rows, device=scales.device)[:, None]
    b = torch.arange(nb, device=scales.device)[None, :]
    out[scale_at(r, b, 16 * nb)] = scales
    return out


def matmul(x, w, fx, fw):
    """(products, sums of their terms' magnitudes) of values x [m, k], w [n, k] and their factors."""
    return (x @ w.T) * fx[:, None] * fw, (x.abs() @ w.abs().T) * fx[:, None].abs() * fw.abs()


def beam_select(logits, scores, k):
    """(scores, beams, tokens) of each group's k best, equal scores in the order of (beam, token)."""
    logits, scores = logits.double(), scores.double()
    top = logits.amax(-1, keepdim=True)
    base = scores - torch.log(torch.exp(logits - top).sum(-1))
    counts = torch.isfinite(base) & torch.isfinite(top[..., 0])
    s = torch.where(counts[..., None], base[..., None] + (logits - top), -torch.inf).flatten(1)
    best, at = torch.sort(s, dim=1, descending=True, stable=True)
    return best[:, :k], at[:, :k] // logits.shape[-1], at[:, :k] % logits.shape[-1]
