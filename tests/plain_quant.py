"""The quantised cache written out plainly (layout and rounding of csrc/quant_format.cuh), on the CPU."""
from __future__ import annotations

import numpy as np
import torch

MOST = 2.0 ** 60


def groups(x: torch.Tensor) -> torch.Tensor:
    """[..., D] as [..., group, its 32 channels]: channel c is in group (c // 4) % (D / 32)."""
    D = x.shape[-1]
    order = sorted(range(D), key=lambda c: ((c // 4) % (D // 32), c))
    return x[..., order].unflatten(-1, (D // 32, 32))


def ungroup(x: torch.Tensor) -> torch.Tensor:
    D = x.shape[-2] * 32
    order = sorted(range(D), key=lambda c: ((c // 4) % (D // 32), c))
    back = torch.empty(D, dtype=torch.long)
    back[torch.tensor(order)] = torch.arange(D)
    return x.flatten(-2)[..., back]


def quantise(x: torch.Tensor, bits: int):
    """Codes [..., D] (unpacked, int64) and scales [..., D / 32] (bfloat16) of float32 x, step by step in 32 bits."""
    L = 2 ** (bits - 1)
    x = torch.where(x.abs() < 3.38e38, x, torch.zeros_like(x)).clamp(-MOST, MOST)        # (NaN compares false)
    g = groups(x.float())
    hi, lo = g.amax(-1), g.amin(-1)
    scale = (torch.where(hi >= -lo, hi, lo) / -L).bfloat16()
    s = scale.float().unsqueeze(-1)
    q = torch.where(s == 0, torch.zeros_like(g), g / torch.where(s == 0, torch.ones_like(s), s))
    return ungroup(torch.round(q).clamp(-L, L - 1) + L).long(), scale


def values(codes: torch.Tensor, scales: torch.Tensor, bits: int) -> torch.Tensor:
    """What unpacked codes and scales stand for, in float64."""
    return ungroup((groups(codes.double()) - 2 ** (bits - 1)) * scales.double().unsqueeze(-1))


def pack(codes: torch.Tensor, bits: int) -> torch.Tensor:
    return (codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8) if bits == 4 else codes.to(torch.uint8)


def unpack(raw: torch.Tensor, bits: int) -> torch.Tensor:
    raw = raw.long()
    return torch.stack([raw % 16, raw // 16], -1).flatten(-2) if bits == 4 else raw


def heads(x: torch.Tensor, weight, eps: float, cos_sin, rot: int) -> torch.Tensor:
    """Norm and rotation of float32 heads [T, heads, D] in the order of operations the write kernel states."""
    if weight is not None:
        mean = (x.double() ** 2).sum(-1, keepdim=True).div(x.shape[-1]).float()
        # (numpy's square root and division are rounded once; torch's reciprocal on the CPU is not always)
        x = x * torch.from_numpy(np.float32(1) / np.sqrt(mean.numpy() + np.float32(eps))) * weight.float()
    if rot:
        a, b, c, s = x[..., :rot // 2], x[..., rot // 2:rot], cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
        x = torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)
    return x


def attention(q, keys, vals, start: int, window: int, scale: float):
    """One entry in float64: q [n, heads, D] at positions start.., keys and vals [start + n, kv heads, D].
    Returns the result and, for tolerances, the same sum with |values|."""
    n, nq, _ = q.shape
    group = nq // keys.shape[1]
    pos, j = torch.arange(start, start + n)[:, None], torch.arange(start + n)[None]
    seen = (j <= pos) & ((j > pos - window) if window else True)
    k, v = keys.double().repeat_interleave(group, 1), vals.double().repeat_interleave(group, 1)
    s = torch.einsum("nhd,jhd->hnj", q.double(), k) * scale
    p = torch.softmax(s.masked_fill(~seen, -torch.inf), -1)
    return torch.einsum("hnj,jhd->nhd", p, v), torch.einsum("hnj,jhd->nhd", p, v.abs())
