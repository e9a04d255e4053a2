"""Sequence mixers over point clouds in a space-filling order (no counterpart in the reference).

``morton_order`` puts each cloud's points in the order of their Morton codes; along it, neighbours in space
lie near each other. ``SerializedBlock`` alternates the two operators that use the order: a gated scan in both
directions (``functional.gated_scan``), which carries what is far away, and attention over a window of rows
with a learned bias by distance (``functional.window_attention``).

    order = morton_order(pos, ptr)
    block = SerializedBlock(channels=64, heads=4, window=128, radius=0.05).cuda()
    y = block(feats[order], pos[order], ptr)      # rows in Morton order
    out = torch.empty_like(y); out[order] = y     # back in the callers' order
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor, nn

from .functional import gated_scan, window_attention


def _spread(v: Tensor) -> Tensor:
    """Bits 0..9 of v at bits 0, 3, ..., 27."""
    for shift, mask in ((16, 0x030000FF), (8, 0x0300F00F), (4, 0x030C30C3), (2, 0x09249249)):
        v = (v | (v << shift)) & mask
    return v


def morton_order(pos: Tensor, ptr: Tensor) -> Tensor:
    """[N] int64 permutation: each cloud's rows (clouds stay in place) by the 30-bit Morton code of their
    positions within the cloud's bounding cube; equal codes keep their order. Clouds are packed by ptr
    [B + 1]; rows of no cloud stay where they are."""
    n, clouds = pos.shape[0], ptr.numel() - 1
    ptr = ptr.to(pos.device, torch.int64)
    # cloud + 1 of each row: 0 before the first cloud, clouds + 1 behind the last
    at = torch.searchsorted(ptr, torch.arange(n, device=pos.device), right=True)
    p = pos.detach().float()
    rows = at[:, None].expand(-1, 3)
    low = torch.full((clouds + 2, 3), float("inf"), device=p.device).scatter_reduce_(0, rows, p, "amin")
    high = torch.full((clouds + 2, 3), -float("inf"), device=p.device).scatter_reduce_(0, rows, p, "amax")
    side = (high - low).amax(1).clamp(min=1e-30)
    cell = ((p - low[at]) / side[at, None] * 1023.0).long().clamp_(0, 1023)
    code = _spread(cell[:, 0]) | (_spread(cell[:, 1]) << 1) | (_spread(cell[:, 2]) << 2)
    code = torch.where((at > 0) & (at <= clouds), code, 0)
    return torch.argsort((at << 30) | code, stable=True)


class SerializedScan(nn.Module):
    """Gated scan along the rows, in both directions (or, ``causal``, forwards alone), between two linear maps."""

    def __init__(self, channels: int, causal: bool = False):
        super().__init__()
        self.causal = causal
        ways = 1 if causal else 2
        self.ways, self.inner = ways, nn.Linear(channels, 2 * ways * channels)
        self.outer = nn.Linear(ways * channels, channels)
        # memories from a few rows to a few hundred
        self.decay = nn.Parameter(torch.linspace(-5.0, 0.5, channels).repeat(ways, 1))

    def forward(self, x: Tensor, ptr: Tensor, state: Optional[Tensor] = None):
        """(y, state): ``state`` [B, channels] goes on with a stream (causal only)."""
        parts = self.inner(x).chunk(2 * self.ways, 1)
        ys, last = [], None
        for w in range(self.ways):
            h, end = gated_scan(parts[2 * w], parts[2 * w + 1], self.decay[w], ptr, h0=state if w == 0 else None,
                                reverse=w == 1)
            ys.append(h)
            last = end if w == 0 else last
        return self.outer(torch.cat(ys, 1) if self.ways > 1 else ys[0]), last


class SerializedAttention(nn.Module):
    """Attention over ``window`` rows to either side (``causal``: to the left alone) and each cloud's first
    ``sinks`` rows, with a learned bias by the distance of the two points."""

    def __init__(self, channels: int, heads: int, window: int = 128, sinks: int = 0, kv_heads: Optional[int] = None,
                 buckets: int = 32, radius: float = 0.05, steps: int = 4, causal: bool = False):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if channels % heads or heads % kv_heads:
            raise ValueError("channels must be a multiple of heads, and heads of kv_heads")
        self.heads, self.kv_heads, self.dim = heads, kv_heads, channels // heads
        self.window, self.sinks, self.radius, self.steps = (window, 0 if causal else window), sinks, radius, steps
        self.qkv = nn.Linear(channels, (heads + 2 * kv_heads) * self.dim)
        self.outer = nn.Linear(channels, channels)
        self.bias = nn.Parameter(torch.zeros(heads, buckets))

    def forward(self, x: Tensor, pos: Tensor, ptr: Tensor) -> Tensor:
        rows = self.qkv(x).view(x.shape[0], self.heads + 2 * self.kv_heads, self.dim)
        q, k, v = rows.split([self.heads, self.kv_heads, self.kv_heads], 1)  # views: no copy
        y = window_attention(q, k, v, ptr, window=self.window, num_sinks=self.sinks, bias=self.bias, pos_q=pos,
                             radius=self.radius, steps=self.steps)
        return self.outer(y.flatten(1))


class SerializedBlock(nn.Module):
    """x + scan(norm(x)), then x + attention(norm(x)), over rows in a space-filling (or a scan) order."""

    def __init__(self, channels: int, heads: int, window: int = 128, sinks: int = 0, kv_heads: Optional[int] = None,
                 buckets: int = 32, radius: float = 0.05, steps: int = 4, causal: bool = False):
        super().__init__()
        self.norm_scan, self.norm_attn = nn.LayerNorm(channels), nn.LayerNorm(channels)
        self.scan = SerializedScan(channels, causal)
        self.attn = SerializedAttention(channels, heads, window, sinks, kv_heads, buckets, radius, steps, causal)

    def forward(self, x: Tensor, pos: Tensor, ptr: Tensor) -> Tensor:
        x = x + self.scan(self.norm_scan(x), ptr)[0]
        return x + self.attn(self.norm_attn(x), pos, ptr)
