"""Float64 definitions of the tower operators (test infrastructure; CPU torch, autograd gives their gradients).

``qk_norm_rotary``: per-head RMS norm and rotation by position.  ``relative_attention``: attention with a learned relative position bias
by buckets.  ``orthogonalize``: the quintic Newton-Schulz iteration.  Nothing here comes from the product.
"""

from __future__ import annotations

import math
from typing import Optional

import torch


def rotate(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x [B, L, H, D], table [P, rot] (cosines | sines), positions [B, L]."""
    rot = table.shape[1]
    rows = table[positions.long()].to(x.dtype)[:, :, None]
    c, s = rows[..., : rot // 2], rows[..., rot // 2:]
    out = x.clone()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., second] * c + x[..., first] * s
    return out


def qk_norm_rotary(x: torch.Tensor, w: Optional[torch.Tensor], table: Optional[torch.Tensor], positions: Optional[torch.Tensor],
                   interleaved: bool, eps: float) -> torch.Tensor:
    """One side (queries or keys) in x's type."""
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        y = y * w
    if table is None or table.shape[1] == 0:
        return y
    B, L = x.shape[:2]
    if positions is None:
        positions = torch.arange(L)
    return rotate(y, table, positions.expand(B, L), interleaved)


def bucket(rel: int, num_buckets: int, max_distance: int, bidirectional: bool) -> int:
    """Bucket of the distance rel = key - query by integer arithmetic: half of a side's buckets hold one distance each, the others begin
    where (distance / near) ** (side - near) reaches (max_distance / near) ** step."""
    side = num_buckets // 2 if bidirectional else num_buckets
    base = side if bidirectional and rel > 0 else 0
    dist = abs(rel) if bidirectional else max(-rel, 0)
    near = side // 2
    if dist < near:
        return base + dist
    step = 0
    while step < side - near - 1 and dist ** (side - near) * near ** (step + 1) >= max_distance ** (step + 1) * near ** (side - near):
        step += 1
    return base + near + step


def bucket_map(lq: int, lk: int, offset: int, num_buckets: int, max_distance: int, bidirectional: bool) -> torch.Tensor:
    row = {r: bucket(max(-max_distance, min(max_distance, r)), num_buckets, max_distance, bidirectional)
           for r in range(-(lq - 1) - offset, lk - offset)}
    return torch.tensor([[row[j - i - offset] for j in range(lk)] for i in range(lq)], dtype=torch.long).reshape(lq, lk)


def relative_attention(q, k, v, table, max_distance=128, bidirectional=True, scale=None, causal=False, keep=None, q_offset=0):
    """q [B, H, Lq, D], k / v [B, Hk, Lk, D], table [buckets, H], keep bool [B, Lk] or None, q_offset int or list of B -> [B, Lq, H, D].
    Keys that are not kept do not enter at all (their values may be NaN); a row without keys is zero."""
    B, H, lq, D = q.shape
    Hk, lk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = []
    for b in range(B):
        off = q_offset if isinstance(q_offset, int) else int(q_offset[b])
        kept = torch.arange(lk) if keep is None else keep[b].nonzero()[:, 0]
        bias = table[bucket_map(lq, lk, off, table.shape[0], max_distance, bidirectional)][:, kept]      # [lq, kept, H]
        seen = kept[None] <= torch.arange(lq)[:, None] + off if causal else torch.ones(lq, len(kept), dtype=torch.bool)
        kb, vb = (t[b][:, kept].repeat_interleave(H // Hk, 0) for t in (k, v))
        z = (q[b] @ kb.transpose(1, 2)) * scale + bias.permute(2, 0, 1)
        z = z.masked_fill(~seen, -math.inf)
        empty = ~(seen & (z > -math.inf).any(0)).any(1) if len(kept) else torch.ones(lq, dtype=torch.bool)
        if len(kept) == 0:
            out.append((q[b] * 0 + (k[b].sum() + v[b].sum() + table.sum()) * 0).transpose(0, 1))
            continue
        z = z.masked_fill(empty[None, :, None], 0.0)
        p = torch.softmax(z, -1) * (~empty)[None, :, None]
        out.append((p @ vb).transpose(0, 1))
    return torch.stack(out)


def orthogonalize(g, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """One matrix [r, c] in float64."""
    a, b, c = coefficients
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (x.square().sum().sqrt() + eps)
    for _ in range(steps):
        p = x @ x.T
        x = a * x + (b * p + c * p @ p) @ x
    return x.T if tall else x
