"""ORACLE (test infrastructure only; never imported by the product path).

CPU restatement in 64 bits of the norms and rotation of queries and KV rows
(``sas_norm_rope_v1``), their gradients, and the cache append. The reference
has none of them: its operator starts from rotated rows
(sparse_attn_sharedkv_tilelang/api.py:129-153).

Pins (tests/test_rope.py): known rotations by 0, 90 and 180 degrees, rows of unit
mean square after a norm, inverse of the rotation, gradients against central
differences; a planted mistake (a mean over one channel too many) fails them.
"""

from __future__ import annotations

from typing import Optional

import torch


def rotate(y: torch.Tensor, cs: torch.Tensor, half: bool, inverse: bool) -> torch.Tensor:
    """Rows ``y [..., D]`` with their last channels rotated by the (cos, sin) pairs
    ``cs [..., R / 2, 2]``, one pair at a time."""
    y = y.clone()
    R = 2 * cs.shape[-2]
    base = y.shape[-1] - R
    for i in range(R // 2):
        p, q = (base + i, base + i + R // 2) if half else (base + 2 * i, base + 2 * i + 1)
        c, s = cs[..., i, 0], cs[..., i, 1] * (-1 if inverse else 1)
        a, b = y[..., p].clone(), y[..., q].clone()
        y[..., p] = a * c - b * s
        y[..., q] = a * s + b * c
    return y


def norm(x: torch.Tensor, n: int, w: Optional[torch.Tensor], eps: float, mean_over: Optional[int] = None) -> torch.Tensor:
    """``mean_over`` exists so a test can plant a wrong divisor."""
    if n == 0:
        return x.clone()
    r = 1.0 / torch.sqrt((x[..., :n] ** 2).sum(-1, keepdim=True) / (mean_over or n) + eps)
    h = x[..., :n] * r
    return torch.cat([h if w is None else h * w, x[..., n:]], -1)


def norm_rope(x, n, w, cs, half=False, inverse=False, eps=1e-6, mean_over=None):
    y = norm(x.double(), n, None if w is None else w.double(), eps, mean_over)
    return y if cs is None else rotate(y, cs.double(), half, inverse)


def norm_rope_grad(dy, x, n, w, cs, half=False, inverse=False, eps=1e-6):
    """(dx, dw, sum |terms of dw|) from the formulas in the header of the kernels."""
    x, dy = x.double(), dy.double()
    u = dy if cs is None else rotate(dy, cs.double(), half, not inverse)
    if n == 0:
        return u, None, None
    r = 1.0 / torch.sqrt((x[..., :n] ** 2).mean(-1, keepdim=True) + eps)
    g = u[..., :n] if w is None else u[..., :n] * w.double()
    m = (g * x[..., :n]).mean(-1, keepdim=True) * r * r
    dx = torch.cat([r * (g - x[..., :n] * m), u[..., n:]], -1)
    terms = u[..., :n] * x[..., :n] * r
    terms = terms.reshape(-1, n)
    return dx, terms.sum(0), terms.abs().sum(0)


def slots(cu, used, T):
    """Each token's (sequence, cache position), or None where it is padding."""
    cu, used = cu.tolist(), used.tolist()
    out = [None] * T
    for b, kv in enumerate(used):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            if 0 <= cu[b] + i < T and kv - n + i >= 0:
                out[cu[b] + i] = (b, kv - n + i)
    return out


def rows_of(places, table, bs, num_blocks):
    """Flat cache row of each place, or None."""
    bt = table.tolist()
    out = []
    for p in places:
        if p is None or p[1] // bs >= len(bt[p[0]]):
            out.append(None)
            continue
        blk = bt[p[0]][p[1] // bs]
        out.append(blk * bs + p[1] % bs if 0 <= blk < num_blocks else None)
    return out
