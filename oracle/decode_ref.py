"""Oracle of the decode operators in plain torch and 64 bits: rotary positions,
the rows of a page pool, and attention of one token over a page table. Runs on
any device; nothing of the product is used."""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch


def rotate(x: torch.Tensor, positions: torch.Tensor, angles: torch.Tensor, gain: float = 1.0,
           interleaved: bool = False, transpose: bool = False) -> torch.Tensor:
    """``x [..., heads, D]`` by ``positions [...]``; ``angles`` fp64 radians per
    position of each pair. fp64."""
    y = x.double().clone()
    n = angles.numel()
    a = positions.double()[..., None, None] * angles.double().to(x.device)
    c, s = gain * a.cos(), gain * a.sin()
    if transpose:
        s = -s
    i = torch.arange(n, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    u, w = y[..., first], y[..., second]
    y[..., first] = u * c - w * s
    y[..., second] = w * c + u * s
    return y


def rotate_magnitude(x: torch.Tensor, n: int, gain: float, interleaved: bool) -> torch.Tensor:
    """|x_a| + |x_b| of each value's pair, times gain (0 for the other values):
    what the errors of a rotation scale with."""
    y = torch.zeros_like(x, dtype=torch.float64)
    i = torch.arange(n, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    m = (x[..., first].double().abs() + x[..., second].double().abs()) * gain
    y[..., first] = m
    y[..., second] = m
    return y


def encode(x: torch.Tensor, precision: str, group: int) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rows ``[..., D]`` as a pool stores them: (payload, scales in x's dtype)."""
    if precision == "fp32":
        return x, None
    if precision == "fp16":
        return x.to(torch.float16), None
    D = x.shape[-1]
    g = D if precision == "int8" else (group if D % group == 0 else D)
    steps = 127.0 if precision == "int8" else 7.0
    y = x.double().reshape(*x.shape[:-1], D // g, g)
    # a quotient is rounded to fp32 and then to the row type
    s = (y.abs().amax(-1, keepdim=True) / steps).float().to(x.dtype)
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (y / s.double()).float().to(x.dtype).double().round().clamp(-steps - 1, steps)
    q = torch.where(torch.isnan(q), torch.full_like(q, -steps - 1), q).reshape(x.shape)
    scales = s.squeeze(-1)
    if precision == "int8":
        return q.to(torch.int8), scales
    nib = (q + 8).to(torch.uint8)
    if D % 2:
        nib = torch.cat((nib, torch.zeros_like(nib[..., :1])), -1)
    return nib[..., 0::2] * 16 + nib[..., 1::2], scales


def decode(payload: torch.Tensor, scales: Optional[torch.Tensor], precision: str, D: int) -> torch.Tensor:
    """The values of stored rows, fp64."""
    if precision in ("fp32", "fp16"):
        return payload.double()
    if precision == "int8":
        return payload.double() * scales.double()
    nib = torch.stack((payload // 16, payload % 16), -1).flatten(-2)[..., :D].double() - 8.0
    G = scales.shape[-1]
    return (nib.unflatten(-1, (G, D // G)) * scales.double()[..., None]).flatten(-2)


def pool_values(pool, name: str) -> torch.Tensor:
    """All rows of a pool-like object's ``k`` or ``v``, fp64 ``[pages, heads,
    page_size, D]``."""
    return decode(getattr(pool, name), getattr(pool, "scale_" + name), pool.precision, pool.head_dim)


def visible(page_table: torch.Tensor, lengths: torch.Tensor, pages: int, page_size: int,
            window: Optional[int]) -> list:
    """For each sequence the (page, offset) pairs of the positions that take part."""
    out = []
    width = page_table.shape[1]
    for b in range(page_table.shape[0]):
        hi = min(max(int(lengths[b]), 0), width * page_size)
        lo = max(0, hi - window) if window else 0
        row = []
        for t in range(lo, hi):
            p = int(page_table[b, t // page_size])
            if 0 <= p < pages:
                row.append((p, t % page_size))
        out.append(row)
    return out


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
           lengths: torch.Tensor, sm_scale: float, window: Optional[int] = None):
    """``q [B, Hq, D]``, all rows ``k``, ``v [pages, Hk, page_size, D]`` -> fp64
    (out, lse, weight, reach, peak): for error bounds, ``weight`` = sum p |v|, ``reach``
    = the largest sm_scale * sum |q k| of a row's positions, and ``peak`` = the larger of
    128 max_t (p_t max_d |v_td|) and max_t p_t max |v|."""
    B, Hq, D = q.shape
    pages, Hk, P, _ = k.shape
    group = Hq // Hk
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(out)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=q.device)
    reach = torch.zeros(B, Hq, dtype=torch.float64, device=q.device)
    peak = torch.zeros_like(reach)
    for b, places in enumerate(visible(page_table.cpu(), lengths.cpu(), pages, P, window)):
        if not places:
            continue
        at = torch.tensor(places, device=q.device)
        kb, vb = k[at[:, 0], :, at[:, 1]], v[at[:, 0], :, at[:, 1]]  # [n, Hk, D]
        for h in range(Hq):
            kh, vh, x = kb[:, h // group], vb[:, h // group], q[b, h].double()
            s = sm_scale * (kh @ x)
            lse[b, h] = torch.logsumexp(s, 0)
            p = torch.softmax(s, 0)
            out[b, h] = p @ vh
            weight[b, h] = p @ vh.abs()
            reach[b, h] = abs(sm_scale) * (kh.abs() @ x.abs()).max()
            row = vh.abs().amax(1)
            peak[b, h] = torch.maximum(128 * (p * row).max(), p.max() * row.max())
    return out, lse, weight, reach, peak
