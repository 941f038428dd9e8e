"""What the kernels in few bits compute, in 64 bits from the formulas, on any device."""
from __future__ import annotations

import math

import torch

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def values4(x: torch.Tensor):
    """(the values that the rows of x stand for in 4 bits, the scale bytes [rows, blocks of 32])."""
    rows, width = x.shape
    blocks = -(-width // 32)
    b = torch.zeros((rows, blocks * 32), dtype=torch.float64, device=x.device)
    b[:, :width] = x.double()
    b = b.view(rows, blocks, 32)
    finite = b.isfinite().all(dim=-1)
    a = torch.where(finite.unsqueeze(-1), b, torch.zeros_like(b)).abs().amax(dim=-1)
    mant, e = torch.frexp(a)                       # a = mant * 2^e, mant in [0.5, 1)
    e = e - 3 + (mant > 0.875).to(e.dtype)
    e = torch.where(a > 0, e.clamp(min=-127), torch.full_like(e, -127))
    unit = torch.ldexp(torch.ones_like(a), e)
    t = (b / unit.unsqueeze(-1)).nan_to_num(0, 0, 0)
    mag, q = t.abs(), torch.zeros_like(t)
    for lo, hi, code in zip(MAGNITUDES[:-1], MAGNITUDES[1:], range(1, 8)):
        mid = (lo + hi) / 2
        up = (mag > mid) | ((mag == mid) & (code % 2 == 0))     # a tie goes to the even code
        q = torch.where(up, torch.full_like(q, hi), q)
    v = torch.copysign(q, t) * unit.unsqueeze(-1)
    v = torch.where(finite.unsqueeze(-1), v, torch.full_like(v, float("nan")))
    byte = torch.where(finite, e + 127, torch.full_like(e, 255))
    return v.view(rows, -1)[:, :width], byte


def scale_bytes(scales: torch.Tensor, rows: int, width: int) -> torch.Tensor:
    """The tiles of scales as [rows, blocks of 32], the blocks behind ``width`` (up to the last tile) among them."""
    return scales.permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:rows].int()


def code_values(codes: torch.Tensor) -> torch.Tensor:
    """4-bit codes as their values, the padding of a row among them."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=torch.float64, device=codes.device)
    c = codes.long()
    return table[torch.stack((c % 16, c // 16), dim=-1).view(codes.shape[0], -1)]


def to8(x: torch.Tensor):
    """Vectors (last axis; 64-bit) as the values of their 8-bit codes, and their scales."""
    a = x.abs().amax(dim=-1)
    t = x * torch.where(a >= 2.0 ** -100, 448 / a, torch.zeros_like(a)).unsqueeze(-1)
    e = (torch.frexp(t)[1] - 1).clamp(min=-6)
    step = torch.ldexp(torch.ones_like(t), e - 3)
    return (torch.round(t / step) * step).clamp(-448, 448), torch.where(a >= 2.0 ** -100, a / 448, torch.zeros_like(a))


def turned(x, weight, eps, cos, sin, rot_dim, positions, interleaved):
    """x [n, heads, d] in 64 bits: normed (where there is a weight) and turned by position."""
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps) * weight.double()
    if not rot_dim:
        return x
    c, s = (t.double()[positions.long()].unsqueeze(1) for t in (cos, sin))
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:rot_dim:2], x[..., 1:rot_dim:2]
        out[..., 0:rot_dim:2], out[..., 1:rot_dim:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :rot_dim // 2], x[..., rot_dim // 2:rot_dim]
        out[..., :rot_dim // 2], out[..., rot_dim // 2:rot_dim] = a * c - b * s, a * s + b * c
    return out


def first_visible(pos: int, span: int) -> int:
    if span > 0:
        return max(0, pos - span + 1)
    return (pos // -span) * -span if span < 0 else 0


def attention(q, k, v, k_scale, v_scale, table, row_request, positions, scale, span):
    """(out, sum of p |v|, largest |score|'s sum of products) of every row and head, in 64 bits.  k, v: 64-bit codes."""
    n, h, d = q.shape
    page, kv = k.shape[2], k.shape[1]
    out = torch.zeros((n, h, d), dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(out)
    size = torch.zeros((n, h, 1), dtype=torch.float64, device=q.device)
    for r in range(n):
        pos = int(positions[r])
        if pos < 0:
            continue
        j = torch.arange(first_visible(pos, span), pos + 1, device=q.device)
        of = table[int(row_request[r])].long()[j // page]
        keys = k[of, :, j % page] * k_scale[of, :, j % page].double().unsqueeze(-1)        # [keys, kv, d]
        vals = v[of, :, j % page] * v_scale[of, :, j % page].double().unsqueeze(-1)
        for g in range(kv):
            rows = slice(g * (h // kv), (g + 1) * (h // kv))
            qq = q[r, rows].double()
            p = torch.softmax(qq @ keys[:, g].t() * scale, dim=-1)
            out[r, rows], weight[r, rows] = p @ vals[:, g], p @ vals[:, g].abs()
            size[r, rows] = (qq.abs() @ keys[:, g].abs().t()).amax(dim=-1, keepdim=True) * abs(scale)
    return out, weight, size
