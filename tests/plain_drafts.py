"""The operators of decoding with drafted tokens in 64 bits, from their definitions, and bounds for how far 32-bit sums may be off."""
from __future__ import annotations

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # a rounding's error, relative to the value


def first_visible(position: int, span: int) -> int:
    if span > 0:
        return max(0, position - span + 1)
    return position // -span * -span if span < 0 and position >= 0 else 0


def tree_attention(q, k, v, table, q_start, context, positions, seen, scale, span):
    """(o, off): the result in 64 bits, and how far a kernel may be off that keeps sums in 32 bits and rounds the softmax's
    numbers to the inputs' type, a row and number each.

    With a = p @ |v|: a score is a sum of d products, off by (d + 2) 2^-24 of the sum of their magnitudes at most, which moves p by
    that much, and the sums over p and p v by as much again (the denominator); the exponential and its argument's rounding add 2^-22
    and the score's magnitude times 2^-24; the running sums of n terms n 2^-24 each; rounding p to bfloat16 moves the sum by 2^-8 a at most."""
    n, heads, d = q.shape
    pages, kv, places, _ = k.shape
    o = torch.zeros((n, heads, d), dtype=torch.float64)
    off = torch.zeros((n, heads, d), dtype=torch.float64)
    rounded = q.dtype == torch.bfloat16
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    table, start, context = table.tolist(), q_start.tolist(), context.tolist()
    words = seen.tolist()
    for r, c in enumerate(context):
        t = start[r + 1] - start[r]
        c = max(c, 0)
        place = [j for j in range(c + t) if j // places < len(table[r]) and 0 <= table[r][j // places] < pages]
        if not place or not t:
            continue
        pg = torch.tensor([table[r][j // places] for j in place])
        sl = torch.tensor([j % places for j in place])
        kk, vv = k[pg, :, sl], v[pg, :, sl]
        mask = torch.zeros((t, len(place)), dtype=torch.bool)
        for i in range(t):
            row = start[r] + i
            lo = first_visible(int(positions[row]), span) if span else 0
            for x, j in enumerate(place):
                if j < c:
                    mask[i, x] = j >= lo
                else:
                    b = j - c
                    mask[i, x] = b // 32 < len(words[row]) and bool(words[row][b // 32] >> (b % 32) & 1)
        rows = slice(start[r], start[r + 1])
        some = mask.any(1)
        for h in range(heads):
            g = h // (heads // kv)
            s = (q[rows, h] @ kk[:, g].t()) * scale
            s = torch.where(mask, s, torch.full_like(s, float("-inf")))
            p = torch.where(mask, torch.exp(s - torch.where(some, s.max(1).values, 0.0)[:, None]), torch.zeros_like(s))
            p = p / torch.where(some, p.sum(1), 1.0)[:, None]
            # (what a row does not see is left out, whatever stands there)
            finite = torch.where(torch.isfinite(vv[:, g]), vv[:, g], 0.0)
            mean, spread = p @ finite, p @ finite.abs()
            for x in torch.nonzero(~torch.isfinite(vv[:, g]).all(1)).flatten().tolist():
                mean[mask[:, x]] += torch.where(torch.isfinite(vv[x, g]), 0.0, vv[x, g])
            o[rows, h] = mean
            size = (q[rows, h].abs() @ kk[:, g].abs().t() * abs(scale)).nan_to_num(0.0, 0.0, 0.0)
            delta = ((d + 2) * size + s.abs().nan_to_num(0.0, 0.0, 0.0) + 4).masked_fill(~mask, 0).max(1).values * 2.0 ** -24
            off[rows, h] = (2 * delta + 2 * len(place) * 2.0 ** -24)[:, None] * spread
            if rounded:
                off[rows, h] += 2.0 ** -8 * spread
    return o, off


def log_probs(logits, tokens, top):
    """(log probabilities of the tokens, entropy, ids of the likeliest, their log probabilities) in 64 bits."""
    x = logits.cpu().double()
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
    rows, vocab = x.shape
    m = x.max(1).values
    none = torch.isinf(m)
    z = x - torch.where(none, torch.zeros_like(m), m)[:, None]
    e = torch.exp(z)
    total = torch.where(none, torch.full_like(m, float("nan")), e.sum(1))
    lse = torch.log(total)
    t = tokens.cpu().long()
    inside = (t >= 0) & (t < vocab)
    lp = torch.where(inside, z.gather(1, t.clamp(0, vocab - 1)), torch.full((), float("-inf"), dtype=torch.float64)) - lse[:, None]
    w = torch.where(e > 0, e * z, torch.zeros_like(z))
    entropy = lse - w.sum(1) / total
    order = torch.sort(torch.where(torch.isnan(logits.cpu().double()), torch.full_like(x, float("nan")), x).nan_to_num(-1e308, 1e308, -1e307),
                       dim=1, descending=True, stable=True)
    ids = order.indices[:, :top]
    given = ~torch.isnan(logits.cpu().double()).gather(1, ids)
    best = torch.where(given, z.gather(1, ids) - lse[:, None], torch.full((), float("-inf"), dtype=torch.float64))
    ids = torch.where(given, ids, torch.full_like(ids, -1))
    if top > vocab:
        ids = torch.cat((ids, torch.full((rows, top - vocab), -1)), 1)
        best = torch.cat((best, torch.full((rows, top - vocab), float("-inf"), dtype=torch.float64)), 1)
    return lp, entropy, ids, best
