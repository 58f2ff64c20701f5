"""The cache held in 4 bits, plainly and in 64 bits: the format, the attention of single tokens, and what an eviction leaves.
Written from the definitions, one request and head at a time."""
import math

import torch

F64 = torch.float64


def codes_of(rows):
    """Rows [..., D] -> (codes int, scale, mid): scale and mid rounded to bfloat16, as float64."""
    x = rows.to(F64)
    lo, hi = x.min(-1).values, x.max(-1).values
    scale = ((hi - lo) / 15).to(torch.bfloat16).to(F64)
    mid = ((hi + lo) / 2).to(torch.bfloat16).to(F64)
    cell = torch.floor((x - mid.unsqueeze(-1)) / scale.unsqueeze(-1)) + 8
    cell = torch.where((scale == 0).unsqueeze(-1), torch.full_like(cell, 8.0), cell)
    return cell.clamp(0, 15).to(torch.int64), scale, mid


def fields(data, P, D):
    """Bytes [..., P * (D / 2 + 4)] -> (codes int64 [..., P, D], scale [..., P], mid [..., P] as float64)."""
    d = data.cpu()
    lead = d.shape[:-1]
    word = d[..., : P * D // 2].contiguous().view(torch.int32).view(*lead, P, D // 8).to(torch.int64) & 0xFFFFFFFF
    codes = torch.zeros(*lead, P, D, dtype=torch.int64)
    for i in range(8):   # value 2 i of a word in nibble i, value 2 i + 1 in nibble i + 4
        nibble = i // 2 + 4 * (i % 2)
        codes[..., i::8] = (word >> (4 * nibble)) & 15
    f = d[..., P * D // 2:].contiguous().view(torch.bfloat16).view(*lead, P, 2).to(F64)
    return codes, f[..., 0], f[..., 1]


def values(data, P, D):
    codes, scale, mid = fields(data, P, D)
    return mid.unsqueeze(-1) + scale.unsqueeze(-1) * (codes.to(F64) - 7.5)


def pack(codes, scale, mid, P, D):
    """The reverse of ``fields``: codes [..., P, D], scale and mid [..., P]."""
    lead = codes.shape[:-2]
    word = torch.zeros(*lead, P, D // 8, dtype=torch.int64)
    for i in range(8):
        word |= codes[..., i::8].to(torch.int64) << (4 * (i // 2 + 4 * (i % 2)))
    word = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
    f = torch.stack([scale, mid], -1).to(torch.bfloat16).contiguous()
    return torch.cat([word.contiguous().view(torch.uint8).view(*lead, P * D // 2), f.view(torch.uint8).view(*lead, P * 4)], -1)


def rotate(x, positions, inv_freq, rot, interleaved):
    """x [T, heads, D] float64."""
    y = x.clone()
    if inv_freq is None or rot == 0:
        return y
    half = rot // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        theta = positions.to(F64) * float(inv_freq[i])
        c, s = torch.cos(theta).unsqueeze(1), torch.sin(theta).unsqueeze(1)
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def in_sight(t, p, window, keep_first, chunk):
    if t > p:
        return False
    if chunk > 0:
        return t >= p - p % chunk
    if window > 0:
        return p - t < window or t < keep_first
    return True


def decode(q, pool, table, ctx, H, kv, D, P, scale, window=0, keep_first=0, chunk=0, sink=None, slopes=None):
    """One token per row of q [B, H * D] at position ctx[b].  -> (out, tol, weight): out [B, H, D]; tol: how far a bfloat16 operand of the
    tensor cores may move each output (weights times scale rounded by half a step, 2^-8); mass: sum of p |v| and of |q| |k| for float32 sums;
    weight {(page, head, offset): what the key received}.  ``sink``: None, True, or a score per head."""
    B, G = q.shape[0], H // kv
    out, step = torch.zeros(B, H, D, dtype=F64), torch.zeros(B, H, D, dtype=F64)
    mass, got = torch.zeros(B, H, D, dtype=F64), {}
    q = q.cpu().to(F64).view(B, H, D)
    pool, table = pool.cpu(), table.cpu()
    for b in range(B):
        p = int(ctx[b])
        live = [t for t in range(p + 1) if in_sight(t, p, window, keep_first, chunk)]
        pages = sorted({int(table[b, t // P]) for t in live})
        where = {pg: i for i, pg in enumerate(pages)}
        codes, sc, mid = fields(pool[pages], P, D)                       # [pages, 2, kv, P, ...]
        pi = torch.tensor([where[int(table[b, t // P])] for t in live])
        oi = torch.tensor([t % P for t in live])
        tt = torch.tensor(live, dtype=F64)
        for h in range(H):
            g = h // G
            kc, ks, km = codes[pi, 0, g, oi].to(F64), sc[pi, 0, g, oi], mid[pi, 0, g, oi]
            vc, vs, vm = codes[pi, 1, g, oi].to(F64), sc[pi, 1, g, oi], mid[pi, 1, g, oi]
            K, V = km[:, None] + ks[:, None] * (kc - 7.5), vm[:, None] + vs[:, None] * (vc - 7.5)
            s = (K @ q[b, h]) * scale
            if slopes is not None:
                s = s - float(slopes[h]) * (p - tt)
            top = s.max()
            e = torch.exp(s - top)
            total = e.sum()
            if sink is not None:
                total = total + math.exp((0.0 if sink is True else float(sink[h])) - float(top))
            w = e / total
            out[b, h] = w @ V
            step[b, h] = 2.0 ** -8 * (w @ (vs[:, None] * (vc - 7)).abs())
            size = float(((ks[:, None] * (kc - 7)).abs() @ q[b, h].abs() + (km - 0.5 * ks).abs() * q[b, h].abs().sum()).max()) * abs(scale)
            mass[b, h] = (1 + size) * (w @ (V.abs() + vs[:, None] * 7.5))
            for i, t in enumerate(live):
                at = (int(table[b, t // P]), g, t % P)
                got[at] = got.get(at, 0.0) + float(w[i])
    return out, step, mass, got


def stay(weights, keep, first, recent):
    """Indices, ascending, of the keys of one head that stay: weights is a list of floats."""
    n = len(weights)
    if n <= keep:
        return list(range(n))
    sure = set(range(first)) | set(range(n - recent, n))
    rest = [t for t in range(n) if t not in sure]
    rest.sort(key=lambda t: (-math.inf if weights[t] != weights[t] else weights[t], -t), reverse=True)
    # (a weight that is not a number counts as lighter than all others, minus infinity included)
    numbers = [t for t in rest if weights[t] == weights[t]]
    others = sorted(t for t in rest if weights[t] != weights[t])
    return sorted(sure | set((numbers + others)[: keep - first - recent]))
