"""Operators of a cache held in 4 bits: writing rows, laying them out for prompts, attention of single tokens over them, and
eviction by accumulated attention weight.

``own`` false: the plain form, elementary torch operations in 32 bits (angles in 64).  ``own`` true: the framework's kernels.

A layer's pool is uint8 [pages, 2 (K, V), kv heads, page_tokens * (head_dim / 2 + 4)].  The bytes of one page, plane and head are
``page_tokens`` rows of ``head_dim / 2`` bytes of codes, then ``page_tokens`` pairs (scale, mid) of bfloat16.  A row x is held as

    scale = bf16((max/2 - min/2) / 7.5)     mid = bf16(min/2 + max/2)     code = clamp(floor((x - mid) / scale) + 8, 0, 15)

and stands for mid + scale * (code - 7.5); with scale 0 for mid.  Of eight values in a little-endian 32-bit word value 2 i lies in
nibble i and value 2 i + 1 in nibble i + 4.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
F32, F64, BF16, I32 = torch.float32, torch.float64, torch.bfloat16, torch.int32
# places of the eight nibbles of a word, by value
PLACES = [16 * (d % 2) + 4 * (d // 2) for d in range(8)]


def listed():
    """Head counts: 16 on 16 and 28 on 4 of 128 are bench.py's two configurations, 4,096 and 8,192 tokens its contexts, batches 1, 8
    and 64 its batches; pages of 64 tokens are the engine's default."""
    return [
        # the write of one generated token of one request (its rows are read back as a prompt kernel would read them)
        dict(name="write 1 token", op="write", heads=16, kv=16, dim=128, rot=128, swap=False, n=1, reqs=1, far=4095, page=64, lens=1),
        # portions of four prompts in one step
        dict(name="write 2048 tokens", op="write", heads=28, kv=4, dim=128, rot=128, swap=False, n=2048, reqs=4, far=30000, page=64, lens=2),
        # a long prompt's portion, every head with keys of its own
        dict(name="write 8192 tokens", op="write", heads=16, kv=16, dim=128, rot=128, swap=False, n=8192, reqs=1, far=0, page=64, lens=3),
        # one generated token: one request, a batch, a full batch over grouped heads, one request with a very long context
        dict(name="decode 1 x 4096", op="decode", heads=16, kv=16, dim=128, reqs=1, ctx=4096, least=4096, page=64, lens=4, dtype="bf16"),
        dict(name="decode 8 x 4096", op="decode", heads=16, kv=16, dim=128, reqs=8, ctx=4096, least=4096, page=64, lens=5, dtype="bf16"),
        dict(name="decode 64 x 8192 ragged", op="decode", heads=28, kv=4, dim=128, reqs=64, ctx=8192, least=777, page=64, lens=6, dtype="bf16"),
        dict(name="decode 1 x 131001", op="decode", heads=28, kv=4, dim=128, reqs=1, ctx=131001, least=131001, page=64, lens=7, dtype="bf16"),
        # a float32 model
        dict(name="decode 8 x 2000 f32", op="decode", heads=16, kv=8, dim=64, reqs=8, ctx=2000, least=1, page=64, lens=8, dtype="f32"),
        # the same step where the cache will be evicted from: every key's weight is added up
        dict(name="weigh 8 x 4096", op="weigh", heads=16, kv=16, dim=128, reqs=8, ctx=4096, least=4096, page=64, lens=9, dtype="bf16"),
        dict(name="weigh 64 x 4096 ragged", op="weigh", heads=28, kv=4, dim=128, reqs=64, ctx=4096, least=100, page=64, lens=10, dtype="bf16"),
        # half of one request's keys leave, in every layer; a batch of long requests, down to what each may keep
        dict(name="evict 1 x 4096", op="evict", layers=24, kv=16, dim=128, reqs=1, ctx=4096, least=4096, keep=2048, first=4, recent=512, page=64, lens=11),
        dict(name="evict 8 x 8192 ragged", op="evict", layers=28, kv=4, dim=128, reqs=8, ctx=8192, least=2500, keep=4000, first=16, recent=1001, page=64, lens=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["write", "decode", "decode", "weigh", "evict"])
    heads, kv, dim = rng.choice([(16, 16, 128), (28, 4, 128), (16, 8, 64), (12, 1, 64), (8, 2, 256), (20, 20, 64)])
    c = dict(op=op, kv=kv, dim=dim, page=rng.choice([16, 64, 64, 128]), lens=rng.randrange(1 << 30))
    if op == "write":
        n = _log(rng, 1, 8192 * 48 // max(48, heads + 2 * kv) // (2 if dim > 128 else 1))
        c.update(heads=heads, rot=rng.choice([dim, dim // 2]), swap=rng.random() < 0.5, n=n, reqs=rng.randint(1, min(8, n)), far=_log(rng, 1, 100000))
    elif op == "evict":
        reqs = _log(rng, 1, 8)
        layers = rng.randint(1, 24)
        ctx = _log(rng, 16, min(40000, (28 * 8 * 8192 * 4 * 128) // (2 * reqs * layers * kv * dim)))
        keep = rng.randint(1, ctx)
        first = rng.randint(0, min(keep, 64))
        c.update(layers=layers, reqs=reqs, ctx=ctx, least=rng.randint(1, ctx), keep=keep, first=first, recent=rng.randint(0, keep - first))
    else:
        reqs = _log(rng, 1, 64)
        f32 = rng.random() < 0.25
        most = (64 * 8192 * 4 * 128) // (reqs * kv * dim * (4 if f32 else 1) * (2 if op == "weigh" else 1))
        ctx = _log(rng, 1, min(131072, most))
        c.update(heads=heads, reqs=reqs, ctx=ctx, least=rng.randint(1, ctx), dtype="f32" if f32 else "bf16")
    return c


# ---------------------------------------------------------------------------
# sizes that follow from a case


def _lens(case):
    """Tokens of every request, from ``least`` to ``ctx`` (a write: ``n`` tokens over ``reqs`` requests)."""
    r = random.Random(case["lens"])
    if case["op"] == "write":
        cuts = sorted(r.sample(range(1, case["n"]), case["reqs"] - 1))
        return [b - a for a, b in zip([0] + cuts, cuts + [case["n"]])]
    lens = [r.randint(case["least"], case["ctx"]) for _ in range(case["reqs"])]
    lens[r.randrange(len(lens))] = case["ctx"]
    return lens


def _row(case):
    return case["dim"] // 2 + 4


def work(case):
    lens, kv, D = _lens(case), case["kv"], case["dim"]
    n = sum(lens)
    rows = 2 * kv * _row(case)   # bytes of a token in the cache
    if case["op"] == "write":
        H = case["heads"]
        return {"bytes": n * ((H + 2 * kv) * D * 2 + H * D * 2 + rows + 2 * kv * D * 2), "flops": n * (6 * (H + kv) + 12 * kv) * D}
    if case["op"] == "evict":
        stay = sum(min(x, case["keep"]) for x in lens)
        return {"bytes": case["layers"] * (n * kv * 4 + stay * (2 * rows + 8 * kv)), "flops": case["layers"] * n * kv}
    el = 4 if case["dtype"] == "f32" else 2
    extra = 8 * kv * n if case["op"] == "weigh" else 0
    return {"bytes": n * rows + 2 * len(lens) * case["heads"] * D * el + extra, "flops": 4 * n * case["heads"] * D}


# ---------------------------------------------------------------------------
# the format, in torch


def _quantise(x):
    """Rows [..., D] float32 -> codes [..., D] int32, scale and mid [...] bfloat16."""
    lo, hi = x.amin(-1) * 0.5, x.amax(-1) * 0.5
    scale = ((hi - lo) / 7.5).to(BF16)
    mid = (lo + hi).to(BF16)
    s, m = scale.float().unsqueeze(-1), mid.float().unsqueeze(-1)
    code = torch.where(s == 0, torch.full_like(x, 8.0), torch.floor((x - m) / s) + 8.0)
    return code.clamp(0, 15).to(I32), scale, mid


def _pack(codes, scale, mid):
    """codes [n, heads, P, D], scale and mid [n, heads, P] -> bytes [n, heads, P * (D / 2 + 4)]."""
    n, h, P, D = codes.shape
    shifts = torch.tensor(PLACES, dtype=I32, device=codes.device)
    words = (codes.view(n, h, P, D // 8, 8) << shifts).sum(-1, dtype=torch.int64)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(I32)
    factors = torch.stack([scale, mid], -1).contiguous().view(torch.uint8)
    return torch.cat([words.contiguous().view(torch.uint8).view(n, h, P * D // 2), factors.view(n, h, P * 4)], -1)


def _values(data, P, D):
    """Bytes [..., P * (D / 2 + 4)] -> values [..., P, D] float32."""
    lead = data.shape[:-1]
    words = data[..., : P * D // 2].contiguous().view(I32).view(*lead, P, D // 8, 1)
    factors = data[..., P * D // 2:].contiguous().view(BF16).view(*lead, P, 2).float()
    codes = (words >> torch.tensor(PLACES, dtype=I32, device=data.device)) & 15
    x = codes.view(*lead, P, D).float() - 7.5
    s, m = factors[..., :1], factors[..., 1:]
    return m + s * x


def _rotate(x, positions, inv_freq, rot, swap):
    """Pairs (i, i + rot / 2), with ``swap`` (2 i, 2 i + 1), of x [T, heads, D] float32 by position * inv_freq."""
    angle = positions.double().unsqueeze(-1) * inv_freq.double()
    c, s = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if swap else (r[..., : rot // 2], r[..., rot // 2:])
    y = (a * c - b * s, a * s + b * c)
    y = torch.stack(y, -1).flatten(-2) if swap else torch.cat(y, -1)
    return torch.cat([y, rest], -1)


# ---------------------------------------------------------------------------
# inputs


def _tables(lens, page, gen, spare=0):
    """Block table [requests, width] (-1 behind a request's pages) over pages in random order, the number of pages, and ``spare``
    further tables of that many pages per request."""
    need = [-(-x // page) for x in lens]
    total = sum(need) + spare * len(lens)
    order = torch.randperm(total, generator=gen, device=DEV).to(I32)
    width = max(need)
    table = torch.full((len(lens), width), -1, dtype=I32, device=DEV)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    return table, total, order[at:].view(len(lens), spare).contiguous()


def _pool(shape, P, D, gen):
    """A pool whose rows hold normally distributed keys and values."""
    pages, planes, kv = shape
    pool = torch.empty((pages, planes, kv, P * (D // 2 + 4)), dtype=torch.uint8, device=DEV)
    flat = pool.view(pages * planes, kv, -1)
    step = max(1, (1 << 26) // (kv * P * D))
    for a in range(0, flat.shape[0], step):
        n = min(step, flat.shape[0] - a)
        x = torch.randn((n, kv, P, D), generator=gen, device=DEV)
        flat[a:a + n] = _pack(*_quantise(x))
    return pool


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    lens, kv, D, P = _lens(case), case["kv"], case["dim"], case["page"]
    st = dict(case=case, lens=lens, n_tokens=torch.tensor(lens, dtype=I32, device=DEV))
    if case["op"] == "write":
        T, H, rot = case["n"], case["heads"], case["rot"]
        table, pages, _ = _tables(lens, P, gen)
        at, slots, positions = torch.tensor(lens), [], []
        host = table.cpu()
        for i, n in enumerate(lens):
            t = torch.arange(n)
            slots.append(host[i, t // P] * P + (t % P).to(I32))
            positions.append(case["far"] + 17 * i + t)
        st.update(
            qkv=torch.randn((T, (H + 2 * kv) * D), generator=gen, device=DEV).to(BF16), table=table,
            positions=torch.cat(positions).to(I32).to(DEV), slots=torch.cat(slots).to(I32).to(DEV),
            inv_freq=(1e6 ** (-torch.arange(0, rot, 2, dtype=F64) / rot)).float().to(DEV),
            segs=torch.arange(len(lens), dtype=I32, device=DEV), ctx=torch.zeros(len(lens), dtype=I32, device=DEV), seg_qn=at.to(I32).to(DEV),
            q_out=torch.zeros((T, H * D), dtype=BF16, device=DEV),
            pool=torch.zeros((pages, 2, kv, P * (D // 2 + 4)), dtype=torch.uint8, device=DEV),
            wide=torch.zeros((pages, 2, kv, P, D), dtype=BF16, device=DEV))
    elif case["op"] == "evict":
        stay = -(-min(case["keep"], max(lens)) // P)
        table, pages, dst = _tables(lens, P, gen, stay)
        L = case["layers"]
        pool = torch.randint(0, 256, (L, pages, 2, kv, P * (D // 2 + 4)), generator=gen, device=DEV, dtype=torch.uint8)
        # what a key has received in all: most next to nothing, a few a great deal
        weights = torch.randn((L, pages, kv, P), generator=gen, device=DEV).mul_(2.5).exp_()
        st.update(table=table, dst=dst, pool=pool, weights=weights,
                  kept=torch.full((L, len(lens), kv, case["keep"]), -1, dtype=I32, device=DEV))
    else:
        table, pages, _ = _tables(lens, P, gen)
        dt, H, B = (F32 if case["dtype"] == "f32" else BF16), case["heads"], len(lens)
        st.update(table=table, pool=_pool((pages, 2, kv), P, D, gen), q=torch.randn((B, H * D), generator=gen, device=DEV).mul_(1.5).to(dt),
                  out=torch.zeros((B, H * D), dtype=dt, device=DEV), ctx=st["n_tokens"] - 1,
                  rows=torch.arange(B, dtype=I32, device=DEV), weights=None, scores=None)
        if case["op"] == "weigh":
            st["weights"] = torch.rand((pages, kv, P), generator=gen, device=DEV)
            st["scores"] = torch.empty(B * H * table.shape[1] * P, dtype=F32, device=DEV)
        # scratch that a program keeps for its steps: partial results of the key ranges, and their counters
        units = B * H + 8 * 16 * torch.cuda.get_device_properties(DEV).multi_processor_count
        st.update(part_o=torch.empty(units * D, dtype=F32, device=DEV), part_ml=torch.empty(2 * units, dtype=F32, device=DEV),
                  counters=torch.zeros(B * H, dtype=I32, device=DEV))
    return st


# ---------------------------------------------------------------------------
# one pass


def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    if op == "write":
        return _plain_write(st)
    if op == "evict":
        return _plain_evict(st)
    return _plain_decode(st)


def _run_own(st):
    from locus_b200 import kernels as K

    c = st["case"]
    sizes = dict(n_kv_heads=c["kv"], head_dim=c["dim"], page_tokens=c["page"])
    if c["op"] == "write":
        K.rope_kv_write_q4(st["qkv"], st["positions"], st["inv_freq"], st["q_out"], st["pool"], st["slots"], n_heads=c["heads"],
                           rot_dim=c["rot"], interleaved=c["swap"], **sizes)
        K.expand_q4(st["pool"], st["wide"], segs=st["segs"], n_segs=len(st["lens"]), seg_ctx=st["ctx"], seg_qn=st["seg_qn"],
                    block_table=st["table"], max_keys=max(st["lens"]), **sizes)
        return st["q_out"], st["wide"]
    if c["op"] == "evict":
        K.evict_q4(st["pool"], st["weights"], block_table=st["table"], dst_table=st["dst"], n_tokens=st["n_tokens"], n_items=len(st["lens"]),
                   keep=c["keep"], first=c["first"], recent=c["recent"], kept=st["kept"], max_tokens=max(st["lens"]), **sizes)
        return _moved(st)
    K.attn_decode_q4(st["q"], st["pool"], st["out"], seg_q0=st["rows"], seg_ctx=st["ctx"], block_table=st["table"], items=st["rows"],
                     n_items=len(st["lens"]), n_heads=c["heads"], window=0, scale=c["dim"] ** -0.5, part_o=st["part_o"],
                     part_ml=st["part_ml"], counters=st["counters"], weights=st["weights"], scores=st["scores"], **sizes)
    return (st["out"], st["weights"]) if c["op"] == "weigh" else st["out"]


def _moved(st):
    """What an eviction leaves: which keys stayed, and the pools (rows and weights in the pages of ``dst``, the others as they were)."""
    return st["kept"], st["pool"], st["weights"]


def _plain_write(st):
    c = st["case"]
    H, kv, D, P = c["heads"], c["kv"], c["dim"], c["page"]
    x = st["qkv"].float().view(c["n"], H + 2 * kv, D)
    turned = _rotate(x[:, : H + kv], st["positions"], st["inv_freq"], c["rot"], c["swap"])
    st["q_out"].copy_(turned[:, :H].reshape(c["n"], H * D))
    rows = torch.stack([turned[:, H:], x[:, H + kv:]], 1)            # [T, 2, kv, D]
    code, scale, mid = _quantise(rows)
    value = mid.float().unsqueeze(-1) + scale.float().unsqueeze(-1) * (code.float() - 7.5)
    page, off = (st["slots"] // P).long(), (st["slots"] % P).long()
    st["wide"].permute(0, 3, 1, 2, 4)[page, off] = value.to(BF16)
    return st["q_out"], st["wide"]


def _plain_decode(st):
    c = st["case"]
    H, kv, D, P = c["heads"], c["kv"], c["dim"], c["page"]
    B, W = st["table"].shape
    data = st["pool"][st["table"].clamp(min=0).long()]               # [B, W, 2, kv, bytes]
    x = _values(data.permute(0, 2, 3, 1, 4), P, D).flatten(3, 4)     # [B, 2, kv, W * P, D]
    q = st["q"].float().view(B, kv, H // kv, D)
    s = (q @ x[:, 0].transpose(-1, -2)) * D ** -0.5                  # [B, kv, G, W * P]
    live = torch.arange(W * P, device=DEV) < st["n_tokens"].unsqueeze(1)
    s = s.masked_fill(~live[:, None, None], -math.inf)
    e = (s - s.amax(-1, keepdim=True)).exp()
    p = e / e.sum(-1, keepdim=True)
    st["out"].copy_((p @ x[:, 1]).reshape(B, H * D))
    if c["op"] != "weigh":
        return st["out"]
    got = p.sum(2).view(B, kv, W, P).permute(0, 2, 1, 3)             # [B, W, kv, P]
    here = st["table"] >= 0
    st["weights"].index_add_(0, st["table"][here].long(), got[here])
    return st["out"], st["weights"]


def _plain_evict(st):
    c = st["case"]
    P, keep, first, recent = c["page"], c["keep"], c["first"], c["recent"]
    L, kv, D = c["layers"], c["kv"], c["dim"]
    B, W = st["table"].shape
    n = st["n_tokens"].long()
    pages = st["table"].clamp(min=0).long()
    w = st["weights"][:, pages].permute(0, 1, 3, 2, 4).reshape(L, B, kv, W * P)
    t = torch.arange(W * P, device=DEV)
    held = t < n[:, None]
    always = held & ((t < first) | (t >= n[:, None] - recent))
    w = w.masked_fill(always[None, :, None], math.inf).masked_fill(~held[None, :, None], -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    m = order.shape[-1]                                              # (no request has more than that many tokens)
    chosen = torch.arange(m, device=DEV) < n[:, None]
    order = order.masked_fill(~chosen[None, :, None], W * P).sort(-1).values
    st["kept"].fill_(-1)
    st["kept"][..., :m] = order.masked_fill(~chosen[None, :, None], -1).to(I32)
    # rows and weights of the keys that stay, one behind the other in the pages of dst
    src = torch.where(chosen[None, :, None], order, 0)
    l, b, h, j = torch.nonzero(chosen[None, :, None].expand(L, B, kv, m), as_tuple=True)
    src = src[l, b, h, j]
    p0, o0 = pages[b, src // P], src % P
    p1, o1 = st["dst"].long()[b, j // P], j % P
    rows = st["pool"][..., : P * D // 2].view(*st["pool"].shape[:-1], P, D // 2)
    factors = st["pool"][..., P * D // 2:].view(*st["pool"].shape[:-1], P, 4)
    for_k, for_v = torch.zeros_like(l), torch.ones_like(l)
    rows[l, p1, for_k, h, o1], rows[l, p1, for_v, h, o1] = rows[l, p0, for_k, h, o0], rows[l, p0, for_v, h, o0]
    factors[l, p1, for_k, h, o1], factors[l, p1, for_v, h, o1] = factors[l, p0, for_k, h, o0], factors[l, p0, for_v, h, o0]
    st["weights"][l, p1, h, o1] = st["weights"][l, p0, h, o0]
    return _moved(st)


# ---------------------------------------------------------------------------
# the definition, in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    kv, D, P = case["kv"], case["dim"], case["page"]
    if case["op"] == "evict":
        # keys are chosen and bytes are moved: only the weights are numbers, and they move as they are
        weights = st["weights"].to(F64)
        was = weights.clone()
        table, dst = st["table"].tolist(), st["dst"].tolist()
        for i, n in enumerate(st["lens"]):
            mine = torch.tensor(table[i][: -(-n // P)], device=DEV)
            there = torch.tensor(dst[i], device=DEV)
            w = was[:, mine].transpose(1, 2).reshape(case["layers"], kv, -1)[..., :n]
            if n > case["keep"]:
                rank = w.clone()
                rank[..., : case["first"]] = math.inf
                rank[..., n - case["recent"]:] = math.inf
                # (equal weights: the earlier key is the heavier one)
                best = torch.argsort(-rank, dim=-1, stable=True)[..., : case["keep"]]
                w = torch.gather(w, -1, torch.sort(best, -1).values)
            for a in range(0, w.shape[-1], P):
                weights[:, there[a // P], :, : min(P, w.shape[-1] - a)] = w[..., a:a + P]
        return None, None, weights
    H = case["heads"]
    if case["op"] == "write":
        half = case["rot"] // 2
        x = st["qkv"].to(F64).view(-1, H + 2 * kv, D)
        y = x.clone()
        theta = st["positions"].to(F64)[:, None, None] * st["inv_freq"].to(F64)
        one = torch.arange(0, case["rot"], 2, device=DEV) if case["swap"] else torch.arange(half, device=DEV)
        two = one + (1 if case["swap"] else half)
        a, b = x[:, : H + kv, one], x[:, : H + kv, two]
        y[:, : H + kv, one] = torch.cos(theta) * a - torch.sin(theta) * b
        y[:, : H + kv, two] = torch.cos(theta) * b + torch.sin(theta) * a
        wide = torch.zeros(st["wide"].shape, dtype=F64, device=DEV)
        page, off = torch.div(st["slots"], P, rounding_mode="floor").long(), torch.remainder(st["slots"], P).long()
        for plane, rows in ((0, y[:, H:H + kv]), (1, y[:, H + kv:])):
            top, bottom = rows.max(-1, keepdim=True).values, rows.min(-1, keepdim=True).values
            step = ((top - bottom) / 15).to(BF16).to(F64)
            centre = ((top + bottom) / 2).to(BF16).to(F64)
            cell = torch.floor((rows - centre) / step).clamp(-8, 7)
            held = torch.where(step > 0, centre + step * (cell + 0.5), centre)
            for h in range(kv):
                wide[page, plane, h, off] = held[:, h]
        return y[:, :H].reshape(-1, H * D), wide
    out = torch.zeros((len(st["lens"]), H, D), dtype=F64, device=DEV)
    weights = st["weights"].to(F64) if case["op"] == "weigh" else None
    G = H // kv
    place = torch.tensor([4 * (d // 2 % 4) + 16 * (d % 2) for d in range(D)], device=DEV)
    word = torch.arange(D, device=DEV) // 8
    for i, n in enumerate(st["lens"]):
        mine = st["table"][i, : -(-n // P)].long()
        got = st["pool"][mine]                                        # [pages, 2, kv, bytes]
        b = got[..., : P * D // 2].to(torch.int64).view(len(mine), 2, kv, P, D // 8, 4)
        b = b[..., 0] + b[..., 1] * 256 + b[..., 2] * 65536 + b[..., 3] * 16777216
        f = got[..., P * D // 2:].contiguous().view(BF16).view(len(mine), 2, kv, P, 2).to(F64)
        for h in range(kv):
            K_, V_ = ((f[:, z, h, :, 1:] + f[:, z, h, :, :1] * (((b[:, z, h][..., word] >> place) & 15).to(F64) - 7.5)).reshape(-1, D)[:n] for z in (0, 1))
            qh = st["q"][i].to(F64).view(H, D)[h * G:(h + 1) * G]
            p = torch.softmax(qh @ K_.T / math.sqrt(D), -1)
            out[i, h * G:(h + 1) * G] = p @ V_
            if weights is not None:
                t = torch.arange(n, device=DEV)
                weights[mine[t // P], h, t % P] += p.sum(0)
    out = out.reshape(len(st["lens"]), H * D)
    return (out, weights) if weights is not None else out
