"""The cache held in 4 bits, on the GPU, against tests/plain_q4.py in 64 bits.

Tolerances.  A rounding to bfloat16 is off by at most 2^-8 of the value.  Attention in bfloat16 rounds its output once and every weight times its
value's scale once: ``plain_q4.decode`` gives that bound per element.  Sums in float32: an error of a few 2^-24 of the sum of the operands'
sizes; 2^-18 of ``mass`` stands for all of them (at most some hundred roundings per score and per output)."""
import math

import pytest
import torch

import locus_b200.kernels as K
import plain_q4 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32
SUMS = 2.0 ** -18


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(*shape, dtype=F32, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed)) * scale).to(dtype)


def sizes(nkv, D, P):
    return dict(n_kv_heads=nkv, head_dim=D, page_tokens=P)


def poison(n_pages, nkv, D, P, layers=None):
    """A pool of rows whose factors are not numbers."""
    shape = (n_pages, 2, nkv, K.q4_page_bytes(D, P))
    return torch.full(((layers,) if layers else ()) + shape, 255, dtype=torch.uint8)


def filled(table, lens, nkv, D, P, seed, n_pages, shift=0.3):
    """A pool that holds random rows for every request, NaN factors everywhere else."""
    pool = poison(n_pages, nkv, D, P)
    for b, n in enumerate(lens):
        for pg in range(-(-n // P)):
            page, m = int(table[b, pg]), min(P, n - pg * P)
            rows = rnd(2, nkv, P, D, seed=seed * 1000003 + b * 131 + pg) + shift
            codes, scale, mid = plain.codes_of(rows)
            scale[..., m:], mid[..., m:] = math.nan, math.nan
            pool[page] = plain.pack(codes, scale, mid, P, D)
    return pool


def tables(lens, P, seed, extra_width=0):
    need = [-(-n // P) for n in lens]
    order = torch.randperm(sum(need) + 2, generator=gen(seed)).to(I32)
    t = torch.full((len(lens), max(need) + extra_width), -1, dtype=I32)
    at = 1
    for b, k in enumerate(need):
        t[b, :k] = order[at:at + k]
        at += k
    return t, sum(need) + 2


# ---------------------------------------------------------------------------
# writing and reading


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,D,rot,swap,P,T", [
    (4, 2, 64, 64, False, 16, 1), (7, 1, 128, 128, False, 64, 37), (3, 3, 256, 256, False, 32, 9), (4, 2, 128, 64, False, 48, 21),
    (5, 5, 64, 20, False, 16, 19), (2, 1, 256, 12, False, 16, 5), (4, 4, 128, 128, True, 16, 33), (6, 2, 64, 22, True, 64, 3), (4, 2, 128, 0, False, 64, 40),
])
def test_rows_that_are_written(dtype, nh, nkv, D, rot, swap, P, T):
    qkv = rnd(T, (nh + 2 * nkv) * D, dtype=dtype, seed=T, scale=2.0)
    positions = (torch.arange(T) * 7919 % 100003).to(I32)
    inv = (1e4 ** (-torch.arange(0, rot, 2).double() / max(rot, 1))).float() if rot else None
    n_pages = -(-T // P) + 3
    slots = torch.randperm(n_pages * P, generator=gen(T + 1))[:T].to(I32)
    pool = poison(n_pages, nkv, D, P).to(DEV)
    before = pool.cpu()
    q = torch.zeros(T, nh * D, dtype=dtype, device=DEV)
    weights = torch.full((n_pages, nkv, P), 3.0, device=DEV)
    K.rope_kv_write_q4(qkv.to(DEV), positions.to(DEV), inv.to(DEV) if rot else None, q, pool, slots.to(DEV), n_heads=nh, rot_dim=rot,
                       interleaved=swap, weights=weights, **sizes(nkv, D, P))
    x = qkv.double().view(T, nh + 2 * nkv, D)
    turned = plain.rotate(x[:, : nh + nkv], positions, inv, rot, swap)
    # q: float32 arithmetic (sine and cosine to a few units of 2^-23, two products), one rounding to the model's type
    tol = (2.0 ** -8 if dtype == BF16 else 0) * turned[:, :nh].abs() + 2.0 ** -20 * x.abs().max()
    assert ((q.cpu().double().view(T, nh, D) - turned[:, :nh]).abs() <= tol).all()
    codes, scale, mid = plain.fields(pool, P, D)
    page, off = (slots // P).long(), (slots % P).long()
    for plane, rows in ((0, turned[:, nh:]), (1, x[:, nh + nkv:])):
        c, s, m = codes[page, plane, :, off], scale[page, plane, :, off], mid[page, plane, :, off]
        lo, hi = rows.min(-1).values, rows.max(-1).values
        slack = 2.0 ** -20 * rows.abs().max()
        assert ((s - (hi - lo) / 15).abs() <= 2.0 ** -8 * (hi - lo) / 15 + slack).all()
        assert ((m - (hi + lo) / 2).abs() <= 2.0 ** -8 * (hi + lo).abs() / 2 + slack).all()
        # the cell that an element lies in, for the factors that were stored; an element within 2^-18 of a border may lie on either side
        at = (rows - m.unsqueeze(-1)) / s.unsqueeze(-1) + 8
        near = 2.0 ** -18 * (1 + rows.abs().max() / s.min())
        assert ((c >= torch.floor(at - near).clamp(0, 15)) & (c <= torch.floor(at + near).clamp(0, 15))).all()
        if plane == 1 and dtype == BF16:
            want = plain.codes_of(rows)   # nothing is rounded on the way to a value's row
            assert torch.equal(c, want[0]) and torch.equal(s, want[1]) and torch.equal(m, want[2])
    w = weights.cpu()
    assert (w[page, :, off] == 0).all() and int((w == 0).sum()) == T * nkv
    # nothing but these rows was written
    untouched = torch.ones(n_pages, P, dtype=torch.bool)
    untouched[page, off] = False
    was_c, _, _ = plain.fields(before, P, D)
    assert torch.equal(codes.permute(0, 3, 1, 2, 4)[untouched], was_c.permute(0, 3, 1, 2, 4)[untouched])
    assert torch.isnan(scale.permute(0, 3, 1, 2)[untouched]).all()


def test_rows_without_a_range_and_rows_that_are_not_finite():
    nh, nkv, D, P, T = 1, 1, 128, 16, 9
    qkv = rnd(T, 3 * D, seed=4)
    v = qkv[:, 2 * D:]
    v[0] = 1.5
    v[1] = 0.0
    v[2, 5] = math.inf
    v[3, 7] = -math.inf
    v[4, 127] = math.nan
    v[5] = torch.linspace(-3e38, 3e38, D)            # (float32 steps overflow: infinities and NaN)
    v[6] = torch.linspace(-3e38, 3e38, D, dtype=torch.float64).float()
    assert not torch.isfinite(v[5]).all() and torch.isfinite(v[6]).all()
    v[7] *= 1e-36
    v[8] = torch.where(torch.arange(D) < 64, 1.0, -1.0) * 1e-44   # (subnormal)
    pool = poison(1, nkv, D, P).to(DEV)
    K.rope_kv_write_q4(qkv.to(DEV), torch.zeros(T, dtype=I32, device=DEV), None, torch.empty(T, D, device=DEV), pool,
                       torch.arange(T, dtype=I32, device=DEV), n_heads=nh, rot_dim=0, interleaved=False, **sizes(nkv, D, P))
    got = plain.values(pool, P, D)[0, 1, 0]
    assert (got[0] == 1.5).all() and (got[1] == 0).all()
    assert torch.isnan(got[2:6]).all()
    step = 6e38 / 15
    assert ((got[6] - v[6].double()).abs() <= step * (0.5 + 2.0 ** -8 * 7.5)).all()
    for i in (7, 8):
        codes, scale, mid = plain.codes_of(v[i].double())
        c, s, m = (f[0, 1, 0, i] for f in plain.fields(pool, P, D))
        assert torch.equal(c, codes) and s == scale and m == mid


def test_q_alone_is_rotated_where_another_call_owns_the_cache():
    nh, nkv, D, P, T = 2, 1, 64, 16, 5
    qkv, inv = rnd(T, 4 * D, seed=8, dtype=BF16), torch.ones(32)
    pool = poison(2, nkv, D, P).to(DEV)
    q = torch.zeros(T, nh * D, dtype=BF16, device=DEV)
    K.rope_kv_write_q4(qkv.to(DEV), torch.arange(T, dtype=I32, device=DEV), inv.to(DEV), q, pool, torch.arange(T, dtype=I32, device=DEV), n_heads=nh,
                       rot_dim=64, interleaved=False, write_kv=False, **sizes(nkv, D, P))
    assert (pool == 255).all()
    want = plain.rotate(qkv.double().view(T, 4, D)[:, :nh], torch.arange(T), inv, 64, False)
    assert ((q.cpu().double().view(T, nh, D) - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nkv,D,P,lens", [(2, 64, 16, [1, 16, 17, 100]), (1, 128, 64, [130]), (3, 256, 32, [31, 33])])
def test_expand(dtype, nkv, D, P, lens):
    table, n_pages = tables(lens, P, 5, extra_width=1)
    pool = filled(table, lens, nkv, D, P, 6, n_pages)
    if len(lens) > 2:
        table[3, 0] = -1   # a page that went back
    out = torch.full((n_pages, 2, nkv, P, D), 7.0, dtype=dtype, device=DEV)
    ctx = torch.tensor([n - 1 for n in lens], dtype=I32)
    segs = torch.tensor(list(range(len(lens)))[::-1], dtype=I32)
    K.expand_q4(pool.to(DEV), out, segs=segs.to(DEV), n_segs=len(lens), seg_ctx=ctx.to(DEV), seg_qn=torch.ones(len(lens), dtype=I32, device=DEV),
                block_table=table.to(DEV), max_keys=max(lens), **sizes(nkv, D, P))
    want = torch.full((n_pages, 2, nkv, P, D), 7.0, dtype=dtype)
    all_values = plain.values(pool, P, D).float()   # (exact: one sum of 24 bits)
    for b, n in enumerate(lens):
        for t in range(n):
            page = int(table[b, t // P])
            if page >= 0:
                want[page, :, :, t % P] = all_values[page, :, :, t % P].to(dtype)
    assert torch.equal(out.cpu(), want)


# ---------------------------------------------------------------------------
# attention of single tokens


def run_decode(q, pool, table, lens, H, kv, D, P, weights=None, stream_args=None, part_units=None, dup=None, **mask):
    B = len(lens)
    dt = q.dtype
    items = torch.arange(B, dtype=I32) if dup is None else torch.tensor(dup, dtype=I32)
    n = len(items)
    rows = torch.arange(B, dtype=I32)
    ctx = torch.tensor([x - 1 for x in lens], dtype=I32)
    units = K.decode_units_q4(n, H, DEV, fixed_ranges=mask.get("keep_first", 0) > 0) if part_units is None else part_units
    out = torch.full((B, H * D), 9.0, dtype=dt, device=DEV)
    counters = torch.zeros(n * H, dtype=I32, device=DEV)
    scores = torch.empty(n * H * table.shape[1] * P, device=DEV) if weights is not None else None
    extra = 2 * n * H + 8 if weights is not None else 0
    args = dict(mask)
    args.setdefault("window", 0)
    for k in ("slopes", "sink"):
        if isinstance(args.get(k), torch.Tensor):
            args[k] = args[k].to(DEV)
    K.attn_decode_q4(q.to(DEV), pool, out, seg_q0=rows.to(DEV), seg_ctx=ctx.to(DEV), block_table=table.to(DEV), items=items.to(DEV), n_items=n,
                     n_heads=H, scale=D ** -0.5, part_o=torch.empty(units * D + extra, device=DEV), part_ml=torch.empty(2 * units, device=DEV),
                     counters=counters, weights=weights, scores=scores, **args, **sizes(kv, D, P))
    assert not counters.any()
    assert K.attn_q4_error() == 0
    return out, ctx


def check(out, ref, dtype, H, D):
    want, step, mass, _ = ref
    got = out.cpu().double().view(-1, H, D)
    tol = SUMS * mass + (2.0 ** -8 * want.abs() + step if dtype == BF16 else 0)
    worst = ((got - want).abs() / tol).max()
    assert worst <= 1, f"off by {float(worst):.2f} times the bound"


DECODE = [
    # heads, kv heads, size, page, lengths
    (4, 4, 64, 16, [1]), (4, 4, 128, 64, [1, 2, 15, 16, 17, 33]), (7, 1, 128, 64, [63, 64, 65, 200]), (28, 4, 128, 64, [500, 3, 129]),
    (16, 2, 64, 32, [97, 31]), (12, 1, 128, 16, [45, 160]), (20, 1, 64, 48, [100]), (9, 1, 256, 32, [70, 5]), (3, 3, 256, 16, [40]), (2, 1, 128, 128, [300, 129, 128]),
    (40, 2, 128, 64, [70]),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,kv,D,P,lens", DECODE)
def test_decode(dtype, H, kv, D, P, lens):
    table, n_pages = tables(lens, P, 3, extra_width=2)
    pool = filled(table, lens, kv, D, P, 11, n_pages).to(DEV)
    q = rnd(len(lens), H * D, dtype=dtype, seed=12, scale=1.5)
    out, ctx = run_decode(q, pool, table, lens, H, kv, D, P)
    check(out, plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5), dtype, H, D)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,kv,D,P", [(7, 1, 128, 64), (4, 4, 64, 48), (2, 1, 256, 16)])
def test_decode_at_every_cut(dtype, H, kv, D, P):
    """Lengths and numbers of requests that end ranges, stages and pages at many places.  Values are sums of few terms, so the output's error is that
    of the weights alone: float32 to a few units of 2^-22 of the rows' sizes."""
    for lens in ([33 * i + 7 for i in range(12)], [641], [16 * i + 1 for i in range(1, 30)], [1000, 17, 480, 481, 479, 64, 63], [48, 80, 112, 144, 176, 208, 240]):
        table, n_pages = tables(lens, P, 25)
        pool = filled(table, lens, kv, D, P, 26, n_pages).to(DEV)
        q = rnd(len(lens), H * D, dtype=dtype, seed=27, scale=1.5)
        out, ctx = run_decode(q, pool, table, lens, H, kv, D, P)
        ref = plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5)
        check(out, ref, dtype, H, D)
        if dtype == F32:
            # the norm of a request's error: scores of up to some ten, each off by some units of 2^-24, and as many roundings of the sums
            err = (out.cpu().double().view(-1, H * D) - ref[0].view(-1, H * D)).norm(dim=1) / ref[0].view(-1, H * D).norm(dim=1)
            assert float(err.max()) <= 2.0 ** -18


MASKS = [dict(window=1), dict(window=40), dict(window=100, keep_first=5), dict(window=33, keep_first=70), dict(chunk=48), dict(sink=True), dict(window=20, sink=True, keep_first=3),
         dict(sink="learned"), dict(slopes=True), dict(slopes=True, window=50)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mask", MASKS, ids=lambda m: "-".join(f"{k}{v}" for k, v in m.items()))
@pytest.mark.parametrize("H,kv,D,P", [(8, 2, 64, 16), (12, 1, 128, 64)])
def test_decode_masks(dtype, mask, H, kv, D, P):
    lens = [1, 20, 97, 260]
    table, n_pages = tables(lens, P, 21)
    pool = filled(table, lens, kv, D, P, 22, n_pages).to(DEV)
    q = rnd(len(lens), H * D, dtype=dtype, seed=23, scale=1.5)
    m, ref = dict(mask), dict(mask)
    if m.get("slopes"):
        m["slopes"] = ref["slopes"] = 0.05 * (1 + torch.arange(H).float())
    if m.get("sink") == "learned":
        m["sink"] = ref["sink"] = rnd(H, seed=24)
    if m.get("window"):
        # pages that no key in sight lies in have gone back
        for b, n in enumerate(lens):
            for pg in range(-(-n // P)):
                if not any(plain.in_sight(t, n - 1, m["window"], m.get("keep_first", 0), 0) for t in range(pg * P, min(n, pg * P + P))):
                    table[b, pg] = -1
    out, ctx = run_decode(q, pool, table, lens, H, kv, D, P, **m)
    check(out, plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5, **ref), dtype, H, D)


def test_decode_with_the_least_scratch_and_many_requests():
    H, kv, D, P = 6, 2, 64, 16
    lens = [1 + (37 * i) % 90 for i in range(300)]
    table, n_pages = tables(lens, P, 31)
    pool = filled(table, lens, kv, D, P, 32, n_pages).to(DEV)
    q = rnd(len(lens), H * D, dtype=BF16, seed=33)
    ref = plain.decode(q, pool, table, torch.tensor(lens) - 1, H, kv, D, P, D ** -0.5)
    for units in (len(lens) * H, None):
        out, _ = run_decode(q, pool, table, lens, H, kv, D, P, part_units=units)
        check(out, ref, BF16, H, D)


def test_scores_far_apart_and_rows_that_are_not_numbers():
    """A head whose scores reach hundreds, with the largest first, last and rising; and a request with a row that is not finite, which
    spoils its own output and no other's."""
    H, kv, D, P = 2, 1, 128, 64
    lens = [200, 200, 200]
    table, n_pages = tables(lens, P, 41)
    pool = poison(n_pages, kv, D, P)
    for b, n in enumerate(lens):
        size = torch.linspace(60, 0.1, n) if b == 0 else torch.linspace(0.1, 60, n)
        rows = rnd(2, n, D, seed=42 + b)
        rows[0] = torch.sign(rnd(1, D, seed=50)) * size[:, None] * (1 + 0.02 * rnd(n, D, seed=51))
        if b == 2:
            rows[1, 77, 3] = math.nan
        codes, scale, mid = plain.codes_of(rows)
        bad = ~torch.isfinite(rows).all(-1)
        scale[bad] = math.nan
        for pg in range(-(-n // P)):
            m = min(P, n - pg * P)
            full = [torch.zeros(2, 1, P, D, dtype=torch.int64), torch.full((2, 1, P), math.nan, dtype=torch.float64), torch.zeros(2, 1, P, dtype=torch.float64)]
            for f, x in zip(full, (codes, scale, mid)):
                f[:, 0, :m] = x[:, pg * P:pg * P + m]
            pool[int(table[b, pg])] = plain.pack(*full, P, D)
    q = torch.cat([torch.sign(rnd(1, D, seed=50)), rnd(1, D, seed=52)], 0).reshape(1, -1).repeat(3, 1).to(BF16)
    out, ctx = run_decode(q, pool.to(DEV), table, lens, H, kv, D, P)
    ref = plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5)
    check(out[:2], tuple(x[:2] for x in ref[:3]) + (None,), BF16, H, D)
    assert torch.isnan(out[2]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_query_that_is_not_finite(dtype, value):
    """... spoils its own head's output and no other's."""
    H, kv, D, P = 6, 2, 128, 64
    lens = [70, 130]
    table, n_pages = tables(lens, P, 71)
    pool = filled(table, lens, kv, D, P, 72, n_pages).to(DEV)
    q = rnd(2, H * D, dtype=dtype, seed=73)
    ref = plain.decode(q, pool, table, torch.tensor(lens) - 1, H, kv, D, P, D ** -0.5)
    q[1, 4 * D + 9] = value
    out, _ = run_decode(q, pool, table, lens, H, kv, D, P)
    got = out.view(2, H, D)
    assert torch.isnan(got[1, 4]).all()
    got[1, 4] = ref[0][1, 4].to(DEV, dtype)
    check(out, ref, dtype, H, D)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_queries_of_very_different_sizes(dtype):
    """Heads of 2^-100 to 2^100, heads of zeros, and heads with one element 2^10 times the others.  Whole numbers of 16 bits hold such a head's small elements to
    2^-15 of the largest: half a unit each, so a score is off by at most that times the row's sum of |scale (code - 7.5)|, and a weight by as much of itself."""
    H, kv, D, P = 8, 1, 128, 64
    lens = [150]
    table, n_pages = tables(lens, P, 81)
    pool = filled(table, lens, kv, D, P, 82, n_pages)
    q = rnd(1, H * D, seed=83).view(H, D)
    q[0] *= 2.0 ** -100
    q[1] *= 2.0 ** -110
    q[2] = 0
    q[3, 5], q[4, 127] = 2.0 ** 10, -2.0 ** 10
    q = q.reshape(1, -1).to(dtype)
    out, ctx = run_decode(q, pool.to(DEV), table, lens, H, kv, D, P)
    ref = plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5)
    if dtype == BF16:
        got, want = out.cpu().double().view(H, D), ref[0][0]
        codes, scale, mid = plain.fields(pool[table[0, :3].long()], P, D)
        live = torch.arange(3 * P) < lens[0]
        rows = (scale.unsqueeze(-1) * (codes.double() - 7.5)).abs()[:, 0, 0].reshape(-1, D).sum(1)[live]
        values = plain.values(pool[table[0, :3].long()], P, D)[:, 1, 0].reshape(-1, D)[live].abs().max()
        for h in (3, 4):
            off = float(2.0 ** -15 * 2.0 ** 10 * rows.max() * D ** -0.5)    # of a score; the weights' change is at most twice that of their sum
            assert ((got[h] - want[h]).abs() <= 2 * off * values + 2.0 ** -8 * want[h].abs() + ref[1][0, h] + SUMS * ref[2][0, h]).all()
            out.view(H, D)[h] = want[h].to(DEV, dtype)
    check(out, ref, dtype, H, D)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["spread", "hidden", "large", "level"])
def test_values_of_very_different_sizes(dtype, kind):
    """Rows of v from 2^-30 to 2^30 side by side; rows 2^60 times the others' size whose keys weigh nothing; rows near the type's largest number; and
    rows far from zero with little range.  (The bound is relative to what the keys contribute, as everywhere.)"""
    H, kv, D, P = 5, 1, 128, 64
    lens = [200, 63]
    table, n_pages = tables(lens, P, 91)
    pool = poison(n_pages, kv, D, P)
    side = torch.sign(rnd(1, D, seed=92))
    for b, n in enumerate(lens):
        k, v = 0.02 * rnd(n, D, seed=93 + b), rnd(n, D, seed=95 + b)
        if kind == "spread":
            v *= 2.0 ** torch.randint(-30, 31, (n, 1), generator=gen(97)).float()
        elif kind == "hidden":
            big = torch.arange(n) % 5 == 2
            v[big] *= 2.0 ** 60
            k[big] -= 30 * side          # (scores about 300 below the others')
        elif kind == "large":
            v *= 2.0 ** 120 / v.abs().max()
        else:
            v = 2.0 ** 118 * (1 + 2.0 ** -6 * v)
        codes, scale, mid = plain.codes_of(torch.stack([k, v]))
        for pg in range(-(-n // P)):
            m = min(P, n - pg * P)
            full = [torch.zeros(2, 1, P, D, dtype=torch.int64), torch.full((2, 1, P), math.nan, dtype=torch.float64), torch.zeros(2, 1, P, dtype=torch.float64)]
            for f, x in zip(full, (codes, scale, mid)):
                f[:, 0, :m] = x[:, pg * P:pg * P + m]
            pool[int(table[b, pg])] = plain.pack(*full, P, D)
    q = (side * (1 + 0.01 * rnd(H, D, seed=99))).reshape(1, -1).repeat(2, 1).to(dtype)
    out, ctx = run_decode(q, pool.to(DEV), table, lens, H, kv, D, P)
    assert torch.isfinite(out).all()
    check(out, plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5), dtype, H, D)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,kv,D,P,lens", [(4, 4, 128, 64, [1, 70, 130]), (7, 1, 64, 16, [33, 18]), (20, 1, 128, 32, [50]), (6, 2, 256, 16, [20, 1])])
def test_decode_adds_the_weights_up(dtype, H, kv, D, P, lens):
    table, n_pages = tables(lens, P, 61, extra_width=1)
    pool = filled(table, lens, kv, D, P, 62, n_pages).to(DEV)
    q = rnd(len(lens), H * D, dtype=dtype, seed=63)
    start = rnd(n_pages, kv, P, seed=64).abs()
    weights = start.to(DEV)
    out, ctx = run_decode(q, pool, table, lens, H, kv, D, P, weights=weights, sink=True)
    ref = plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5, sink=True)
    check(out, ref, dtype, H, D)
    want = start.double().clone()
    for (page, h, off), w in ref[3].items():
        want[page, h, off] += w
    # a weight of up to one per head: the scores' float32 sums, the exponential, the running sum
    assert ((weights.cpu().double() - want).abs() <= 2.0 ** -17 * (H // kv) + 2.0 ** -22 * want).all()
    again = start.to(DEV)
    run_decode(q, pool, table, lens, H, kv, D, P, weights=again, sink=True)
    assert torch.equal(again, weights)   # the same bits
    # slots that no key of these requests lies in are as they were
    held = torch.zeros(n_pages, P, dtype=torch.bool)
    for (page, _, off) in ref[3]:
        held[page, off] = True
    assert torch.equal(weights.cpu().permute(0, 2, 1)[~held], start.permute(0, 2, 1)[~held])


def test_addresses_that_break_the_alignment_are_refused():
    H, kv, D, P, lens = 2, 2, 64, 16, [20]
    table, n_pages = tables(lens, P, 68)
    pool = filled(table, lens, kv, D, P, 69, n_pages).to(DEV)
    off = lambda n: torch.zeros(n + 1, device=DEV)[1:]  # noqa: E731
    with pytest.raises(K.KernelError, match="weights and scores"):
        run_decode(rnd(1, H * D), pool, table, lens, H, kv, D, P, weights=off(n_pages * kv * P).view(n_pages, kv, P))
    i32 = lambda x: torch.tensor(x, dtype=I32, device=DEV)  # noqa: E731
    kw = dict(seg_q0=i32([0]), seg_ctx=i32([19]), block_table=table.to(DEV), items=i32([0]), n_items=1, n_heads=H, scale=1.0, window=0,
              counters=torch.zeros(H, dtype=I32, device=DEV), **sizes(kv, D, P))
    q, out = torch.zeros(1, H * D, device=DEV), torch.zeros(1, H * D, device=DEV)
    for over, says in ((dict(part_o=off(64 * D)), "part_o"), (dict(part_ml=off(64)), "part_ml")):
        with pytest.raises(K.KernelError, match=says):
            K.attn_decode_q4(q, pool, out, **{**kw, "part_o": torch.zeros(64 * D, device=DEV), "part_ml": torch.zeros(64, device=DEV), **over})
    with pytest.raises(K.KernelError, match="q, the pool"):
        K.attn_decode_q4(off(H * D).view(1, -1), pool, out, part_o=torch.zeros(64 * D, device=DEV), part_ml=torch.zeros(64, device=DEV), **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,kv,D,lens", [(8, 2, 256, [9]), (8, 2, 128, [9, 300]), (4, 4, 128, [1500]), (7, 1, 64, [40]), (24, 2, 128, [70])])
def test_weights_are_float32(dtype, H, kv, D, lens):
    """Whatever the model's type: scores of up to ten, formed in three roundings of half a unit of 2^-23, move a weight by 1.3e-6 of itself at most, q's
    24 or 22 bits by less; in the norm over the keys that is below 2^-19."""
    P = 64
    for seed in (12, 13, 14):
        table, n_pages = tables(lens, P, 3)
        pool = filled(table, lens, kv, D, P, 11, n_pages).to(DEV)
        q = rnd(len(lens), H * D, dtype=dtype, seed=seed)
        weights = torch.zeros(n_pages, kv, P, device=DEV)
        out, ctx = run_decode(q, pool, table, lens, H, kv, D, P, weights=weights)
        ref = plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5)
        want = torch.zeros(n_pages, kv, P, dtype=torch.float64)
        for (page, h, off), w in ref[3].items():
            want[page, h, off] += w
        assert float((weights.cpu().double() - want).norm() / want.norm()) <= 2.0 ** -19


def test_weights_of_long_requests():
    """Lengths around what a block of the adding kernel takes."""
    H, kv, D, P = 4, 2, 64, 64
    lens = [256, 257, 1023, 1024, 1025, 2100]
    table, n_pages = tables(lens, P, 65)
    pool = filled(table, lens, kv, D, P, 66, n_pages).to(DEV)
    q = rnd(len(lens), H * D, dtype=F32, seed=67)
    weights = torch.zeros(n_pages, kv, P, device=DEV)
    out, ctx = run_decode(q, pool, table, lens, H, kv, D, P, weights=weights)
    ref = plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5)
    check(out, ref, F32, H, D)
    want = torch.zeros(n_pages, kv, P, dtype=torch.float64)
    for (page, h, off), w in ref[3].items():
        want[page, h, off] += w
    # (scores of up to some ten, off by some units of 2^-24 each: a weight by as much of itself)
    assert ((weights.cpu().double() - want).abs() <= 2.0 ** -17 * want).all()


def test_calls_at_the_same_time_with_scratch_of_their_own():
    H, kv, D, P = 8, 2, 128, 64
    cases = []
    for i, lens in enumerate(([700, 30, 1500], [64] * 20)):
        table, n_pages = tables(lens, P, 101 + i)
        pool = filled(table, lens, kv, D, P, 103 + i, n_pages).to(DEV)
        q = rnd(len(lens), H * D, dtype=BF16, seed=105 + i).to(DEV)
        n, units = len(lens), K.decode_units_q4(len(lens), H, DEV)
        i32 = lambda x: torch.tensor(x, dtype=I32, device=DEV)  # noqa: E731
        kw = dict(seg_q0=i32(list(range(n))), seg_ctx=i32([x - 1 for x in lens]), block_table=table.to(DEV), items=i32(list(range(n))), n_items=n, n_heads=H,
                  scale=D ** -0.5, window=0, part_o=torch.empty(units * D, device=DEV), part_ml=torch.empty(2 * units, device=DEV),
                  counters=torch.zeros(n * H, dtype=I32, device=DEV), **sizes(kv, D, P))
        want, _ = run_decode(q, pool, table, lens, H, kv, D, P)
        cases.append((torch.cuda.Stream(), q, pool, torch.empty_like(q), kw, want))
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, q, pool, out, kw, _ in cases:
            with torch.cuda.stream(stream):
                out.fill_(9.0)
                K.attn_decode_q4(q, pool, out, **kw)
        torch.cuda.synchronize()
        for _, _, _, out, kw, want in cases:
            assert torch.equal(out, want) and not kw["counters"].any()


def test_weights_of_a_request_that_is_listed_twice():
    H, kv, D, P, lens = 4, 2, 64, 16, [40, 40]
    table, n_pages = tables([40], P, 71)
    table = table.repeat(2, 1)   # two segments of the same pages
    pool = filled(table[:1], [40], kv, D, P, 72, n_pages).to(DEV)
    q = rnd(1, H * D, seed=73).repeat(2, 1)
    weights = torch.zeros(n_pages, kv, P, device=DEV)
    run_decode(q, pool, table, lens, H, kv, D, P, weights=weights)
    assert abs(float(weights.sum()) - 2 * H) <= 2.0 ** -16 * 2 * H


# ---------------------------------------------------------------------------
# eviction


def evicted(pool, weights, table, dst, lens, keep, first, recent, kv, D, P):
    """What ``evict_q4`` should leave: (kept, pool, weights) of one layer."""
    pool, weights = pool.clone(), weights.clone()
    was_c, was_s, was_m = plain.fields(pool, P, D)
    raw = pool.clone()
    kept = torch.full((len(lens), kv, keep), -1, dtype=I32)
    new_w = weights.clone()
    for b, n in enumerate(lens):
        for h in range(kv):
            w = [float(weights[int(table[b, t // P]), h, t % P]) for t in range(n)]
            idx = plain.stay(w, keep, first, recent)
            kept[b, h, : len(idx)] = torch.tensor(idx, dtype=I32)
            for j, t in enumerate(idx):
                a, i, c, k = int(table[b, t // P]), t % P, int(dst[b, j // P]), j % P
                new_w[c, h, k] = weights[a, h, i]
                for plane in (0, 1):
                    row = D // 2
                    pool[c, plane, h, k * row:(k + 1) * row] = raw[a, plane, h, i * row:(i + 1) * row]
                    f = P * row
                    pool[c, plane, h, f + 4 * k: f + 4 * k + 4] = raw[a, plane, h, f + 4 * i: f + 4 * i + 4]
    return kept, pool, new_w


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kv,D,P,lens,keep,first,recent", [
    (1, 64, 16, [1], 1, 0, 0), (2, 128, 16, [40, 3, 17], 16, 2, 5), (3, 64, 64, [300, 64, 65], 64, 0, 64), (2, 256, 32, [90, 200], 77, 10, 0),
    (1, 128, 64, [1500], 1, 0, 0), (1, 128, 64, [1300, 900], 700, 4, 100), (4, 64, 16, [33], 40, 1, 1), (2, 64, 16, [100], 50, 50, 0), (1, 64, 16, [1200], 1100, 0, 3),
])
def test_evict(in_place, kv, D, P, lens, keep, first, recent):
    L = 3
    table, n_pages = tables(lens, P, 81, extra_width=1)
    width = -(-min(keep, max(lens)) // P)
    dst = table if in_place else n_pages + torch.randperm(len(lens) * width, generator=gen(82)).to(I32).view(len(lens), width)
    total = n_pages + len(lens) * width
    pool = torch.randint(0, 256, (L, total, 2, kv, K.q4_page_bytes(D, P)), generator=gen(83), dtype=torch.uint8)
    weights = rnd(L, total, kv, P, seed=84).abs()
    weights[1] = (weights[1] * 3).round()           # many ties
    weights[2, :, :, ::3] = math.nan
    weights[2, :, :, 1::3] = -0.0
    weights[2, :, :, 2::6] = -math.inf
    kept = torch.full((L, len(lens), kv, keep), 77, dtype=I32, device=DEV)
    dpool, dweights = pool.to(DEV), weights.to(DEV)
    t = table.to(DEV)
    K.evict_q4(dpool, dweights, block_table=t, dst_table=None if in_place else dst.to(DEV), n_tokens=torch.tensor(lens, dtype=I32, device=DEV),
               n_items=len(lens), keep=keep, first=first, recent=recent, kept=kept, max_tokens=max(lens), **sizes(kv, D, P))
    for l in range(L):
        want = evicted(pool[l], weights[l], table, dst, lens, keep, first, recent, kv, D, P)
        assert torch.equal(kept[l].cpu(), want[0]), f"layer {l}"
        assert torch.equal(dpool[l].cpu(), want[1])
        assert torch.equal(dweights[l].cpu().view(I32), want[2].view(I32))


@pytest.mark.parametrize("n,keep,first,recent", [(9000, 4000, 4, 300), (8193, 8192, 0, 0), (8192, 1, 0, 0), (8194, 5000, 1, 1), (20000, 19999, 0, 7)])
@pytest.mark.parametrize("kind", ["close", "equal", "wide", "two", "infinite", "negative"])
def test_which_keys_stay(n, keep, first, recent, kind):
    """The choice alone, over weights that crowd a few numbers or span all of float32, against a sort (ties: the earlier key)."""
    kv, D, P = 1, 64, 64
    pages = -(-n // P)
    w = {"close": lambda: 1 + 1e-6 * rnd(pages * P, seed=n).abs(), "equal": lambda: torch.full((pages * P,), 0.25),
         "wide": lambda: torch.exp(40 * rnd(pages * P, seed=n)), "two": lambda: (rnd(pages * P, seed=n) > 0).float(),
         "infinite": lambda: torch.where(rnd(pages * P, seed=n) > 0, math.inf, rnd(pages * P, seed=n + 1)), "negative": lambda: rnd(pages * P, seed=n).round(decimals=2)}[kind]()
    pool = torch.zeros(1, pages, 2, kv, K.q4_page_bytes(D, P), dtype=torch.uint8, device=DEV)
    kept = torch.empty(1, 1, kv, keep, dtype=I32, device=DEV)
    K.evict_q4(pool, w.view(1, pages, kv, P).to(DEV), block_table=torch.arange(pages, dtype=I32, device=DEV).view(1, -1), n_items=1, keep=keep, first=first,
               n_tokens=torch.tensor([n], dtype=I32, device=DEV), recent=recent, kept=kept, max_tokens=n, **sizes(kv, D, P))
    rank = w[:n].double()
    rank[:first] = rank[n - recent:] = math.inf
    order = torch.argsort(rank, descending=True, stable=True)
    if kind == "infinite":   # (the first and the last stay whatever the others are)
        sure = torch.zeros(n, dtype=torch.bool)
        sure[:first] = sure[n - recent:] = True
        order = torch.cat([sure.nonzero().view(-1), order[~sure[order]]])
    assert kept.view(-1).tolist() == sorted(order[:keep].tolist())


def test_evict_from_a_request_longer_than_shared_memory_holds():
    kv, D, P, n, keep = 1, 64, 64, 60001, 12345
    table = torch.arange(-(-n // P), dtype=I32).view(1, -1)
    pool = torch.randint(0, 256, (1, table.shape[1], 2, kv, K.q4_page_bytes(D, P)), generator=gen(91), dtype=torch.uint8).to(DEV)
    weights = (rnd(1, table.shape[1], kv, P, seed=92).abs() * 50).round().to(DEV)
    kept = torch.empty(1, 1, kv, keep, dtype=I32, device=DEV)
    want = plain.stay(weights.cpu().view(-1)[:n].tolist(), keep, 3, 1000)
    rows = pool[0, :, 0, 0, : P * 32].reshape(-1, 32)[:n].clone()
    K.evict_q4(pool, weights, block_table=table.to(DEV), n_tokens=torch.tensor([n], dtype=I32, device=DEV), n_items=1, keep=keep, first=3,
               recent=1000, kept=kept, max_tokens=n, **sizes(kv, D, P))
    assert kept.view(-1).tolist() == want
    assert torch.equal(pool[0, :, 0, 0, : P * 32].reshape(-1, 32)[:keep], rows[torch.tensor(want, device=DEV)])


# ---------------------------------------------------------------------------
# together


def test_write_attend_weigh_evict_and_go_on():
    """Three requests decode against the cache, give up half of their keys and decode on; the same in plain form, from the pool's own rows."""
    H, kv, D, P, keep, first, recent = 4, 2, 64, 16, 24, 2, 6
    lens = [50, 31, 40]
    table, n_pages = tables(lens, P, 101, extra_width=1)
    pool, weights = poison(n_pages, kv, D, P).to(DEV), torch.full((n_pages, kv, P), math.nan, device=DEV)
    inv = (1e4 ** (-torch.arange(0, D, 2).double() / D)).float()
    total = [0.0] * 3

    def write(b, t0, n, slot0, seed):
        qkv = rnd(n, (H + 2 * kv) * D, seed=seed)
        q = torch.empty(n, H * D, device=DEV)
        at = torch.arange(slot0, slot0 + n)
        slots = (table[b, at // P] * P + at % P).to(I32)
        K.rope_kv_write_q4(qkv.to(DEV), torch.arange(t0, t0 + n, dtype=I32, device=DEV), inv.to(DEV), q, pool, slots.to(DEV), n_heads=H, rot_dim=D,
                           interleaved=False, weights=weights, **sizes(kv, D, P))
        return q

    def attend(q, now):
        before = weights.clone()
        out, ctx = run_decode(q, pool, table, now, H, kv, D, P, weights=weights)
        ref = plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5)
        check(out, ref, F32, H, D)
        want = before.cpu().double()
        for at, w in ref[3].items():
            want[at] += w
        held = ~torch.isnan(want)
        assert ((weights.cpu().double() - want)[held].abs() <= 2.0 ** -16).all() and torch.isnan(weights.cpu()[~held]).all()

    q = torch.cat([write(b, 0, n, 0, 110 + b)[-1:] for b, n in enumerate(lens)])
    attend(q, lens)
    before, w_before = pool.cpu(), weights.cpu()
    kept = torch.empty(1, 3, kv, keep, dtype=I32, device=DEV)
    K.evict_q4(pool.unsqueeze(0), weights.unsqueeze(0), block_table=table.to(DEV), n_tokens=torch.tensor(lens, dtype=I32, device=DEV), n_items=3,
               keep=keep, first=first, recent=recent, kept=kept, max_tokens=max(lens), **sizes(kv, D, P))
    want = evicted(before, w_before, table, table, lens, keep, first, recent, kv, D, P)
    assert torch.equal(kept[0].cpu(), want[0]) and torch.equal(pool.cpu(), want[1])
    for step in range(3):
        now = [keep + step + 1] * 3
        q = torch.cat([write(b, n + step, 1, keep + step, 120 + 3 * step + b) for b, n in enumerate(lens)])
        attend(q, now)


def test_captured_and_replayed_with_other_lengths_and_on_another_stream():
    H, kv, D, P = 8, 2, 128, 64
    long = [300, 130]
    table, n_pages = tables(long, P, 131)
    pool = filled(table, long, kv, D, P, 132, n_pages).to(DEV)
    q = rnd(2, H * D, dtype=BF16, seed=133).to(DEV)
    out = torch.zeros(2, H * D, dtype=BF16, device=DEV)
    weights = torch.zeros(n_pages, kv, P, device=DEV)
    units = K.decode_units_q4(2, H, DEV)
    ctx = torch.tensor([9, 5], dtype=I32, device=DEV)
    st = dict(seg_q0=torch.arange(2, dtype=I32, device=DEV), seg_ctx=ctx, block_table=table.to(DEV), items=torch.arange(2, dtype=I32, device=DEV),
              n_items=2, n_heads=H, window=0, scale=D ** -0.5, part_o=torch.empty(units * D + 64, device=DEV), part_ml=torch.empty(2 * units, device=DEV),
              counters=torch.zeros(2 * H, dtype=I32, device=DEV), weights=weights, scores=torch.empty(2 * H * table.shape[1] * P, device=DEV), **sizes(kv, D, P))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.attn_decode_q4(q, pool, out, **st)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    ref = plain.decode(q, pool, table, [9, 5], H, kv, D, P, D ** -0.5)
    check(out, ref, BF16, H, D)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g), K.pdl_scope():
        K.attn_decode_q4(q, pool, out, **st)
    for now in ([300, 130], [1, 2], [64, 65]):
        ctx.copy_(torch.tensor(now, dtype=I32) - 1)
        out.zero_()
        weights.zero_()
        g.replay()
        torch.cuda.synchronize()
        ref = plain.decode(q, pool, table, [n - 1 for n in now], H, kv, D, P, D ** -0.5)
        check(out, ref, BF16, H, D)
        assert abs(float(weights.sum()) - 2 * H) <= 2.0 ** -16 * 2 * H


def test_rows_far_into_a_large_pool():
    """Offsets beyond 32 bits: pages at the end of a pool of more than 4 GB."""
    H, kv, D, P = 2, 1, 64, 64
    n_pages = (1 << 32) // (2 * kv * K.q4_page_bytes(D, P)) + 40
    pool = torch.empty(n_pages, 2, kv, K.q4_page_bytes(D, P), dtype=torch.uint8, device=DEV)
    lens = [100]
    small, _ = tables(lens, P, 141)
    table = torch.tensor([[n_pages - 1, n_pages - 7]], dtype=I32)
    rows = filled(small, lens, kv, D, P, 142, 4).to(DEV)
    pool[table[0].long().to(DEV)] = rows[small[0].long().to(DEV)]
    q = rnd(1, H * D, dtype=BF16, seed=143)
    out, ctx = run_decode(q, pool, table, lens, H, kv, D, P)
    check(out, plain.decode(q, rows, small, ctx, H, kv, D, P, D ** -0.5), BF16, H, D)
    qkv = rnd(3, (H + 2) * D, dtype=BF16, seed=144)
    slots = torch.tensor([(n_pages - 7) * P + 40 + i for i in range(3)], dtype=torch.int64)
    assert int(slots.max()) < 1 << 31
    K.rope_kv_write_q4(qkv.to(DEV), torch.zeros(3, dtype=I32, device=DEV), None, torch.empty(3, H * D, dtype=BF16, device=DEV), pool, slots.to(I32).to(DEV),
                       n_heads=H, rot_dim=0, interleaved=False, **sizes(kv, D, P))
    got = plain.fields(pool[n_pages - 7: n_pages - 6], P, D)[0][0, 1, 0, 40:43]
    assert torch.equal(got, plain.codes_of(qkv.double()[:, 3 * D:])[0])
