"""The cache held in 4 bits at the ends of its range, on the GPU, against tests/plain_q4.py in 64 bits: rows of very different sizes beside one
another, and how exact the weights and outputs are whatever the rows hold.  Bounds are derived at each test."""
import math

import pytest
import torch

import locus_b200.kernels as K
import plain_q4 as plain
from test_cache_q4_gpu import BF16, DECODE, DEV, F32, SUMS, check, filled, poison, rnd, run_decode, tables

pytestmark = pytest.mark.gpu


def pool_of(table, n_pages, rows, P):
    """A pool of one key/value head that holds rows[b] [2, n, D] (keys, values) of request b."""
    D = rows[0].shape[-1]
    pool = poison(n_pages, 1, D, P)
    for b, x in enumerate(rows):
        codes, scale, mid = plain.codes_of(x)
        for pg in range(-(-x.shape[1] // P)):
            m = min(P, x.shape[1] - pg * P)
            full = [torch.zeros(2, 1, P, D, dtype=torch.int64), torch.full((2, 1, P), math.nan, dtype=torch.float64), torch.zeros(2, 1, P, dtype=torch.float64)]
            for f, y in zip(full, (codes, scale, mid)):
                f[:, 0, :m] = y[:, pg * P:pg * P + m]
            pool[int(table[b, pg])] = plain.pack(*full, P, D)
    return pool.to(DEV)


def check_or_zero(out, ref, dtype, H, D):
    """Rows of zeros give zeros (a bound relative to what they hold would be zero over zero)."""
    if not ref[0].any():
        assert not out.any()
    else:
        check(out, ref, dtype, H, D)


def received(ref, n_pages, P):
    want = torch.zeros(n_pages, 1, P, dtype=torch.float64)
    for at, w in ref[3].items():
        want[at] += w
    return want


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("where", ["first", "last", "mixed"])
@pytest.mark.parametrize("large,small", [(2.0 ** 74, 0.0), (2.0 ** 120, 0.0), (2.0 ** 120, 2.0 ** -60), (1.0, 0.0)])
def test_rows_of_zeros_beside_large_rows(dtype, where, large, small):
    """Scores alike, half of the values large, the others next to nothing: these add nothing to the output but count in the denominator, inside a
    warp's range, among the ranges of a block (65 keys, 700) and among blocks (5,000)."""
    H, D, P = 3, 128, 64
    lens = [5000, 700, 65]
    table, n_pages = tables(lens, P, 3)
    rows = []
    for b, n in enumerate(lens):
        k, v = 0.02 * rnd(n, D, seed=4 + b), rnd(n, D, seed=14 + b)
        at = torch.arange(n)
        tiny = at < n // 2 if where == "first" else at >= n - n // 2 if where == "last" else rnd(n, seed=24 + b) > 0
        v *= torch.where(tiny, small, large).unsqueeze(1)
        rows.append(torch.stack([k, v]))
    pool = pool_of(table, n_pages, rows, P)
    q = rnd(len(lens), H * D, dtype=dtype, seed=5)
    weights = torch.zeros(n_pages, 1, P, device=DEV)
    out, ctx = run_decode(q, pool, table, lens, H, 1, D, P, weights=weights)
    alone, _ = run_decode(q, pool, table, lens, H, 1, D, P)
    assert torch.equal(out, alone) and torch.isfinite(out).all()
    ref = plain.decode(q, pool, table, ctx, H, 1, D, P, D ** -0.5)
    check(out, ref, dtype, H, D)
    want = received(ref, n_pages, P)
    # (scores below one, a few roundings of 2^-24; the exponentials, 2^-22 each; the denominator's sum over the keys)
    assert ((weights.cpu().double() - want).abs() <= 2.0 ** -18 * want).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [0.0, 2.0 ** 100])
def test_a_sink_far_above_the_scores(dtype, value):
    """Sinks from far below to far above the keys' scores, over rows of zeros and over large ones: the weights are the keys' share."""
    H, D, P = 5, 128, 64
    lens = [200]
    table, n_pages = tables(lens, P, 33)
    pool = pool_of(table, n_pages, [torch.stack([0.02 * rnd(200, D, seed=34), value * rnd(200, D, seed=35)])], P)
    q = rnd(1, H * D, dtype=dtype, seed=36)
    for sinks in ([-60.0, 0.0, 5.0, 9.0, 3.0], [50.0, 55.0, 52.0, 51.0, 60.0]):
        sink = torch.tensor(sinks)
        weights = torch.zeros(n_pages, 1, P, device=DEV)
        out, ctx = run_decode(q, pool, table, lens, H, 1, D, P, weights=weights, sink=sink)
        ref = plain.decode(q, pool, table, ctx, H, 1, D, P, D ** -0.5, sink=sink)
        check_or_zero(out, ref, dtype, H, D)
        want = received(ref, n_pages, P)
        # as above, and the sink's exponent: 60 / ln 2 = 87 in base 2, a product rounded once (2^-18) and taken off (2^-18)
        assert ((weights.cpu().double() - want).abs() <= 2.0 ** -16 * want).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,lens", [(1, [300, 64]), (7, [130])])
def test_weights_do_not_depend_on_the_sizes_of_values(dtype, H, lens):
    """A key's weight is formed of its score, whatever its value holds: rows of zeros, of 2^-60, 2^60 and 2^100 leave it as exact as rows of ordinary size.
    Scores of up to two: rounded a few times by 2^-24 of two, less the largest one (2^-24 of four), the exponential 2^-22; taken together 2^-20.5 of a
    weight, in the norm over the keys 2^-21.  (A score rounded beside an exponent of 64 or more would be off by up to 2^-18 each time.)"""
    D, P = 128, 64
    table, n_pages = tables(lens, P, 43)
    keys = [0.5 * rnd(n, D, seed=44 + b) for b, n in enumerate(lens)]
    q = rnd(len(lens), H * D, dtype=dtype, seed=45)
    for size in (1.0, 0.0, 2.0 ** -60, 2.0 ** 60, 2.0 ** 100):
        rows = [torch.stack([k, size * rnd(k.shape[0], D, seed=46 + b)]) for b, k in enumerate(keys)]
        pool = pool_of(table, n_pages, rows, P)
        weights = torch.zeros(n_pages, 1, P, device=DEV)
        out, ctx = run_decode(q, pool, table, lens, H, 1, D, P, weights=weights)
        ref = plain.decode(q, pool, table, ctx, H, 1, D, P, D ** -0.5)
        check_or_zero(out, ref, dtype, H, D)
        want = received(ref, n_pages, P)
        off = (weights.cpu().double() - want).norm() / want.norm()
        assert float(off) <= 2.0 ** -21, f"values of {size:g}: off by {float(off):.3g}"


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_an_output_that_starts_between_two_elements_is_refused(dtype):
    H, D, P = 2, 64, 16
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    pool = pool_of(torch.tensor([[0]], dtype=torch.int32), 1, [rnd(2, 9, D, seed=51)], P)
    q = rnd(1, H * D, dtype=dtype, seed=52).to(DEV)
    kw = dict(seg_q0=i32([0]), seg_ctx=i32([8]), block_table=i32([[0]]), items=i32([0]), n_items=1, n_heads=H, n_kv_heads=1, head_dim=D, page_tokens=P, window=0,
              scale=1.0, part_o=torch.zeros(64 * D, device=DEV), part_ml=torch.zeros(128, device=DEV), counters=torch.zeros(H, dtype=torch.int32, device=DEV))
    room = torch.full((H * D + 4,), 7.0, dtype=dtype, device=DEV)
    with pytest.raises(K.KernelError, match="out must start"):
        K.attn_decode_q4(q, pool, room[1:1 + H * D].view(1, -1), **kw)
    assert (room == 7).all()
    K.attn_decode_q4(q, pool, room[2:2 + H * D].view(1, -1), **kw)   # (two elements further on is a place for two)
    want = torch.empty_like(q)
    K.attn_decode_q4(q, pool, want, **kw)
    assert torch.equal(room[2:2 + H * D], want[0]) and (room[:2] == 7).all() and (room[2 + H * D:] == 7).all()


@pytest.mark.parametrize("H", [1, 6])
def test_positions_behind_the_table_and_in_front_of_it(H):
    """A position behind what a request's row describes counts as the last that it describes, one below zero sees no key: neither reads pages of the next
    row or adds to another request's weights."""
    D, P = 64, 16
    lens = [48, 30, 48, 17]
    table, n_pages = tables(lens, P, 61)
    pool = pool_of(table, n_pages, [rnd(2, n, D, seed=62 + b) for b, n in enumerate(lens)], P)
    q = rnd(4, H * D, seed=67)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    units = K.decode_units_q4(4, H, DEV)

    def run(ctx):
        out, weights = torch.full((4, H * D), 9.0, device=DEV), torch.zeros(n_pages, 1, P, device=DEV)
        scores = torch.full((4 * H * 3 * P + 64,), 5.0, device=DEV)
        kw = dict(seg_q0=i32(range(4)), seg_ctx=i32(ctx), block_table=table.to(DEV), items=i32(range(4)), n_items=4, n_heads=H, n_kv_heads=1, head_dim=D,
                  page_tokens=P, window=0, scale=D ** -0.5, part_o=torch.empty(units * D + 64, device=DEV), part_ml=torch.empty(2 * units, device=DEV),
                  counters=torch.zeros(4 * H, dtype=torch.int32, device=DEV))
        K.attn_decode_q4(q.to(DEV), pool, out, weights=weights, scores=scores, **kw)
        assert (scores[-64:] == 5).all() and K.attn_q4_error() == 0
        alone = torch.empty_like(out)
        K.attn_decode_q4(q.to(DEV), pool, alone, **kw)
        assert torch.equal(out.view(torch.int32), alone.view(torch.int32))
        return out, weights

    want, weights = run([47, 29, 47, 16])
    for far in (48, 1000, 2 ** 31 - 1):
        got, now = run([far, 29, far, 16])
        assert torch.equal(got, want) and torch.equal(now, weights)
    got, now = run([47, -1, 47, -100])
    assert torch.equal(got[::2], want[::2]) and torch.isnan(got[1::2]).all()
    used = torch.zeros(n_pages, dtype=torch.bool)
    used[table[::2].reshape(-1).long()] = True
    assert torch.equal(now[used.to(DEV)], weights[used.to(DEV)]) and not now[~used.to(DEV)].any()


# ---------------------------------------------------------------------------
# what is rounded to fewer bits, no more than that


def rounded_once(ref, pool, table, ctx, H, kv, D, P, dtype):
    """The bound of tests/test_cache_q4_gpu.py with what a bfloat16 model's kernel rounds: every weight times its value's scale once to float16 (2^-11 of
    it, or 2^-35 of the largest where that is more: subnormal, 2^-25 beside 2^10), the output once.  ``plain_q4.decode`` allows for 2^-8 of a weight."""
    want, step, mass, _ = ref
    if dtype == F32:
        return SUMS * mass
    floor = torch.zeros_like(want)
    codes, scale, mid = plain.fields(pool, P, D)
    for b in range(want.shape[0]):
        t = torch.arange(int(ctx[b]) + 1)
        vs = scale[table[b, t // P].long(), 1, :, t % P]                       # [keys, kv]
        floor[b] = len(t) * 2.0 ** -35 * 8 * vs.max(0).values.repeat_interleave(H // kv).unsqueeze(1)
    return SUMS * mass + 2.0 ** -8 * want.abs() + 2.0 ** -3 * step + floor


def within(out, tol, ref, H, D):
    got = out.cpu().double().view(-1, H, D)
    worst = float(((got - ref[0]).abs() / tol).max())
    assert worst <= 1, f"off by {worst:.2f} times the bound"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,kv,D,P,lens", DECODE)
def test_attention_to_the_roundings_of_its_operands(dtype, H, kv, D, P, lens):
    table, n_pages = tables(lens, P, 3, extra_width=2)
    pool = filled(table, lens, kv, D, P, 71, n_pages).to(DEV)
    q = rnd(len(lens), H * D, dtype=dtype, seed=72, scale=1.5)
    out, ctx = run_decode(q, pool, table, lens, H, kv, D, P)
    ref = plain.decode(q, pool, table, ctx, H, kv, D, P, D ** -0.5)
    within(out, rounded_once(ref, pool, table, ctx, H, kv, D, P, dtype), ref, H, D)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_that_cancel(dtype):
    """Pairs of keys of nearly one weight and opposite values: what is left of the output is small beside the weights, so that their rounding shows.
    (Weights rounded to bfloat16 would be off by four times the bound.)"""
    H, D, P = 4, 128, 16
    lens = [2] * 8 + [4] * 8
    table, n_pages = tables(lens, P, 73)
    rows = []
    for b, n in enumerate(lens):
        v = rnd(n // 2, D, seed=74 + b)
        rows.append(torch.stack([0.1 * rnd(n, D, seed=94 + b), torch.stack([v, -v], 1).reshape(n, D)]))
    pool = pool_of(table, n_pages, rows, P)
    q = rnd(len(lens), H * D, dtype=dtype, seed=75)
    out, ctx = run_decode(q, pool, table, lens, H, 1, D, P)
    ref = plain.decode(q, pool, table, ctx, H, 1, D, P, D ** -0.5)
    within(out, rounded_once(ref, pool, table, ctx, H, 1, D, P, dtype), ref, H, D)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_queries_of_very_different_sizes_keep_their_small_elements(dtype):
    """Heads of 2^-100 and 2^-110, of zeros, and heads with one element 2^10 times the others: a bfloat16 query goes in as it is and a float32 one with 22 bits
    of each element, so every head keeps the bound of ordinary ones."""
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
    within(out, rounded_once(ref, pool, table, ctx, H, kv, D, P, dtype), ref, H, D)


def test_requests_that_are_preempted_behind_an_eviction(tmp_path):
    """A pool that holds one request's keys, a page and a short portion: requests longer than the pool, beside one another, finish and give everything back, and
    the same run again gives the same tokens."""
    from locus_b200.engine.engine import Engine
    from test_engine_q4_gpu import CASES
    from tiny_configs import make_model_dir, random_tokens

    raw = CASES["heads64"]
    folder = make_model_dir(tmp_path, "A", raw=dict(raw))
    prompts = [random_tokens(n, raw["vocab_size"], n) for n in (40, 150, 90)]
    seen = []
    for _ in range(2):
        eng = Engine.from_model_dir(folder, dtype="bfloat16", kv_bits=4, keep_tokens=48, ctx=96, page_tokens=16, max_running=3)
        assert eng.cfg.chunk == 32 and eng.cache.bound == 96 and eng.stats()["total_pages"] == 6
        out = eng.generate(prompts, 80)
        assert [len(x) for x in out] == [80] * 3
        stats = eng.stats()
        assert stats["evictions"] > 6 and stats["preemptions"] > 0 and stats["free_pages"] == 6
        eng.cache.check_invariants()
        seen.append(out)
    assert seen[0] == seen[1]
