"""The cache manager with pages of 4 bits, on the host: geometry, refusals, and what an eviction does to tables, counts and positions
(the kernel that moves rows replaced by one that records its call)."""
import pytest
import torch

import locus_b200.kernels as K
from locus_b200.cache import CacheError, CacheManager
from locus_b200.parts.base import PagedKvSpec

SPEC = PagedKvSpec(2, 64)


def mk(needs=None, **kw):
    args = dict(page_tokens=16, n_pages=12, n_state_slots=3, max_seq_tokens=160, device="cpu", kv_bits=4, weigh=True)
    args.update(kw)
    return CacheManager(needs or [(SPEC, None, None), (SPEC, None, None), (SPEC, None, 0)], **args)


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(K, "evict_q4", lambda pool, weights, **kw: seen.append((pool, weights, kw)))
    return seen


def test_pages_and_bytes():
    c = mk()
    g = c.groups[0]
    assert g.pool.dtype == torch.uint8 and tuple(g.pool.shape) == (2, 12, 2, 2, 16 * 36)
    assert tuple(g.weights.shape) == (2, 12, 2, 16) and not g.weights.any()
    assert c.bytes_per_token() == 2 * (2 * 2 * 36 + 4 * 2)
    assert mk(weigh=False).bytes_per_token() == 2 * 2 * 2 * 36 and mk(weigh=False).groups[0].weights is None
    views = c.layer_caches()
    assert views[0].weights.shape == (12, 2, 16) and views[2].weights.data_ptr() == views[0].weights.data_ptr() and not views[2].writes
    assert mk(kv_bits=0, weigh=False).groups[0].pool.dtype == torch.float32


def test_what_portions_take_beside_the_pools():
    """A layer's rows in the model's type for every group: the staging buffer has the shape of a layer's pool."""
    other = PagedKvSpec(1, 128)
    needs = [(SPEC, None, None), (SPEC, None, None), (other, None, None)]
    assert mk(needs).staging_bytes_per_token() == (2 * 2 * 64 + 2 * 128) * 4
    assert mk(needs, dtype=torch.bfloat16).staging_bytes_per_token() == (2 * 2 * 64 + 2 * 128) * 2
    assert mk(needs, kv_bits=0, weigh=False).staging_bytes_per_token() == 0


@pytest.mark.parametrize("needs,over,says", [
    (None, dict(kv_bits=8), "kv_bits 8"),
    (None, dict(kv_bits=0), "beside a cache of 4 bits"),
    (None, dict(weigh=False, bound=64), "a bound needs them"),
    (None, dict(page_tokens=24), "pages of 24"),
    ([(PagedKvSpec(2, 48), None, None)], {}, "heads of 64, 128, 256"),
    ([(PagedKvSpec(1, 64, has_v=False), None, None)], {}, "keys and values"),
    ([(PagedKvSpec(1, 64, extra_width=8), None, None)], {}, "keys and values"),
    ([(PagedKvSpec(2, 64, window=32), None, None)], {}, "without a window"),
    ([(PagedKvSpec(2, 64, chunk=32), None, None)], {}, "without chunks"),
])
def test_refused(needs, over, says):
    with pytest.raises(ValueError, match=says):
        mk(needs, **over)


def test_windows_go_with_4_bits_alone():
    assert mk([(PagedKvSpec(2, 64, window=32), None, None)], weigh=False).groups[0].pool.dtype == torch.uint8


def test_an_eviction_gives_pages_back_and_positions_go_on(calls):
    c = mk()
    a, b, short = c.open("a"), c.open("b"), c.open("c")
    for s, n in ((a, 70), (b, 50), (short, 20)):
        assert c.ensure_capacity(s, n)
        c.commit(s, n)
    table = c.table_row(a, 0)
    free = c.free_pages()
    assert c.evict([a, short, b], 33, first=2, recent=10) == 2
    (pool, weights, kw), = calls
    assert pool is c.groups[0].pool and weights is c.groups[0].weights
    assert kw["n_tokens"].tolist() == [70, 50] and kw["n_items"] == 2 and kw["keep"] == 33 and kw["first"] == 2 and kw["recent"] == 10
    assert kw["max_tokens"] == 70 and kw.get("dst_table") is None and tuple(kw["kept"].shape) == (2, 2, 2, 33)
    assert kw["block_table"][0].tolist() == table and kw["block_table"][1].tolist()[4:] == [-1]
    assert a.n_tokens == 33 and a.position == 70 and b.n_tokens == 33 and b.position == 50 and short.n_tokens == 20 and short.position == 20
    assert c.table_row(a, 0) == table[:3] and c.free_pages() == free + 2 + 1
    c.check_invariants()
    assert c.ensure_capacity(a, 20)
    c.commit(a, 20)
    assert a.n_tokens == 53 and a.position == 90
    assert c.evict([a, b], 60) == 0 and len(calls) == 1
    c.release(a)
    assert c.open("d").position == 0
    c.check_invariants()


def test_evictions_that_are_refused(calls):
    c = mk()
    a = c.open("a")
    c.adopt(a, 40)
    for args in ((0, 0, 0), (10, -1, 0), (10, 6, 5)):
        with pytest.raises(ValueError, match="keep"):
            c.evict([a], *args)
    with pytest.raises(CacheError, match="twice"):
        c.evict([a, a], 10)
    with pytest.raises(CacheError, match="weigh"):
        mk(weigh=False).evict([], 10)
    c.release(a)
    with pytest.raises(CacheError, match="not open"):
        c.evict([a], 10)
    assert not calls


def test_a_bound_narrows_tables_and_needs(calls):
    c = mk(max_seq_tokens=4000, bound=80)
    assert c.table_width == 5 and c.pages_needed(0, 4000) == 5 and c.pages_needed(0, 30) == 2
    a = c.open("a")
    c.adopt(a, 75)
    with pytest.raises(CacheError, match="limit of 80"):
        c.ensure_capacity(a, 6)
    c.evict([a], 40)
    for _ in range(20):
        assert c.ensure_capacity(a, 30)
        c.commit(a, 30)
        c.evict([a], 40)
    assert a.position == 75 + 600 and a.n_tokens == 40
    c.check_invariants()
