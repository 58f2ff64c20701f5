"""The cache held in 4 bits on the host: what the native entry points refuse before they touch a device, and the sizes that an engine gives such a
cache."""
from types import SimpleNamespace

import pytest
import torch

import locus_b200.engine.engine as engine_module
import locus_b200.kernels as K
from locus_b200.cache import CacheManager
from locus_b200.parts.base import Mixer, PagedKvSpec

BF16, F32 = 1, 0
AT = 1 << 20   # an address that nothing on the host or the device reads: every call here ends before its launch


def decode_call(**over):
    """Packed arguments of the attention's entry point: one request of 16 keys, one head of 64."""
    a = dict(q=AT, pool=AT, out=AT, seg_q0=AT, seg_ctx=AT, block_table=AT, items=AT, part_o=AT, part_ml=AT, counters=AT, sink=0, slopes=0, weights=0, scores=0, lse=0,
             dt=BF16, table_stride=1, n_items=1, nh=1, nkv=1, hd=64, page_tokens=16, window=0, chunk=0, max_units=64, cost_range=64, cost_join=96, cost_merge=4,
             keep_first=0, sink_flag=0, scale=0.125)
    a.update(over)
    return K._q4_entry("attention_q4", "locus_attn_decode_q4")(K._Q4_DECODE.pack(*a.values()), None)


@pytest.mark.parametrize("over", [
    dict(dt=BF16, out=AT + 2), dict(dt=F32, out=AT + 4), dict(dt=F32, out=AT + 12), dict(q=AT + 8), dict(pool=AT + 4), dict(part_o=AT + 8), dict(part_ml=AT + 4),
    dict(weights=AT + 4, scores=AT, lse=AT), dict(weights=AT, scores=AT + 8, lse=AT), dict(weights=AT, scores=AT, lse=AT + 4),
], ids=lambda o: "-".join(f"{k}{v - AT if v >= AT else v}" for k, v in o.items()))
def test_addresses_that_a_store_cannot_take_are_refused_before_a_launch(over):
    assert decode_call(**over) == K.ERR_UNSUPPORTED


@pytest.mark.parametrize("over", [dict(table_stride=0), dict(table_stride=1 << 27), dict(table_stride=1 << 40), dict(page_tokens=8), dict(n_items=1025)],
                         ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()))
def test_tables_that_describe_no_position_or_too_many_are_refused(over):
    assert decode_call(**over) == K.ERR_UNSUPPORTED


# ---------------------------------------------------------------------------
# an engine whose requests let go of keys: the pool, the portions and the scheduler, with a model of one layer that computes nothing


class StandInRunner:
    """Logits of token 1 for every wanted place; checks that every entry has room and counts what requests hold."""

    def __init__(self, model, cache, **kw):
        self.cache, self.most, self.longest = cache, 0, 0

    def step(self, entries):
        rows = 0
        for e in entries:
            assert e.seq.n_tokens + len(e.tokens) <= self.cache.capacity(e.seq)
            self.cache.commit(e.seq, len(e.tokens))
            self.most, self.longest = max(self.most, e.seq.n_tokens), max(self.longest, len(e.tokens))
            rows += len(e.want)
        return torch.zeros(rows, 4)


class StandInSampler:
    def __init__(self, device, n):
        pass

    def sample(self, logits, params, seeds, counters, histories=None):
        return [1] * len(logits)


class StandInMixer(Mixer):
    reads_q4 = weighs = True

    def cache_needs(self):
        return PagedKvSpec(1, 64), None


def stand_in_model(max_positions, *mixers):
    mixers = mixers or (StandInMixer(""),)
    plan = SimpleNamespace(max_positions=max_positions, order=[SimpleNamespace(layer=i) for i in range(len(mixers))], eos_token_id=-1)
    return SimpleNamespace(plan=plan, blocks=[SimpleNamespace(mixer=m) for m in mixers], dtype=torch.bfloat16, device=torch.device("cpu"),
                           cache_needs=lambda: [m.cache_needs() + (None,) for m in mixers])


@pytest.fixture
def engine_of(monkeypatch):
    monkeypatch.setattr(engine_module, "ModelRunner", StandInRunner)
    monkeypatch.setattr(engine_module, "Sampler", StandInSampler)
    monkeypatch.setattr(K, "evict_q4", lambda *a, **kw: None)

    def make(max_positions=32768, **kw):
        return engine_module.Engine.from_model(stand_in_model(max_positions), kv_bits=4, **kw)

    return make


def finish(eng, *requests):
    ids = [eng.submit([2] * n, new) for n, new in requests]
    eng.run_to_completion()
    got = [eng.get(i) for i in ids]
    assert [(r.status.value, r.error) for r in got] == [("done", "")] * len(ids)
    assert [len(r.generated) for r in got] == [new for _, new in requests]
    assert eng.cache.free_pages() == eng.cache.total_pages()
    eng.cache.check_invariants()


def test_a_pool_of_no_given_size_holds_what_a_request_holds_before_it_lets_go(engine_of):
    eng = engine_of(keep_tokens=4096, keep_first=4, keep_recent=1024)
    assert eng.cache.total_pages() * 64 >= 4096 + 64 + 2048 == eng.cache.bound
    finish(eng, (100, 4300), (7000, 30))
    assert eng.stats()["evictions"] >= 4 and eng.runner.longest <= 2048 and eng.runner.most <= eng.cache.bound
    # as before where nothing is let go of, and where a request cannot become as long
    assert engine_of().cache.total_pages() == 64 and engine_of(keep_tokens=100, chunk=512).cache.total_pages() == 64
    small = engine_of(max_positions=1000, keep_tokens=4096)
    assert small.cache.total_pages() == 16
    finish(small, (500, 400))


@pytest.mark.parametrize("ctx", [1024 + 128, 1500, 2000, 3000, 3136, 4096])
def test_portions_of_a_pool_of_a_given_size_leave_room_for_what_stays(engine_of, ctx):
    """Requests longer than the pool finish in it, alone and beside one another, preempted behind an eviction as well."""
    eng = engine_of(keep_tokens=1024, ctx=ctx, max_running=4)
    pool = eng.cache.total_pages() * 64
    assert eng.cache.bound <= pool and eng.cfg.chunk == (2048 if ctx >= 3136 else pool - 1024 - 64)
    finish(eng, (100, 2 * pool))
    assert eng.stats()["evictions"] > 0 and eng.runner.most <= eng.cache.bound and eng.runner.longest <= eng.cfg.chunk
    finish(eng, (3000, 300), (50, 1900), (700, 1500))
    assert eng.stats()["preemptions"] > 0 or ctx >= 3000


@pytest.mark.parametrize("ctx,chunk,least", [(1024, 2048, 1152), (1151 - 64, 2048, 1152), (1088, 16, 1104), (512, 64, 1152)])
def test_a_pool_too_small_to_let_go_of_keys_is_refused(engine_of, ctx, chunk, least):
    with pytest.raises(ValueError, match=f"at least {least}"):
        engine_of(keep_tokens=1024, ctx=ctx, chunk=chunk)
    finish(engine_of(keep_tokens=1024, ctx=least, chunk=chunk), (1500, 30))


def test_a_negative_count_of_tokens_is_refused(engine_of):
    with pytest.raises(ValueError, match="keep_tokens -1"):
        engine_of(keep_tokens=-1)


# ---------------------------------------------------------------------------
# what a cache of 4 bits takes beside its pools


@pytest.mark.parametrize("weigh", [False, True])
def test_the_scratch_of_a_cache_of_4_bits_is_known_beforehand(weigh, tmp_path, monkeypatch):
    """What the mixers say they take is what a runner holds once it is built, before its first step: nothing is left to be found out with the pool in place."""
    from locus_b200.engine.step import ModelRunner
    from locus_b200.models import load_model
    from tiny_configs import config, make_model_dir
    import emulated_kernels

    emulated_kernels.install(monkeypatch)
    model = load_model(make_model_dir(tmp_path, "A", raw=dict(config("A"), head_dim=64, num_key_value_heads=2)), torch.float32, "cpu")
    cache = CacheManager(model.cache_needs(), page_tokens=16, n_pages=8, n_state_slots=3, max_seq_tokens=300, dtype=torch.float32, device="cpu", kv_bits=4, weigh=weigh)
    runner = ModelRunner(model, cache, max_tokens=32, max_segments=3)
    mixer = model.blocks[0].mixer
    said = mixer.q4_scratch(3, cache.table_width * 16, weigh, "cpu")
    held = {k[0]: t for k, t in runner.rt._bufs.items() if k[0].startswith("attention.q4")}
    assert {k: t.numel() for k, t in held.items() if k != "attention.q4_wide"} == said
    assert ("attention.q4_scores" in said) == weigh and (not weigh or said["attention.q4_scores"] == 3 * mixer.n_heads * 19 * 16)
    wide = held["attention.q4_wide"]
    assert wide.numel() * wide.element_size() == cache.n_pages * 16 * cache.staging_bytes_per_token()
    plain_cache = CacheManager(model.cache_needs(), page_tokens=16, n_pages=8, n_state_slots=3, max_seq_tokens=300, dtype=torch.float32, device="cpu")
    assert not any(k[0].startswith("attention.q4") for k in ModelRunner(model, plain_cache, max_tokens=32, max_segments=3).rt._bufs)


def test_a_share_of_the_memory_covers_the_scratch(engine_of, monkeypatch):
    """1,024 requests that keep 8,192 tokens: their scores alone are more than a gigabyte."""
    free = 8 << 30
    scratch = {"part": 10 << 20, "scores": 28 * 1024 * 10304}

    class Device:   # of a model that computes nothing: only its kind is looked at
        type, index = "cuda", 0

    class WithScratch(StandInMixer):
        def q4_scratch(self, max_segments, table_tokens, weigh, device):
            assert (max_segments, table_tokens, weigh) == (1024, 10304, True)
            return scratch

    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (free, free))
    monkeypatch.setattr(engine_module, "CacheManager", lambda *a, **kw: CacheManager(*a, **dict(kw, device="cpu", allocate_device=False)))
    model = stand_in_model(32768, WithScratch("0"), WithScratch("1"))
    model.device = Device()
    eng = engine_module.Engine.from_model(model, kv_bits=4, keep_tokens=8192, max_running=1024, kv_fraction=0.5)
    c = eng.cache
    per = c.bytes_per_token() + c.staging_bytes_per_token()
    taken = c.n_pages * 64 * per + 4 * sum(scratch.values())   # (the layers share it)
    assert free // 2 - 64 * per < taken <= free // 2
    with pytest.raises(ValueError, match="holds no page"):
        engine_module.Engine.from_model(model, kv_bits=4, keep_tokens=8192, max_running=1024, kv_fraction=0.05)


def test_what_stays_can_be_said_on_the_command_line():
    from locus_b200.cli import build_parser

    a = build_parser().parse_args(["--kv-bits", "4", "--keep-tokens", "4096", "--keep-first", "8", "--keep-recent", "1024", "model", "5,17"])
    assert (a.kv_bits, a.keep_tokens, a.keep_first, a.keep_recent) == (4, 4096, 8, 1024)
    a = build_parser().parse_args(["model", "5,17"])
    assert (a.keep_tokens, a.keep_first, a.keep_recent) == (0, 4, 0)
