"""Models on a cache held in 4 bits, through the engine on the GPU: logits against the plain implementation with its keys and values put
through the same format, portions and single tokens alike; and requests that let go of keys."""
import pytest
import torch

import locus_b200.kernels as K
import plain_q4
import plain_qwen2moe as plain
from tiny_configs import config, make_model_dir, random_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# A key or value that lies next to a border of its cell may fall to the other side, which moves it by a cell (a fifteenth of its row's range, a third of the
# values' spread at these sizes).  float32: a millionth of a cell off, none or a handful of the rows' elements.  bfloat16: the projected values are
# 2^-9 off in the mean, 15 / 4 of that in cells, so up to 3 % of the elements move, and the rows by a twentieth of their spread.
TOL = {torch.float32: 0.01, torch.bfloat16: 0.1}


def dense(name, **over):
    raw = config(name)
    raw.update(mlp_only_layers=list(range(raw["num_hidden_layers"])), use_sliding_window=raw.get("use_sliding_window", False), **over)
    return raw


CASES = {
    "grouped128": dense("D"),
    "heads64": dense("A", head_dim=64, num_key_value_heads=2),
    "window64": dense("C", head_dim=64),
    "experts64": dict(config("B"), head_dim=64),
}


@pytest.fixture(scope="module", params=list(CASES))
def model_case(request, tmp_path_factory):
    raw = CASES[request.param]
    d = make_model_dir(tmp_path_factory.mktemp("q4"), "A", raw=dict(raw))
    return request.param, raw, d


def reference(raw, folder, tokens, monkeypatch):
    """float64 logits of every position, keys and values through the 4-bit format."""
    _, weights = plain.load_folder(folder)
    attention = plain.attention

    def held(x):
        codes, scale, mid = plain_q4.codes_of(x)
        return mid.unsqueeze(-1) + scale.unsqueeze(-1) * (codes.double() - 7.5)

    monkeypatch.setattr(plain, "attention", lambda q, k, v, window=0: attention(q, held(k), held(v), window))
    return plain.forward(raw, weights, tokens, dtype=torch.float64)


def runner_of(folder, dtype, *, use_graphs=False, weigh=False, n_pages=64, max_seq=512):
    from locus_b200.cache import CacheManager
    from locus_b200.engine.step import ModelRunner
    from locus_b200.models import load_model

    model = load_model(folder, dtype, DEV)
    cache = CacheManager(model.cache_needs(), page_tokens=16, n_pages=n_pages, n_state_slots=4, max_seq_tokens=max_seq, dtype=dtype, device=DEV,
                         poison=True, kv_bits=4, weigh=weigh)
    return ModelRunner(model, cache, max_tokens=320, max_segments=4, use_graphs=use_graphs), cache


def feed(runner, cache, rid, tokens, portions):
    from locus_b200.engine.step import StepEntry

    seq = cache.get(rid) or cache.open(rid)
    at, out = 0, []
    for n in portions:
        assert cache.ensure_capacity(seq, n)
        out.append(runner.step([StepEntry(seq, tokens[at:at + n], list(range(n)))]).double().cpu())
        at += n
    assert at == len(tokens)
    return torch.cat(out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits(model_case, dtype, monkeypatch):
    name, raw, folder = model_case
    tokens = random_tokens(90, raw["vocab_size"], 3)
    ref = reference(raw, folder, tokens, monkeypatch)
    runner, cache = runner_of(folder, dtype)
    for rid, portions in (("whole", [90]), ("singly", [1] * 90), ("mixed", [1, 1, 30, 1, 2, 17, 1, 37])):
        got = feed(runner, cache, rid, tokens, portions)
        cache.release(cache.get(rid))
        # (routed experts may change sides with a moved element: the mean over positions then counts)
        off = ((got - ref).norm(dim=1) / ref.norm(dim=1))
        assert float(off.mean() if "experts" in name else off.max()) <= TOL[dtype] * (2 if "experts" in name else 1), f"{rid}: {float(off.max()):.3g}"
    runner.check_device_errors()


@pytest.mark.parametrize("weigh", [False, True])
def test_replayed_steps_and_several_requests(model_case, weigh):
    """Decode steps from graphs, of one and of three requests, give what eager steps give; the weights sum up to what was handed out."""
    name, raw, folder = model_case
    if weigh and "window" in name:
        pytest.skip("weights go with no window")
    from locus_b200.engine.step import StepEntry

    prompts = {"a": random_tokens(40, raw["vocab_size"], 5), "b": random_tokens(7, raw["vocab_size"], 6), "c": random_tokens(23, raw["vocab_size"], 7)}
    nexts = {r: random_tokens(6, raw["vocab_size"], 8 + i) for i, r in enumerate(prompts)}
    seen = []
    for graphs in (False, True):
        runner, cache = runner_of(folder, torch.bfloat16, use_graphs=graphs, weigh=weigh)
        out = []
        for r, p in prompts.items():
            feed(runner, cache, r, p, [len(p)])
        for i in range(6):
            entries = []
            for r in prompts:
                assert cache.ensure_capacity(cache.get(r), 1)
                entries.append(StepEntry(cache.get(r), [nexts[r][i]], [0]))
            out.append(runner.step(entries).float().cpu().clone())
        seen.append(torch.stack(out))
        if weigh:
            heads = raw["num_attention_heads"]
            for r, p in prompts.items():
                rows = cache.table_row(cache.get(r), 0)
                n = len(p) + 6
                for lc in cache.layer_caches():
                    w = torch.cat([lc.weights[pg] for pg in rows], -1)[:, :n]
                    # one query of the prompt and six single ones, each 1 per head
                    assert abs(float(w.sum()) - 7 * heads) <= 1e-3 * heads
    assert torch.equal(seen[0], seen[1])
    assert runner.stats["graph_replays"] > 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_keeping_the_weights_changes_no_output(tmp_path, dtype):
    """Bit for bit, single tokens beside portions too: a portion's last token has its weights added up by the kernel of single tokens, but its output
    comes from the portion's kernel either way."""
    from locus_b200.engine.step import StepEntry

    raw = CASES["heads64"]
    folder = make_model_dir(tmp_path, "A", raw=dict(raw))
    tokens = random_tokens(80, raw["vocab_size"], 12)
    seen = []
    for weigh in (False, True):
        runner, cache = runner_of(folder, dtype, weigh=weigh)
        out = [feed(runner, cache, "a", tokens[:40], [33, 1, 6])]
        a, b = cache.get("a"), cache.open("b")
        assert cache.ensure_capacity(a, 1) and cache.ensure_capacity(b, 21)
        out.append(runner.step([StepEntry(a, tokens[40:41], [0]), StepEntry(b, tokens[41:62], list(range(21)))]).double().cpu())
        seen.append(torch.cat(out))
    assert torch.equal(seen[0], seen[1])


def test_generation_with_and_without_letting_go(tmp_path):
    from locus_b200.engine.engine import Engine

    raw = CASES["heads64"]
    folder = make_model_dir(tmp_path, "A", raw=dict(raw))
    prompts = [random_tokens(60, raw["vocab_size"], 1), random_tokens(21, raw["vocab_size"], 2)]
    args = dict(dtype="bfloat16", page_tokens=16, ctx=512, max_running=4)
    plain_q = Engine.from_model_dir(folder, kv_bits=4, **args).generate(prompts, 40)
    # a bound that is never reached changes nothing
    eng = Engine.from_model_dir(folder, kv_bits=4, keep_tokens=200, **args)
    assert eng.generate(prompts, 40) == plain_q and eng.stats()["evictions"] == 0
    eng = Engine.from_model_dir(folder, kv_bits=4, keep_tokens=32, keep_first=2, keep_recent=8, **args)
    most = []
    eng.on_token = lambda r, t: most.append(max(s.n_tokens for s in eng.cache.live()) if eng.cache.live() else 0)
    got = eng.generate(prompts, 40)
    assert [len(g) for g in got] == [40, 40] and eng.stats()["evictions"] >= 4
    assert max(most[2:]) <= 32 + 16 and eng.cache.free_pages() == eng.cache.total_pages()
    eng.cache.check_invariants()
    again = Engine.from_model_dir(folder, kv_bits=4, keep_tokens=32, keep_first=2, keep_recent=8, **args).generate(prompts, 40)
    assert again == got   # the same choice every time
    # a request longer than the pool: its keys fit because they go
    small = Engine.from_model_dir(folder, kv_bits=4, keep_tokens=32, **dict(args, ctx=96, max_running=1, chunk=32, max_batch_tokens=32))
    out = small.generate([random_tokens(30, raw["vocab_size"], 4)], 120)
    assert len(out[0]) == 120 and small.stats()["total_pages"] == 6


def test_positions_go_on_behind_an_eviction(tmp_path):
    """A token fed behind an eviction is rotated by its position, not by its place: in the first layer, whose rows depend on the token and its position
    alone, its rows are those of the same token in a cache that kept everything."""
    raw = CASES["grouped128"]
    folder = make_model_dir(tmp_path, "D", raw=dict(raw))
    tokens = random_tokens(70, raw["vocab_size"], 9)
    runner, cache = runner_of(folder, torch.float32, weigh=True)
    feed(runner, cache, "all", tokens, [60] + [1] * 10)
    feed(runner, cache, "some", tokens[:60], [60])
    seq = cache.get("some")
    assert cache.evict([seq], 20, 2, 5) == 1
    feed(runner, cache, "some", tokens[60:], [1] * 10)
    assert seq.n_tokens == 30 and seq.position == 70
    D, P = raw["head_dim"], 16
    pool = cache.layer_caches()[0].pool

    def rows(rid, t):
        page = cache.table_row(cache.get(rid), 0)[t // P]
        return [f[..., t % P, :] if f.dim() == 4 else f[..., t % P] for f in plain_q4.fields(pool[page], P, D)]

    for i in range(10):
        for x, y in zip(rows("all", 60 + i), rows("some", 20 + i)):
            assert torch.equal(x, y)


def test_engines_that_are_refused(tmp_path):
    from locus_b200.engine.engine import Engine

    folder = make_model_dir(tmp_path, "A", raw=dict(CASES["heads64"]))
    window = make_model_dir(tmp_path / "w", "C", raw=dict(CASES["window64"]))
    small = make_model_dir(tmp_path / "s", "A")
    for d, args, says in ((folder, dict(keep_tokens=10), "kv_bits"), (folder, dict(kv_bits=4, keep_tokens=10, keep_first=8, keep_recent=8), "keep_tokens 10"),
                          (folder, dict(kv_bits=3), "kv_bits 3"), (folder, dict(kv_bits=4, max_running=1025), "at most 1024"), (window, dict(kv_bits=4, keep_tokens=64), "window"), (small, dict(kv_bits=4), "heads of 64")):
        with pytest.raises(ValueError, match=says):
            Engine.from_model_dir(d, page_tokens=16, ctx=256, **args)


@pytest.mark.parametrize("keep", [0, 64])
def test_a_share_of_the_memory_covers_the_staging_buffer(tmp_path, keep):
    """kv_fraction bounds the pools and the buffer that a prompt's portion is laid out in, and leaves an evicted request's positions alone."""
    from locus_b200.engine.engine import Engine

    raw = CASES["heads64"]
    folder = make_model_dir(tmp_path, "A", raw=dict(raw))
    free, share = torch.cuda.mem_get_info(DEV)[0], 2e-4
    eng = Engine.from_model_dir(folder, page_tokens=16, kv_bits=4, keep_tokens=keep, kv_fraction=share)
    c = eng.cache
    assert 0 < c.n_pages * 16 * (c.bytes_per_token() + c.staging_bytes_per_token()) <= free * share
    assert c.max_seq_tokens == (raw["max_position_embeddings"] if keep else min(raw["max_position_embeddings"], c.n_pages * 16))
    assert len(eng.generate([random_tokens(30, raw["vocab_size"], 3)], 4)[0]) == 4
    staged = [t for k, t in eng.runner.rt._bufs.items() if k[0] == "attention.q4_wide"]
    assert len(staged) == 1 and staged[0].numel() * staged[0].element_size() == c.n_pages * 16 * c.staging_bytes_per_token()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_shaped_form(dtype, monkeypatch, tmp_path):
    """Attention whose projections go through the kernel of shaped heads (here without any of its options) reads and writes the same rows."""
    from locus_b200.cache import CacheManager
    from locus_b200.config.base import load_config
    from locus_b200.engine.step import ModelRunner
    from locus_b200.models.model import Model
    from locus_b200.parts.base import PartSpec
    from locus_b200.weights.loader import load_weights
    from locus_b200.weights.safetensors_io import ModelFiles

    raw = CASES["heads64"]
    folder = make_model_dir(tmp_path, "A", raw=dict(raw))
    tokens = random_tokens(50, raw["vocab_size"], 13)
    ref = reference(raw, folder, tokens, monkeypatch)
    entry, cfg = load_config(folder)
    files = ModelFiles(folder)
    plan = entry.plan(cfg, files)
    for i, layer in enumerate(plan.layers):
        object.__setattr__(layer, "mixer", PartSpec(layer.mixer.kind, {**layer.mixer.args, "shaped": True}))
    model = Model(plan, dtype, DEV)
    load_weights(model, files)
    files.close()
    assert model.blocks[0].mixer.shaped
    cache = CacheManager(model.cache_needs(), page_tokens=16, n_pages=32, n_state_slots=4, max_seq_tokens=256, dtype=dtype, device=DEV, poison=True, kv_bits=4, weigh=True)
    runner = ModelRunner(model, cache, max_tokens=320, max_segments=4)
    for rid, portions in (("whole", [50]), ("mixed", [1, 1, 20, 1, 2, 25])):
        got = feed(runner, cache, rid, tokens, portions)
        assert float(((got - ref).norm(dim=1) / ref.norm(dim=1)).max()) <= TOL[dtype]
