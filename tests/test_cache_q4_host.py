"""The cache held in 4 bits on the host: the plain format against itself, and what its entry points refuse."""
import pytest
import torch

import locus_b200.kernels as K
import plain_q4 as plain

I32 = torch.int32
NH, KV, D, P = 4, 2, 64, 16


def test_the_plain_format_reads_back_what_it_packs():
    x = torch.randn(3, 2, KV, P, D, generator=torch.Generator().manual_seed(1))
    codes, scale, mid = plain.codes_of(x)
    data = plain.pack(codes, scale, mid, P, D)
    assert tuple(data.shape) == (3, 2, KV, K.q4_page_bytes(D, P))
    c, s, m = plain.fields(data, P, D)
    assert torch.equal(c, codes) and torch.equal(s, scale) and torch.equal(m, mid)
    off = (plain.values(data, P, D) - x.double()).abs()
    # half a cell, and the rounding of scale (7.5 cells of it) and of mid
    assert (off <= (s * (0.5 + 7.5 * 2.0 ** -8) + m.abs() * 2.0 ** -8).unsqueeze(-1)).all()


def test_the_plain_selection():
    nan = float("nan")
    assert plain.stay([3.0, 1.0, 3.0, 2.0, 3.0], 3, 0, 1) == [0, 2, 4]
    assert plain.stay([3.0, 1.0, 3.0, 2.0, 3.0], 2, 0, 1) == [0, 4]
    assert plain.stay([nan, float("-inf"), nan, 0.0, 0.0], 4, 0, 1) == [0, 1, 3, 4]
    assert plain.stay([5.0, 5.0], 3, 1, 1) == [0, 1]


def base(lead=()):
    return torch.zeros(lead + (3, 2, KV, K.q4_page_bytes(D, P)), dtype=torch.uint8)


def write_args(**over):
    a = dict(qkv=torch.zeros(5, (NH + 2 * KV) * D), positions=torch.zeros(5, dtype=I32), inv_freq=torch.ones(D // 2), q_out=torch.zeros(5, NH * D),
             pool=base(), slots=torch.zeros(5, dtype=I32), n_heads=NH, n_kv_heads=KV, head_dim=D, rot_dim=D, interleaved=False, page_tokens=P)
    a.update(over)
    return a


def expand_args(**over):
    a = dict(pool=base(), out=torch.zeros(3, 2, KV, P, D), segs=torch.zeros(2, dtype=I32), n_segs=2, seg_ctx=torch.zeros(2, dtype=I32),
             seg_qn=torch.ones(2, dtype=I32), block_table=torch.zeros(2, 2, dtype=I32), n_kv_heads=KV, head_dim=D, page_tokens=P, max_keys=20)
    a.update(over)
    return a


def evict_args(**over):
    a = dict(pool=base((2,)), weights=torch.zeros(2, 3, KV, P), block_table=torch.zeros(2, 2, dtype=I32), n_tokens=torch.zeros(2, dtype=I32), n_items=2,
             keep=8, first=2, recent=3, kept=torch.zeros(2, 2, KV, 8, dtype=I32), n_kv_heads=KV, head_dim=D, page_tokens=P, max_tokens=30)
    a.update(over)
    return a


def decode_args(**over):
    a = dict(q=torch.zeros(2, NH * D), pool=base(), out=torch.zeros(2, NH * D), seg_q0=torch.zeros(2, dtype=I32), seg_ctx=torch.zeros(2, dtype=I32),
             block_table=torch.zeros(2, 2, dtype=I32), items=torch.zeros(2, dtype=I32), n_items=2, n_heads=NH, n_kv_heads=KV, head_dim=D, page_tokens=P,
             window=0, scale=0.1, part_o=torch.zeros(4000 * D), part_ml=torch.zeros(8000), counters=torch.zeros(8, dtype=I32))
    a.update(over)
    return a


W = dict(weights=torch.zeros(3, KV, P), scores=torch.zeros(2 * NH * 2 * P))
REFUSED = [
    (K.rope_kv_write_q4, write_args, dict(head_dim=96), "heads of 96"),
    (K.rope_kv_write_q4, write_args, dict(page_tokens=24), "pages of 24"),
    (K.rope_kv_write_q4, write_args, dict(pool=base().float()), "uint8"),
    (K.rope_kv_write_q4, write_args, dict(pool=base()[..., :-4]), "pool must be"),
    (K.rope_kv_write_q4, write_args, dict(qkv=torch.zeros(5, 7)), "qkv width"),
    (K.rope_kv_write_q4, write_args, dict(q_out=torch.zeros(5, NH * D, dtype=torch.bfloat16)), "one element type"),
    (K.rope_kv_write_q4, write_args, dict(q_out=torch.zeros(4, NH * D)), "too small"),
    (K.rope_kv_write_q4, write_args, dict(slots=torch.zeros(4, dtype=I32)), "slots"),
    (K.rope_kv_write_q4, write_args, dict(positions=torch.zeros(5, dtype=torch.int64)), "positions"),
    (K.rope_kv_write_q4, write_args, dict(rot_dim=D + 2), "rot_dim"),
    (K.rope_kv_write_q4, write_args, dict(rot_dim=7), "rot_dim"),
    (K.rope_kv_write_q4, write_args, dict(inv_freq=torch.ones(3)), "inv_freq"),
    (K.rope_kv_write_q4, write_args, dict(weights=torch.zeros(3, P, KV)), "weights"),
    (K.rope_kv_write_q4, write_args, {}, "CUDA tensor"),
    (K.expand_q4, expand_args, dict(out=torch.zeros(3, 2, KV, P, D + 1)), "out must have"),
    (K.expand_q4, expand_args, dict(segs=torch.zeros(1, dtype=I32)), "segs"),
    (K.expand_q4, expand_args, dict(block_table=torch.zeros(4, dtype=I32)), "block_table"),
    (K.expand_q4, expand_args, {}, "CUDA tensor"),
    (K.evict_q4, evict_args, dict(keep=0), "keep 0"),
    (K.evict_q4, evict_args, dict(first=6), "keep 8"),
    (K.evict_q4, evict_args, dict(recent=-1), "last -1"),
    (K.evict_q4, evict_args, dict(pool=base()), "layers"),
    (K.evict_q4, evict_args, dict(weights=torch.zeros(3, KV, P)), "weights"),
    (K.evict_q4, evict_args, dict(kept=torch.zeros(2, 2, KV, 7, dtype=I32)), "kept"),
    (K.evict_q4, evict_args, dict(max_tokens=33), "max_tokens"),
    (K.evict_q4, evict_args, dict(max_tokens=0), "max_tokens"),
    (K.evict_q4, evict_args, dict(dst_table=torch.zeros(1, 2, dtype=I32)), "dst_table"),
    (K.evict_q4, evict_args, dict(dst_table=torch.zeros(2, 0, dtype=I32)), "dst_table"),
    (K.evict_q4, evict_args, {}, "CUDA tensor"),
    (K.attn_decode_q4, decode_args, dict(head_dim=80), "heads of 80"),
    (K.attn_decode_q4, decode_args, dict(n_heads=5), "multiple"),
    (K.attn_decode_q4, decode_args, dict(out=torch.zeros(2, NH * D, dtype=torch.bfloat16)), "one element type"),
    (K.attn_decode_q4, decode_args, dict(q=torch.zeros(2, NH * D, dtype=torch.float16), out=torch.zeros(2, NH * D, dtype=torch.float16)), "element type|CUDA tensor"),
    (K.attn_decode_q4, decode_args, dict(counters=torch.zeros(7, dtype=I32)), "counters"),
    (K.attn_decode_q4, decode_args, dict(part_o=torch.zeros(7 * D)), "scratch too small"),
    (K.attn_decode_q4, decode_args, dict(part_ml=torch.zeros(15)), "scratch too small"),
    (K.attn_decode_q4, decode_args, dict(part_o=torch.zeros(15 * D), window=4, keep_first=2), "scratch too small"),
    (K.attn_decode_q4, decode_args, dict(n_items=2000), "at most"),
    (K.attn_decode_q4, decode_args, dict(W, window=4), "neither a window nor chunks"),
    (K.attn_decode_q4, decode_args, dict(W, chunk=4), "neither a window nor chunks"),
    (K.attn_decode_q4, decode_args, dict(W, scores=None), "scores"),
    (K.attn_decode_q4, decode_args, dict(W, scores=torch.zeros(2 * NH * 2 * P - 1)), "scores"),
    (K.attn_decode_q4, decode_args, dict(W, weights=torch.zeros(3, KV, P, dtype=torch.bfloat16)), "weights"),
    (K.attn_decode_q4, decode_args, {}, "CUDA tensor"),
    (K.attn_decode_q4, decode_args, dict(out=torch.zeros(1, NH * D)), "rows of whole heads"),
    (K.attn_decode_q4, decode_args, dict(n_kv_heads=0, pool=torch.zeros(3, 2, 0, P * (D // 2 + 4), dtype=torch.uint8)), "multiple"),
]


@pytest.mark.parametrize("call,args,over,says", REFUSED, ids=[f"{i}-{r[0].__name__}-{r[3].split('|')[0].replace(' ', '_')}" for i, r in enumerate(REFUSED)])
def test_refused_on_the_host(call, args, over, says):
    a = args(**over)
    names = {K.rope_kv_write_q4: ("qkv", "positions", "inv_freq", "q_out", "pool", "slots"), K.expand_q4: ("pool", "out"), K.evict_q4: ("pool", "weights"),
             K.attn_decode_q4: ("q", "pool", "out")}[call]
    with pytest.raises(K.KernelError, match=says):
        call(*[a.pop(n) for n in names], **a)
