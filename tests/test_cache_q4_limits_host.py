"""The cache held in 4 bits on the host: what the native entry points refuse before they touch a device, and the sizes that an engine gives such a
cache."""
import pytest

import locus_b200.kernels as K

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
