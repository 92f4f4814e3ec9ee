"""What the trees' entry points refuse, on the CPU: every refusal comes before any launch, with a reason."""

import ctypes

import pytest

import w4a16
from test_kv_refusals import A, CONFIG, batch, cache


def plan(b=None, parents=A, stride=4, sizes=A * 2, nodes=4, seen=A * 3, positions=A * 4):
    return w4a16.lib.w4a16_kv_tree_plan(ctypes.byref(b or batch()), parents, stride, sizes, nodes, seen, positions, None)


def attend(c=None, b=None, q=A * 256, qs=(256, 64), heads=4, scale=0.125, window=0, out=A * 320, os=(256, 64), lse=None,
           ws=A * 1024, ws_bytes=1 << 28, **tree):
    f = dict(seen=A * 700, positions=A * 701, sizes=A * 702, nodes=4)
    f.update(tree)
    t = w4a16._KvTreeStruct(**f)
    return w4a16.lib.w4a16_paged_tree_attention_bf16(ctypes.byref(c or cache()), ctypes.byref(b or batch()), ctypes.byref(t), q, *qs, heads,
                                                     scale, window, out, *os, lse, ws, ws_bytes, None)


@pytest.mark.parametrize("call,args,why", [
    (plan, dict(b=batch(seqs=-1)), "extents"), (plan, dict(b=batch(rows=(1 << 25) + 1)), "extents"), (plan, dict(nodes=0), "nodes"),
    (plan, dict(nodes=257), "nodes"), (plan, dict(stride=-1), "stride"), (plan, dict(parents=None), "null"), (plan, dict(seen=None), "null"),
    (plan, dict(positions=None), "null"), (plan, dict(b=batch(kv_lens=None)), "null"), (plan, dict(b=batch(starts=None)), "null"),
    (plan, dict(seen=A * 3 + 4), "aligned"), (plan, dict(parents=A + 1), "aligned"), (plan, dict(sizes=A + 2), "aligned"),
    (plan, dict(positions=A * 3), "overlap"), (plan, dict(seen=A), "overlap"), (plan, dict(positions=A * 2), "overlap"),
    (plan, dict(seen=A * 513), "overlap"),
    (attend, dict(nodes=0), "nodes"), (attend, dict(nodes=257), "nodes"), (attend, dict(window=3), "window"), (attend, dict(window=-1), "window"),
    (attend, dict(seen=None), "null"), (attend, dict(positions=None), "null"), (attend, dict(seen=A * 700 + 4), "aligned"),
    (attend, dict(positions=A * 701 + 2), "aligned"), (attend, dict(sizes=A * 702 + 1), "aligned"), (attend, dict(seen=A * 320), "overlap"),
    (attend, dict(lse=A * 701), "overlap"), (attend, dict(sizes=A * 320 + 64), "overlap"), (attend, dict(c=cache(head_dim=32)), "head_dim"),
    (attend, dict(b=batch(max_kv=100000), ws=A * 700), "overlap"), (attend, dict(b=batch(max_kv=100000), ws=None), "workspace"),
    (attend, dict(out=A * 256 + 128), "overlap"), (attend, dict(os=(256, 32)), "each other"),
])
def test_calls(call, args, why):
    assert call(**args) == CONFIG
    assert why in w4a16.last_error()


def test_nothing_to_do():
    for b in (batch(rows=0), batch(seqs=0)):
        assert plan(b=b) == 0 and attend(b=b) == 0
    assert w4a16.lib.w4a16_kv_tree_plan(None, A, 4, None, 4, A * 2, A * 3, None) == CONFIG
    assert w4a16.lib.w4a16_paged_tree_attention_bf16(ctypes.byref(cache()), ctypes.byref(batch()), None, A, 256, 64, 4, 1.0, 0, A, 256, 64,
                                                     None, None, 0, None) == CONFIG
