"""What the verification of trees refuses, on the CPU: every refusal comes before any launch, with a reason."""

import ctypes

import pytest
import torch

import w4a16
from test_kv_refusals import A, CONFIG


def verify(target=A * 256, ts=(400000, 100000), tokens_in=A, parents=A * 2, sizes=A * 3, uniforms=A * 4, accepted=A * 5, path=A * 6, tokens=A * 7,
           seqs=2, nodes=4, vocab=100000, ws=A * 8, ws_bytes=1 << 20):
    return w4a16.lib.w4a16_verify_tree_f32(target, *ts, tokens_in, parents, sizes, uniforms, accepted, path, tokens, seqs, nodes, vocab, ws,
                                           ws_bytes, None)


@pytest.mark.parametrize("args,why", [
    (dict(seqs=-1), "extents"), (dict(seqs=65536), "extents"), (dict(nodes=0), "extents"), (dict(nodes=257), "extents"), (dict(vocab=0), "extents"),
    (dict(vocab=(1 << 28) + 1), "extents"), (dict(target=None), "null"), (dict(tokens_in=None), "null"), (dict(parents=None), "null"),
    (dict(uniforms=None), "null"), (dict(accepted=None), "null"), (dict(path=None), "null"), (dict(tokens=None), "null"), (dict(ws=None), "null"),
    (dict(target=A * 256 + 2), "aligned"), (dict(sizes=A * 3 + 1), "aligned"), (dict(ws=A * 8 + 4), "aligned"), (dict(ws_bytes=16), "workspace"),
    (dict(ts=(-1, 1)), "stride"), (dict(ts=(1, 1 << 44)), "stride"), (dict(accepted=A * 256), "overlap"), (dict(path=A), "overlap"),
    (dict(tokens=A * 2), "overlap"), (dict(path=A * 7), "overlap"), (dict(accepted=A * 3), "overlap"), (dict(ws=A * 4), "overlap"),
])
def test_calls(args, why):
    assert verify(**args) == CONFIG
    assert why in w4a16.last_error()


def test_nothing_to_do():
    need = ctypes.c_size_t(7)
    assert verify(seqs=0) == 0
    assert w4a16.lib.w4a16_verify_tree_workspace(2, 4, 1000, ctypes.byref(need)) == 0 and need.value == 0
    assert w4a16.lib.w4a16_verify_tree_workspace(2, 4, 100000, ctypes.byref(need)) == 0 and need.value > 0
    assert w4a16.lib.w4a16_verify_tree_workspace(2, 4, 1000, None) == CONFIG


def test_binding():
    ints = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(w4a16.W4A16Error):
        w4a16.verify_tree(torch.zeros(1, 2, 5), ints, ints, torch.zeros(1, 2))
