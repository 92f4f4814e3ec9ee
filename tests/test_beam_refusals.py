"""What beam selection, its tables and the moves in the cache refuse, on the CPU: every refusal comes before any launch, with a reason."""

import ctypes

import pytest
import torch

import w4a16
from test_kv_refusals import A, CONFIG, batch, cache


def select(kind="f32", logits=A * 16, strides=(40000, 10000), scores=A, groups=2, beams=4, vocab=10000, take=8, out=A * 2, parents=A * 3,
           tokens=A * 4, ws=A * 5, ws_bytes=1 << 20):
    call = w4a16.lib.w4a16_beam_select_f32 if kind == "f32" else w4a16.lib.w4a16_beam_select_bf16
    return call(logits, *strides, scores, groups, beams, vocab, take, out, parents, tokens, ws, ws_bytes, None)


def tables(table=A, stride=10, pages=10, lens=A * 2, parents=A * 3, groups=2, beams=4, page=16, out=A * 4, out_stride=10, source=A * 5):
    return w4a16.lib.w4a16_beam_tables(table, stride, pages, lens, parents, groups, beams, page, out, out_stride, source, None)


def tails(c=None, table=A * 600, stride=10, pages=10, lens=A * 601, source=A * 602, seqs=3):
    return w4a16.lib.w4a16_kv_copy_tails(ctypes.byref(c or cache()), table, stride, pages, lens, source, seqs, None)


def keep(c=None, b=None, path=A * 600, width=5):
    return w4a16.lib.w4a16_kv_keep_path(ctypes.byref(c or cache()), ctypes.byref(b or batch()), path, width, None)


@pytest.mark.parametrize("call,args,why", [
    (select, dict(groups=-1), "extents"), (select, dict(groups=65536), "extents"), (select, dict(beams=0), "extents"),
    (select, dict(beams=1025), "extents"), (select, dict(vocab=0), "extents"), (select, dict(beams=1000, vocab=1 << 22), "extents"),
    (select, dict(take=0), "take"), (select, dict(take=129), "take"), (select, dict(logits=None), "null"), (select, dict(scores=None), "null"),
    (select, dict(out=None), "null"), (select, dict(parents=None), "null"), (select, dict(tokens=None), "null"), (select, dict(ws=None), "null"),
    (select, dict(logits=A * 16 + 2), "aligned"), (select, dict(kind="bf16", logits=A * 16 + 1), "aligned"), (select, dict(out=A * 2 + 1), "aligned"),
    (select, dict(ws=A * 5 + 8), "aligned"), (select, dict(ws_bytes=64), "workspace"), (select, dict(strides=(-1, 10)), "stride"),
    (select, dict(strides=(1, 1 << 44)), "stride"), (select, dict(out=A * 16), "overlap"), (select, dict(parents=A * 2), "overlap"),
    (select, dict(tokens=A), "overlap"), (select, dict(ws=A * 16 + 16), "overlap"), (select, dict(ws=A * 4), "overlap"),
    (tables, dict(groups=-1), "extents"), (tables, dict(beams=0), "extents"), (tables, dict(beams=1025), "extents"), (tables, dict(pages=-1), "extents"),
    (tables, dict(stride=9), "extents"), (tables, dict(out_stride=9), "extents"), (tables, dict(page=12), "page_size"), (tables, dict(page=4), "page_size"),
    (tables, dict(table=None), "null"), (tables, dict(lens=None), "null"), (tables, dict(parents=None), "null"), (tables, dict(out=None), "null"),
    (tables, dict(source=None), "null"), (tables, dict(out=A * 4 + 2), "aligned"), (tables, dict(out=A), "overlap"), (tables, dict(source=A * 3), "overlap"),
    (tables, dict(source=A * 4 + 64), "overlap"), (tables, dict(out=A * 2), "overlap"),
    (tails, dict(c=cache(head_dim=100)), "head_dim"), (tails, dict(seqs=-1), "extents"), (tails, dict(stride=9), "extents"),
    (tails, dict(c=cache(kv_heads=32768, page_size=8)), "kv_heads"), (tails, dict(table=None), "null"), (tails, dict(lens=None), "null"),
    (tails, dict(source=None), "null"), (tails, dict(source=A * 602 + 2), "aligned"), (tails, dict(source=A), "overlap"), (tails, dict(lens=A * 64), "overlap"),
    (tails, dict(table=A + 64), "overlap"), (tails, dict(c=cache(v=A + 1024)), "overlap"),
    (keep, dict(c=cache(head_dim=100)), "head_dim"), (keep, dict(b=batch(seqs=-1)), "extents"), (keep, dict(width=-1), "width"),
    (keep, dict(path=None), "null"), (keep, dict(path=A * 600 + 2), "aligned"), (keep, dict(path=A), "overlap"),
    (keep, dict(c=cache(format=2, k_scale=A * 600, v_scale=A * 3)), "overlap"),
])
def test_calls(call, args, why):
    assert call(**args) == CONFIG
    assert why in w4a16.last_error()


def test_nothing_to_do():
    assert select(groups=0) == 0 and tables(groups=0) == 0 and tails(seqs=0) == 0 and tails(pages=0) == 0 and keep(width=0) == 0
    assert keep(b=batch(rows=0)) == 0 and keep(b=batch(seqs=0)) == 0
    assert w4a16.lib.w4a16_beam_select_workspace(1, 1, 1, None) == CONFIG


def test_binding():
    for make in (lambda: w4a16.beam_select(torch.zeros(1, 2, 5), torch.zeros(1, 2), 1),
                 lambda: w4a16.beam_tables(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                                           torch.zeros(1, 2, dtype=torch.int32), 8)):
        with pytest.raises(w4a16.W4A16Error):
            make()
