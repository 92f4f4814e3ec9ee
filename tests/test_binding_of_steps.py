"""What the Python entry points of the append, the trees and the beams refuse on the GPU before anything is launched, and what a call takes that
no other test gives it: nothing at all, one of everything, a workspace or a stream of the caller's."""

import ctypes

import pytest
import torch

import w4a16
from test_kv_cache import filled, make_batch

pytestmark = pytest.mark.gpu


@pytest.fixture
def step(cuda):
    class Step:
        cache = filled(12, 16, 2, 64, "fp8", cuda, seed=1)
        batch, _ = make_batch([40, 30], [4, 3], 16, 12, cuda)
        other, _ = make_batch([40, 30], [4, 3], 16, 12, cuda)
        rope = w4a16.Rope.of(64, device=cuda)
        parents = torch.tensor([[-1, 0, 0, 1]] * 2, dtype=torch.int32, device=cuda)
        tree = w4a16.KvTree(parents, batch)
        k, v = (torch.randn(7, 2, 64, device=cuda).to(torch.bfloat16) for _ in range(2))
        q = torch.randn(7, 4, 64, device=cuda).to(torch.bfloat16)
        logits, scores = torch.randn(2, 3, 100, device=cuda), torch.zeros(2, 3, device=cuda)
        target = torch.softmax(torch.randn(2, 4, 100, device=cuda), -1)
        words, uniforms = torch.zeros(2, 4, dtype=torch.int32, device=cuda), torch.rand(2, 4, device=cuda)
        table, lens = batch.page_table, batch.kv_lens

    return Step


@pytest.mark.parametrize("call", [
    lambda s: w4a16.Rope(s.rope.inv_freq.double()), lambda s: w4a16.Rope(s.rope.inv_freq.cpu()), lambda s: w4a16.Rope(s.rope.inv_freq[:3]),
    lambda s: w4a16.Rope(s.rope.inv_freq[::2]), lambda s: w4a16.Rope.of(12), lambda s: w4a16.Rope.of(0),
    lambda s: s.cache.append(s.k[:6], s.v, s.batch, s.rope), lambda s: s.cache.append(s.k, s.v.float(), s.batch, s.rope),
    lambda s: s.cache.append(s.k.cpu(), s.v, s.batch, s.rope), lambda s: s.cache.append(s.k, s.v, s.batch, w4a16.Rope.of(72)),
    lambda s: s.cache.append(s.k, s.v, s.batch, s.rope, q=s.q[:, :, :32]), lambda s: s.cache.append(s.k, s.v, s.batch, s.rope, out=s.q),
    lambda s: s.cache.append(s.k, s.v, s.batch, s.rope, positions=torch.zeros(7, dtype=torch.int64, device=s.k.device)),
    lambda s: s.cache.append(s.k, s.v, s.batch, s.rope, positions=s.tree.positions[:6]),
    lambda s: s.cache.append(s.k, s.v, s.batch, s.rope, q=s.q, out=s.q[:, :2]), lambda s: s.cache.append(s.k, s.v, s.batch, s.rope, q=s.q, out=s.q.float()),
    lambda s: s.cache.append(s.k, s.v, s.batch, s.rope, q=s.q, out=s.q.expand(1, 7, 4, 64)[0].transpose(0, 1)),
    lambda s: w4a16.KvTree(s.parents.long(), s.batch), lambda s: w4a16.KvTree(s.parents.cpu(), s.batch), lambda s: w4a16.KvTree(s.parents[:1], s.batch),
    lambda s: w4a16.KvTree(s.parents.t().contiguous().t(), s.batch), lambda s: w4a16.KvTree(s.parents.repeat(1, 65), s.batch),
    lambda s: w4a16.KvTree(s.parents[:, :0], s.batch), lambda s: w4a16.KvTree(s.parents, s.batch, sizes=s.lens[:1]),
    lambda s: w4a16.KvTree(s.parents, s.batch, sizes=s.lens.long()),
    lambda s: w4a16.paged_attention(s.q, s.cache, s.other, tree=s.tree), lambda s: w4a16.paged_attention(s.q, s.cache, s.batch, causal=False, tree=s.tree),
    lambda s: w4a16.paged_attention(s.q, s.cache, s.batch, window=3, tree=s.tree), lambda s: w4a16.paged_attention(s.q[:, :3], s.cache, s.batch, tree=s.tree),
    lambda s: w4a16.beam_select(s.logits[0], s.scores, 4), lambda s: w4a16.beam_select(s.logits.half(), s.scores, 4),
    lambda s: w4a16.beam_select(s.logits.transpose(1, 2), s.scores, 4), lambda s: w4a16.beam_select(s.logits, s.scores[:, :2], 4),
    lambda s: w4a16.beam_select(s.logits, s.scores, 0), lambda s: w4a16.beam_select(s.logits, s.scores, 129),
    lambda s: w4a16.beam_select(s.logits, s.scores, 4, workspace=torch.empty(8, dtype=torch.uint8, device=s.k.device)),
    lambda s: w4a16.beam_select(s.logits[:, :0], s.scores[:, :0], 4), lambda s: w4a16.beam_select(s.logits[:, :, :0], s.scores, 4),
    lambda s: w4a16.beam_tables(s.table, s.lens, s.words, 16), lambda s: w4a16.beam_tables(s.table.long(), s.lens, s.words[:1, :2], 16),
    lambda s: w4a16.beam_tables(s.table, s.lens, s.words[:1, :2].contiguous(), 17), lambda s: w4a16.beam_tables(s.table, s.lens, s.words[:1, :2].contiguous(), 16, out=s.table),
    lambda s: w4a16.beam_tables(s.table, s.lens, s.words[:1, :2].contiguous(), 16, out=s.table.float()),
    lambda s: s.cache.copy_tails(s.table, s.lens, s.lens[:1]), lambda s: s.cache.copy_tails(s.table, s.lens.long(), s.lens),
    lambda s: s.cache.copy_tails(s.table[0], s.lens, s.lens), lambda s: s.cache.keep_path(s.batch, s.words.long()),
    lambda s: s.cache.keep_path(s.batch, s.words[:1]), lambda s: s.cache.keep_path(s.batch, s.words[:, ::2]), lambda s: s.cache.keep_path(s.batch, s.words[0]),
    lambda s: w4a16.verify_tree(s.target.half(), s.words, s.parents, s.uniforms), lambda s: w4a16.verify_tree(s.target[0], s.words, s.parents, s.uniforms),
    lambda s: w4a16.verify_tree(s.target, s.words[:, :3], s.parents, s.uniforms), lambda s: w4a16.verify_tree(s.target, s.words, s.parents.long(), s.uniforms),
    lambda s: w4a16.verify_tree(s.target, s.words, s.parents, s.uniforms.double()), lambda s: w4a16.verify_tree(s.target.transpose(1, 2), s.words, s.parents, s.uniforms),
    lambda s: w4a16.verify_tree(s.target, s.words, s.parents, s.uniforms, sizes=s.lens[:1]), lambda s: w4a16.verify_tree(s.target, s.words, s.parents, s.uniforms.cpu()),
])
def test_refused(step, call):
    before = [t.clone() for t in (step.cache.k.view(torch.uint8), step.cache.v.view(torch.uint8), step.q, step.table, step.lens, step.tree.seen)]
    with pytest.raises(w4a16.W4A16Error):
        call(step)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (step.cache.k.view(torch.uint8), step.cache.v.view(torch.uint8), step.q, step.table, step.lens,
                                                          step.tree.seen)))


def test_nothing_at_all(cuda):
    """No sequences, no rows, no groups: empty answers."""
    cache, rope = filled(4, 8, 1, 64, "bf16", cuda, seed=1), w4a16.Rope.of(16, device=cuda)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    for seqs in (0, 2):
        lens = torch.full((seqs,), 5, dtype=torch.int32, device=cuda)
        batch = w4a16.KvBatch(torch.zeros(seqs, 1, dtype=torch.int32, device=cuda), lens, torch.zeros(seqs + 1, dtype=torch.int32, device=cuda), 0)
        tree = w4a16.KvTree(torch.zeros(seqs, 3, dtype=torch.int32, device=cuda), batch)
        rows = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=cuda)
        assert cache.append(rows[:, :1], rows[:, :1], batch, rope, q=rows).shape == rows.shape
        assert w4a16.paged_attention(rows, cache, batch, tree=tree).shape == rows.shape
        cache.keep_path(batch, torch.zeros(seqs, 3, dtype=torch.int32, device=cuda))
    assert [t.shape for t in w4a16.beam_select(torch.zeros(0, 3, 9, device=cuda), torch.zeros(0, 3, device=cuda), 2)] == [(0, 2)] * 3
    table, source = w4a16.beam_tables(none.view(0, 4), none, none.view(0, 3), 8)
    assert table.shape == (0, 4) and source.shape == (0,)
    cache.copy_tails(none.view(0, 4), none, none)
    got = w4a16.verify_tree(torch.zeros(0, 3, 9, device=cuda), none.view(0, 3), none.view(0, 3), torch.zeros(0, 3, device=cuda))
    assert [t.shape for t in got] == [(0,), (0, 3), (0, 3)]
    torch.cuda.synchronize()


def test_streams_and_workspaces_of_the_caller(cuda, step):
    """Every entry point under a stream that is not the current one, with workspaces of the caller's: as without."""
    s, side = step, torch.cuda.Stream()
    mine = torch.empty(1 << 22, dtype=torch.uint8, device=cuda)
    stay, up = torch.full_like(s.words, -1), torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    no_tails = torch.full((2,), -1, dtype=torch.int32, device=cuda)

    def run(**on):
        space = dict(on, workspace=mine) if on else {}
        turned = s.cache.append(s.k, s.v, s.batch, s.rope, q=s.q, positions=s.tree.positions, **on)
        s.tree.update(**on)
        got = [turned, *w4a16.paged_attention(turned, s.cache, s.batch, return_lse=True, tree=s.tree, **space)]
        got += w4a16.beam_select(s.logits, s.scores, 5, **space)
        table, source = w4a16.beam_tables(s.table, s.lens, up, 16, **on)
        s.cache.copy_tails(table, s.lens, no_tails, **on)
        verified = w4a16.verify_tree(s.target, s.words, s.parents, s.uniforms, **space)
        s.cache.keep_path(s.batch, stay, **on)
        return [*got, table, source, *verified]

    want = run()
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    got = run(stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_workspace_queries(cuda, step):
    size = ctypes.c_size_t(0)
    for ask in (w4a16.lib.w4a16_paged_tree_attention_workspace, w4a16.lib.w4a16_paged_attention_workspace):
        assert ask(step.cache._ref, step.batch._ref, 4, ctypes.byref(size)) == 0
        assert ask(step.cache._ref, step.batch._ref, 3, ctypes.byref(size)) == w4a16.W4A16_ERR_CONFIG
        assert ask(step.cache._ref, step.batch._ref, 4, None) == w4a16.W4A16_ERR_CONFIG
        assert ask(step.cache._ref, None, 4, ctypes.byref(size)) == w4a16.W4A16_ERR_CONFIG
