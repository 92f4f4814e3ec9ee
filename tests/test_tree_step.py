"""The operators of drafted trees and of beam search together, on the GPU. A step of a tree: grown level by level by beam selection over a
draft's cache, planned, its rows turned and written, attended in two layers, verified, its path kept and the lengths cut back. A step of a beam
search: selection, tables, last pages, the new tokens' append, attention. Each operator against its oracle on what it was given, what
the caches hold after every step against a plain append of the tokens that stand, and the whole step in one graph against the eager one.
Queries, keys and values of a token are rows of fixed tables, so what a cache has to hold is known from the tokens alone."""

import numpy as np
import pytest
import torch

import kv_check
import kv_oracle
import rope_oracle
import tree_oracle
import w4a16
from oracle import oracle
from test_beams import best, tables_of
from test_paged_attention import whole

pytestmark = pytest.mark.gpu

Q_HEADS, KV_HEADS, DIM, VOCAB, PAGE, COLUMNS = 4, 2, 64, 512, 8, 12
HEADS = Q_HEADS + 2 * KV_HEADS


class Layer:
    """A layer's cache, and the queries, keys and values of every token."""

    def __init__(self, pages, fmt, seed, cuda):
        self.cache = w4a16.KvCache.empty(pages, PAGE, KV_HEADS, DIM, fmt, device=cuda)
        self.fmt, gen = fmt, torch.Generator().manual_seed(seed)
        self.of = torch.randn(VOCAB, HEADS, DIM, generator=gen).to(torch.bfloat16).to(cuda)

    def run(self, tokens, batch, rope, positions=None, tree=None):
        """The layer's attention of these tokens, and what it was computed from."""
        q, k, v = self.of[tokens.reshape(-1)].split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
        turned = self.cache.append(k, v, batch, rope, q=q, positions=positions)
        out, lse = w4a16.paged_attention(turned, self.cache, batch, return_lse=True, tree=tree)
        return q, turned, out, lse


def vocabulary(cuda, seed):
    n, k = VOCAB, Q_HEADS * DIM
    return w4a16.TiledWeight.from_artifact(*oracle.quantize(8 * oracle.synth_weight(n, k, seed)), n, k, device=cuda)


def logits_of(attended, weight, seqs, rows):
    return w4a16.gemm_int4_bf16(attended.reshape(seqs * rows, -1), weight).view(seqs, rows, VOCAB)


def check_queries(q, turned, positions, rope):
    want, off = rope_oracle.turned(q.cpu(), torch.as_tensor(positions), rope.inv_freq.cpu(), rope.interleaved)
    got = turned.cpu().double()
    assert ((got - want).abs() <= off + 2.0**-8 * (want.abs() + off) + 2.0**-134).all()


def check_texts(layer, table, texts, rope, cuda):
    """The cache holds the texts' tokens, every one at its place in its text, as a plain append of them all leaves them."""
    lens = [len(t) for t in texts]
    batch = w4a16.KvBatch(torch.tensor(table, dtype=torch.int32, device=cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                          torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=cuda), sum(lens))
    plain = w4a16.KvCache.empty(len(texts) * COLUMNS, PAGE, KV_HEADS, DIM, layer.fmt, device=cuda)
    apart = torch.arange(len(texts) * COLUMNS, dtype=torch.int32, device=cuda).view(-1, COLUMNS)
    own = w4a16.KvBatch(apart, batch.kv_lens, batch.starts, batch.rows)
    tokens = torch.tensor([t for text in texts for t in text], device=cuda)
    _, k, v = layer.of[tokens].split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
    plain.append(k, v, own, rope)
    for a, b in zip(layer.cache.read(batch), plain.read(own)):
        assert torch.equal(a, b)


def same(eager, replayed):
    assert eager.keys() == replayed.keys()
    for name, a in eager.items():
        for x, y in zip(a, replayed[name]):
            assert (x is None and y is None) or torch.equal(x, y), name


SEQS, WIDTH = 2, 3
NODES = 1 + 2 * WIDTH


class TreeStep:
    def __init__(self, fmt, weights, rope, cuda):
        pages = SEQS * COLUMNS + 3
        self.draft, self.layers = Layer(pages, fmt, 1, cuda), [Layer(pages, fmt, 1 + i, cuda) for i in range(2)]
        self.weights, self.rope = weights, rope
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:SEQS * COLUMNS].reshape(SEQS, COLUMNS)
        self.table = order.tolist()
        table = order.to(torch.int32).to(cuda)
        self.kv_lens, self.grown = (torch.zeros(SEQS, dtype=torch.int32, device=cuda) for _ in range(2))
        self.last = torch.tensor([[5], [9]], dtype=torch.int32, device=cuda)
        self.uniforms = torch.zeros(SEQS, NODES, device=cuda)
        self.tokens = torch.zeros(SEQS, NODES, dtype=torch.int32, device=cuda)
        self.parents = torch.full((SEQS, NODES), -1, dtype=torch.int32, device=cuda)

        def batch(lens, rows):
            starts = torch.arange(SEQS + 1, dtype=torch.int32, device=cuda) * rows
            return w4a16.KvBatch(table, lens, starts, SEQS * rows, max_new=rows, max_kv=PAGE * COLUMNS)

        # the levels as they grow: the nodes so far, and of the rows the last ones
        self.levels = []
        for nodes, rows in ((1, 1), (1 + WIDTH, WIDTH), (NODES, WIDTH)):
            level = batch(self.grown, rows)
            self.levels.append((rows, level, w4a16.KvTree(self.parents[:, :nodes], level)))
        self.batch = batch(self.kv_lens, NODES)
        self.tree = w4a16.KvTree(self.parents, self.batch)
        self.zeros = torch.zeros(SEQS, 1, device=cuda)

    def run(self):
        seen = {}
        self.tokens[:, :1] = self.last
        self.grown.copy_(self.kv_lens)
        first, scores, frontier = 0, self.zeros, None
        for i, (rows, batch, tree) in enumerate(self.levels):
            self.grown += rows
            tree.update()
            tokens = self.tokens[:, first:first + rows]
            q, turned, out, lse = self.draft.run(tokens, batch, self.rope, tree.positions, tree)
            seen[f"level {i}"] = q, turned, out, lse, tree.positions.clone(), tree.seen.clone()
            if i == len(self.levels) - 1:
                break
            logits = logits_of(out, self.weights[0], SEQS, rows)
            chosen = w4a16.beam_select(logits, scores, WIDTH)
            seen[f"chosen {i}"] = (logits, scores.clone(), *chosen)
            scores, frontier, words = chosen
            self.parents[:, first + rows:first + rows + WIDTH] = frontier + first
            self.tokens[:, first + rows:first + rows + WIDTH] = words
            first += rows
        self.kv_lens += NODES
        self.tree.update()
        seen["plan"] = self.tree.positions.clone(), self.tree.seen.clone(), self.tokens.clone(), self.parents.clone()
        for i, layer in enumerate(self.layers):
            seen[f"layer {i}"] = layer.run(self.tokens, self.batch, self.rope, self.tree.positions, self.tree)
        # mostly what the draft said
        logits = logits_of(seen["layer 0"][2], self.weights[0], SEQS, NODES) + 0.25 * logits_of(seen["layer 1"][2], self.weights[1], SEQS, NODES)
        target = torch.softmax(logits.float(), -1)
        accepted, path, tokens = w4a16.verify_tree(target, self.tokens, self.parents, self.uniforms)
        seen["verified"] = target, accepted, path, tokens
        for layer in (self.draft, *self.layers):
            layer.cache.keep_path(self.batch, path)
        self.kv_lens -= NODES - 1 - accepted
        self.last.copy_(tokens.gather(1, accepted[:, None].long()))
        return seen


def tree_attention(layer, table, lens, news, parents, nodes, seen):
    """(q, turned, out, lse) of a layer's call against FP64 over what its cache holds now."""
    _, turned, out, lse = seen
    sizes = [nodes] * SEQS
    by, positions = tree_oracle.plan(parents, sizes, lens, news, nodes)
    k, v, there = whole(layer.cache, table, lens, PAGE, layer.cache.num_pages)
    coded = kv_check.sizes(layer.cache, table, lens, PAGE, layer.cache.num_pages)
    views = tree_oracle.visible(by, positions, sizes, lens, news, nodes, 0)
    tree_oracle.check(out, lse, tree_oracle.attention(turned.cpu(), k, v, there, views, DIM**-0.5, coded))


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
def test_trees(cuda, fmt):
    rope = w4a16.Rope.of(DIM, device=cuda)
    weights = [vocabulary(cuda, 11), vocabulary(cuda, 12)]
    eager, captured = (TreeStep(fmt, weights, rope, cuda) for _ in range(2))
    captured.run()  # once before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = captured.run()
    captured.kv_lens.zero_()
    captured.last.copy_(eager.last)
    texts, taken = [[] for _ in range(SEQS)], []
    for n in range(6):
        print(f"tree step {fmt} {n} lens={[len(t) for t in texts]}", flush=True)
        u = torch.rand(SEQS, NODES, generator=torch.Generator().manual_seed(n))
        u[:, 1:] *= 1 if n % 2 else 0.1  # some are taken
        for step in (eager, captured):
            step.uniforms.copy_(u)
        last = eager.last.flatten().tolist()
        before = eager.kv_lens.tolist()
        assert before == [len(t) for t in texts]
        # what the attention reads is gone after the path is kept: taken before that
        keep, checks = w4a16.KvCache.keep_path, []

        def first_look(cache, batch, path):
            if not checks:
                for i, layer in enumerate((eager.draft, *eager.layers)):
                    checks.append([None if t is None else t.clone() for t in (layer.cache.k, layer.cache.v, layer.cache.k_scale,
                                                                             layer.cache.v_scale)])
            keep(cache, batch, path)

        with pytest.MonkeyPatch.context() as patch:
            patch.setattr(w4a16.KvCache, "keep_path", first_look)
            got = eager.run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(got, replayed)
        assert torch.equal(eager.kv_lens, captured.kv_lens) and torch.equal(eager.last, captured.last)
        # the tree
        positions, bits, tokens, parents = (t.cpu() for t in got["plan"])
        lens = [m + NODES for m in before]
        by, at = tree_oracle.plan(parents.tolist(), [NODES] * SEQS, lens, [NODES] * SEQS, NODES)
        assert torch.equal(bits, tree_oracle.bits(by, NODES)) and positions.tolist() == at
        assert tokens[:, 0].tolist() == last
        for i, first in ((0, 0), (1, 1)):
            logits, scores, found, up, words = (t.cpu() for t in got[f"chosen {i}"])
            for s in range(SEQS):
                want, _, _, every = best(logits[s], scores[s], WIDTH)
                assert (np.abs(found[s].numpy() - want) <= 2.0**-21 + np.abs(want) * 2.0**-23).all()
                index = up[s].numpy() * VOCAB + words[s].numpy()
                assert len(set(index)) == WIDTH and (np.abs(every[index] - want) <= 2.0**-20).all()
            behind = slice(1 + first * WIDTH, 1 + (first + 1) * WIDTH)
            assert torch.equal(parents[:, behind], up + first) and torch.equal(tokens[:, behind], words)
        # attention and queries, over the caches as they were
        for layer, tensors in zip((eager.draft, *eager.layers), checks):
            now = [getattr(layer.cache, name) for name in ("k", "v", "k_scale", "v_scale")]
            after = [None if t is None else t.clone() for t in now]
            for t, was in zip(now, tensors):
                if t is not None:
                    t.copy_(was)
            if layer is eager.draft:
                grown = 0
                for i, (rows, _, _) in enumerate(eager.levels):
                    grown += rows
                    *call, places, _ = got[f"level {i}"]
                    check_queries(call[0], call[1], places.cpu(), rope)
                    tree_attention(layer, eager.table, [m + grown for m in before], [rows] * SEQS, parents[:, :grown].tolist(), grown, call)
            else:
                call = got[f"layer {eager.layers.index(layer)}"]
                check_queries(call[0], call[1], positions, rope)
                tree_attention(layer, eager.table, lens, [NODES] * SEQS, parents.tolist(), NODES, call)
            for t, was in zip(now, after):
                if t is not None:
                    t.copy_(was)
        # what stands
        target, accepted, path, new = got["verified"]
        want = tree_oracle.verify(target.cpu().numpy(), tokens.numpy(), parents.numpy(), None, u.numpy())
        for a, b in zip((accepted, path, new), want):
            assert a.tolist() == b.tolist()
        for s in range(SEQS):
            texts[s] += [last[s]] + want[2][s][:want[0][s]].tolist()
            taken.append(int(want[0][s]))
        assert eager.kv_lens.tolist() == [len(t) for t in texts]
        for step in (eager, captured):
            for layer in (step.draft, *step.layers):
                check_texts(layer, step.table, texts, rope, cuda)
    assert len(set(taken)) > 1


GROUPS, BEAMS = 2, 4


class BeamStep:
    def __init__(self, fmt, weight, rope, prompt, cuda):
        seqs = GROUPS * BEAMS
        self.layer = Layer(seqs * COLUMNS, fmt, 1, cuda)
        self.weight, self.rope = weight, rope
        order = torch.randperm(seqs * COLUMNS, generator=torch.Generator().manual_seed(2)).to(torch.int32).reshape(seqs, COLUMNS)
        self.table = order.to(cuda)
        self.kv_lens = torch.full((seqs,), prompt.shape[1], dtype=torch.int32, device=cuda)
        self.scores = torch.full((GROUPS, BEAMS), float("-inf"), device=cuda)
        self.scores[:, 0] = 0
        # the prompt in every group's first beam: the others go on from it
        batch = w4a16.KvBatch(self.table[::BEAMS], self.kv_lens[::BEAMS].contiguous(),
                              torch.arange(GROUPS + 1, dtype=torch.int32, device=cuda) * prompt.shape[1], prompt.numel())
        self.logits = torch.zeros(GROUPS, BEAMS, VOCAB, dtype=torch.bfloat16, device=cuda)
        out = self.layer.run(prompt.to(cuda), batch, rope)[2].view(GROUPS, prompt.shape[1], -1)[:, -1]
        self.logits[:, 0] = logits_of(out.contiguous(), weight, GROUPS, 1)[:, 0]
        starts = torch.arange(seqs + 1, dtype=torch.int32, device=cuda)
        self.batch = w4a16.KvBatch(self.table, self.kv_lens, starts, seqs, max_new=1, max_kv=PAGE * COLUMNS)

    def run(self):
        given = self.logits.clone(), self.scores.clone(), self.table.clone()
        scores, parents, tokens = w4a16.beam_select(self.logits, self.scores, BEAMS)
        table, source = w4a16.beam_tables(self.table, self.kv_lens, parents, PAGE)
        self.layer.cache.copy_tails(table, self.kv_lens, source)
        self.table.copy_(table)
        self.kv_lens += 1
        call = self.layer.run(tokens, self.batch, self.rope)
        self.scores.copy_(scores)
        self.logits.copy_(logits_of(call[2], self.weight, GROUPS, BEAMS))
        return dict(given=given, chosen=(scores, parents, tokens), moved=(table, source), call=call)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
def test_beams(cuda, fmt):
    rope, weight = w4a16.Rope.of(DIM, interleaved=True, device=cuda), vocabulary(cuda, 13)
    prompt = torch.randint(0, VOCAB, (GROUPS, 13), generator=torch.Generator().manual_seed(3))
    eager, captured, spare = (BeamStep(fmt, weight, rope, prompt, cuda) for _ in range(3))
    spare.run()  # once before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = captured.run()
    texts = [prompt[s // BEAMS].tolist() for s in range(GROUPS * BEAMS)]
    moved = 0
    for n in range(20):  # over two pages' ends
        got = eager.run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(got, replayed)
        logits, before, table = (t.cpu() for t in got["given"])
        scores, parents, tokens = (t.cpu().numpy() for t in got["chosen"])
        lens = [len(t) for t in texts]
        for g in range(GROUPS):
            want, _, _, every = best(logits[g], before[g], BEAMS)
            assert (np.abs(scores[g] - want) <= 2.0**-21 + np.abs(want) * 2.0**-23).all()
            index = parents[g].astype(np.int64) * VOCAB + tokens[g]
            assert (parents[g] >= 0).all() and len(set(index)) == BEAMS and (np.abs(every[index] - want) <= 2.0**-20).all()
        new, source = tables_of(table.tolist(), lens, parents.tolist(), PAGE)
        assert got["moved"][0].tolist() == new and got["moved"][1].tolist() == source
        moved += sum(x >= 0 for x in source)
        texts = [texts[s // BEAMS * BEAMS + parents[s // BEAMS, s % BEAMS]] + [int(tokens[s // BEAMS, s % BEAMS])] for s in range(len(texts))]
        q, turned, out, lse = got["call"]
        check_queries(q, turned, lens, rope)
        kv_check.check(out, lse, eager.layer.cache, new, turned.cpu(), [m + 1 for m in lens], [1] * len(lens), PAGE,
                       eager.layer.cache.num_pages, DIM**-0.5)
        for step in (eager, captured):
            check_texts(step.layer, new, texts, rope, cuda)
    assert moved
