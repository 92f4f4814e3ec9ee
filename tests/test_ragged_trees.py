"""Steps of drafted trees of different sizes in one batch, one of a root alone among them, on the GPU: appended, attended, verified, their paths kept
and the lengths cut back by each tree's own size. After every step the caches hold the tokens that stand, as a plain append of them leaves them."""

import numpy as np
import pytest
import torch

import test_tree_attention as short
import tree_oracle
import w4a16
from test_tree_step import COLUMNS, DIM, KV_HEADS, PAGE, Q_HEADS, VOCAB, Layer, check_texts, logits_of, vocabulary

pytestmark = pytest.mark.gpu

SEQS, NODES = 4, 9


@pytest.mark.parametrize("prompt", [0, 5])
@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
def test_steps(cuda, fmt, prompt):
    """`prompt`: rows of other tokens stand before each tree in the first step's call; the paths are then kept by a batch of the trees alone."""
    rope, weight = w4a16.Rope.of(DIM, device=cuda), vocabulary(cuda, 21)
    layer = Layer(SEQS * COLUMNS, fmt, 3, cuda)
    table = torch.arange(SEQS * COLUMNS, dtype=torch.int32, device=cuda).view(SEQS, COLUMNS)
    kv_lens = torch.zeros(SEQS, dtype=torch.int32, device=cuda)
    texts, last, taken = [[] for _ in range(SEQS)], [3, 1, 4, 15], set()
    for n in range(8):
        gen = torch.Generator().manual_seed(n)
        sizes = torch.randint(2, NODES + 1, (SEQS,), generator=gen).to(torch.int32)
        sizes[n % SEQS] = n % 3  # no node or a root: a row either way, the last token's
        rows = sizes.clamp(1, NODES)
        tokens = torch.randint(0, VOCAB, (SEQS, NODES), generator=gen).to(torch.int32)
        tokens[:, 0] = torch.tensor(last, dtype=torch.int32)
        parents = short.random_parents(SEQS, NODES, n, "random")
        before = prompt if n == 0 else 0
        extra = torch.randint(0, VOCAB, (SEQS, before), generator=gen).to(torch.int32)
        news = (rows + before).tolist()
        starts = torch.tensor([0, *np.cumsum(news)], dtype=torch.int32, device=cuda)
        kv_lens += (rows + before).to(cuda)
        batch = w4a16.KvBatch(table, kv_lens, starts, sum(news))
        tree = w4a16.KvTree(parents.to(cuda), batch, sizes=sizes.to(cuda))
        flat = torch.cat([torch.cat([extra[s], tokens[s, :rows[s]]]) for s in range(SEQS)])
        out = layer.run(flat.to(cuda), batch, rope, tree.positions, tree)[2]
        # the target's rows behind the nodes; what the tree holds is likely
        logits = torch.zeros(SEQS, NODES, VOCAB, device=cuda)
        every = logits_of(out, weight, 1, sum(news))[0].float()
        for s in range(SEQS):
            first = int(starts[s]) + before
            logits[s, :rows[s]] = every[first:first + int(rows[s])]
            for i in range(1, int(rows[s])):
                logits[s, parents[s, i], tokens[s, i].long()] += 9.0
        target = torch.softmax(logits, -1)
        uniforms = torch.rand(SEQS, NODES, generator=gen)
        device = [t.to(cuda) for t in (tokens, parents, uniforms, sizes)]
        accepted, path, new = w4a16.verify_tree(target, device[0], device[1], device[2], sizes=device[3])
        want = tree_oracle.verify(target.cpu().numpy(), tokens.numpy(), parents.numpy(), sizes.numpy(), uniforms.numpy())
        for a, b in zip((accepted, path, new), want):
            assert a.tolist() == b.tolist()
        if before:  # the rows of the path's batch are the trees' nodes and no others
            of_trees = torch.tensor([0, *np.cumsum(rows.tolist())], dtype=torch.int32, device=cuda)
            batch = w4a16.KvBatch(table, kv_lens, of_trees, int(rows.sum()))
        layer.cache.keep_path(batch, path)
        kv_lens -= device[3].clamp(1, NODES) - 1 - accepted
        for s in range(SEQS):
            texts[s] += extra[s].tolist() + [last[s]] + want[2][s][:want[0][s]].tolist()
            last[s] = int(want[2][s][want[0][s]])
            taken.add(int(want[0][s]))
        assert kv_lens.tolist() == [len(t) for t in texts]
        check_texts(layer, table.tolist(), texts, rope, cuda)
    assert max(taken) >= 3 and min(taken) == 0
