"""Verification of drafted trees on the GPU against the definition, node by node in FP64 (tree_oracle.verify): equal."""

import numpy as np
import pytest
import torch

import tree_oracle
import w4a16
from test_tree_attention import random_parents

pytestmark = pytest.mark.gpu


def same(cuda, target, tokens, parents, sizes, uniforms):
    dev = [None if t is None else torch.as_tensor(t).to(cuda) for t in (target, tokens, parents, uniforms, sizes)]
    got = w4a16.verify_tree(dev[0], dev[1], dev[2], dev[3], sizes=dev[4])
    want = tree_oracle.verify(*(None if t is None else np.asarray(t) for t in (target, tokens, parents, sizes, uniforms)))
    for a, b in zip(got, want):
        assert a.tolist() == b.tolist()
    return want


def random_case(seqs, nodes, vocab, seed, kind="random"):
    """Trees whose children are mostly the likeliest words, with a few that come twice or are none."""
    gen = torch.Generator().manual_seed(seed)
    target = torch.softmax(2.5 * torch.randn(seqs, nodes, vocab, generator=gen), -1)
    parents = random_parents(seqs, nodes, seed, kind)
    like = target.topk(min(8, vocab), -1).indices
    rank = torch.randint(0, like.shape[-1], (seqs, nodes), generator=gen)
    tokens = like[torch.arange(seqs)[:, None], parents.long().clamp(0, nodes - 1), rank].to(torch.int32)
    odd = torch.rand(seqs, nodes, generator=gen) < 0.05
    tokens[odd] = torch.randint(-2, vocab + 2, (int(odd.sum()),), generator=gen).to(torch.int32)
    return target, tokens, parents, torch.rand(seqs, nodes, generator=gen) * torch.randint(0, 2, (seqs, nodes), generator=gen).clamp(min=0.1)


@pytest.mark.parametrize("kind", ["random", "chain", "star", "roots"])
@pytest.mark.parametrize("seqs,nodes,vocab", [(1, 1, 1), (1, 1, 70000), (3, 2, 2), (4, 26, 1000), (2, 63, 8192), (2, 64, 8193), (3, 65, 16384),
                                              (3, 129, 16385), (2, 256, 301), (2, 200, 20011), (5, 12, 50257), (1, 26, 151936)])
def test_against_the_definition(cuda, seqs, nodes, vocab, kind):
    print(f"tree seqs={seqs} nodes={nodes} vocab={vocab} {kind}", flush=True)
    for seed in range(3):
        target, tokens, parents, uniforms = random_case(seqs, nodes, vocab, seed, kind)
        same(cuda, target, tokens, parents, None, uniforms)
        sizes = torch.randint(-1, nodes + 2, (seqs,), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        same(cuda, target, tokens, parents, sizes, uniforms)


@pytest.mark.parametrize("vocab", [300, 40000])
def test_deep_and_wide(cuda, vocab):
    """Everything taken to the end of a chain of 256; every child of a star refused but the last, or all of them."""
    nodes = 256
    target = torch.full((4, nodes, vocab), 0.25 / vocab)
    tokens = torch.arange(nodes).expand(4, nodes).clone().to(torch.int32) % vocab
    parents = torch.stack([random_parents(1, nodes, 0, kind)[0] for kind in ("chain", "chain", "star", "star")])
    target[0].scatter_(1, tokens[0].roll(-1).long()[:, None], 0.9)
    target[1] = target[0]
    uniforms = torch.full((4, nodes), 0.5)
    uniforms[1, 200] = 0.95
    target[2, 0, int(tokens[2, 255])] = 0.6
    accepted, path, _ = same(cuda, target, tokens, parents, None, uniforms)
    assert accepted.tolist() == [255, 199, 1, 0] and path[2, 1] == 255


def test_borders(cuda):
    """Dyadic probabilities: a product equal to the probability refuses, what refused siblings leave is exact; a word that
    comes twice is refused with the first."""
    target = torch.zeros(6, 4, 8)
    target[:, 0, 1], target[:, 0, 3], target[:, 0, 5], target[:, 0, 6] = 0.25, 0.5, 0.125, 0.125
    target[:, 1:, 2] = 1.0
    tokens = torch.tensor([[0, 1, 3, 5]] * 6, dtype=torch.int32)
    tokens[5] = torch.tensor([0, 1, 1, 5])
    parents = torch.tensor([[-1, 0, 0, 0]] * 6, dtype=torch.int32)
    #                     drawn  1     3       5
    uniforms = torch.tensor([[0.9, 0.25, 0.6, 0.5],     # 1: 0.25 is not < 0.25; 3: 0.6 * 0.75 < 0.5
                             [0.0, 0.24, 0.9, 0.9],
                             [0.5, 0.99, 0.67, 0.49],   # 3: 0.5025 refused; 5: 0.49 * 0.25 < 0.125
                             [0.0, 0.99, 0.99, 0.5],    # 5: 0.125 is not < 0.125; drawn: 6, all that is left
                             [1.0, 0.99, 0.99, 0.99],
                             [0.8, 0.99, 0.0, 0.99]])   # 1 again: refused whatever its number; 3 or 6 drawn
    accepted, path, out = same(cuda, target, tokens, parents, None, uniforms)
    assert accepted.tolist() == [1, 1, 1, 0, 0, 0] and path[:3, 1].tolist() == [2, 1, 3] and out[3, 0] == 6 and out[4, 0] == 6
    assert out[5, 0] == 6


@pytest.mark.parametrize("vocab", [5000, 9000, 40000])
def test_weights_that_are_none(cuda, vocab):
    """Rows of zeros, NaN and infinities, children that hold all of the weight, numbers that are NaN, links that are none."""
    target, tokens, parents, uniforms = random_case(8, 7, vocab, 1)
    parents[:] = torch.tensor([-1, 0, 0, 1, 1, 2, 2])
    target[0] = 0
    target[1, 0] = 0
    target[1, 0, tokens[1, 1].long().clamp(0, vocab - 1)] = 1.0  # nothing left without it
    uniforms[1, 1] = 1.0
    target[2, 0, 5:4000] = float("nan")
    target[2, 0, 7] = float("inf")
    tokens[2, 1] = 7
    tokens[3, 1:] = vocab
    tokens[4, 1:] = -1
    uniforms[5] = float("nan")
    target[6] = -1.0
    parents[7] = torch.tensor([5, 7, -9, 3, 1 << 30, 4, 6])
    same(cuda, target, tokens, parents, None, uniforms)


def test_a_chain_is_verify_drafts(cuda):
    """A chain gives what the verification of drafted tokens gives for chosen tokens."""
    for vocab in (1000, 20011):
        target, tokens, parents, uniforms = random_case(6, 5, vocab, 3, "chain")
        target, tokens, uniforms = target.to(cuda), tokens.clamp(0, vocab - 1).to(cuda), uniforms.to(cuda)
        accepted, path, out = w4a16.verify_tree(target, tokens, parents.to(cuda), uniforms)
        want, drafts = w4a16.verify_drafts(target, tokens[:, 1:].contiguous(), torch.cat([uniforms[:, 1:], uniforms[:, :1]], 1))
        assert torch.equal(accepted, want) and torch.equal(out, drafts)


def test_strided_and_captured(cuda):
    """Rows that stand apart, at odd addresses; a graph with other inputs of each replay; another stream."""
    target, tokens, parents, uniforms = random_case(4, 9, 20011, 7)
    wide = torch.zeros(4, 12, 20017, device=cuda)
    view = wide[:, 2:11, 3:20014]
    dev = [t.to(cuda) for t in (tokens, parents, uniforms)]
    view.copy_(target)
    got = w4a16.verify_tree(view, *dev)
    for a, b in zip(got, tree_oracle.verify(target.numpy(), tokens.numpy(), parents.numpy(), None, uniforms.numpy())):
        assert a.tolist() == b.tolist()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = w4a16.verify_tree(view, *dev)
    for seed in range(2, 6):
        target, *more = random_case(4, 9, 20011, seed)
        view.copy_(target)
        for to, t in zip(dev, more):
            to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        again = w4a16.verify_tree(view, *dev)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = w4a16.verify_tree(view, *dev, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, again))


def test_the_sampled_distribution(cuda):
    """Over many draws the first token is distributed as the root's row, whatever its children: the counts of 40000
    sequences lie within five standard deviations of it."""
    vocab, seqs = 6, 40000
    p = torch.tensor([0.05, 0.3, 0.2, 0.02, 0.33, 0.1])
    gen = torch.Generator().manual_seed(1)
    tokens = torch.tensor([[0, 4, 2, 3]], dtype=torch.int32, device=cuda)
    parents = torch.tensor([[-1, 0, 0, 0]], dtype=torch.int32, device=cuda)
    got = []
    for n in (30000, 10000):
        got.append(w4a16.verify_tree(p.to(cuda).expand(n, 4, vocab), tokens.expand(n, 4).contiguous(), parents.expand(n, 4).contiguous(),
                                     torch.rand(n, 4, generator=gen).to(cuda))[2][:, 0])
    share = torch.bincount(torch.cat(got).cpu().long(), minlength=vocab).double() / seqs
    assert ((share - p).abs() <= 5 * (p * (1 - p) / seqs).sqrt()).all()
