"""Verification of drafted tokens on the GPU against the definition, token by token in FP64 (kv_oracle.verify): equal."""

import numpy as np
import pytest
import torch

import kv_oracle
import w4a16

pytestmark = pytest.mark.gpu


def same(cuda, target, draft, tokens, lens, uniforms):
    dev = [None if t is None else torch.as_tensor(t).to(cuda) for t in (target, tokens, uniforms, draft, lens)]
    accepted, out = w4a16.verify_drafts(dev[0], dev[1], dev[2], draft=dev[3], lens=dev[4])
    some, want = kv_oracle.verify(np.asarray(target), None if draft is None else np.asarray(draft), np.asarray(tokens),
                                  None if lens is None else np.asarray(lens), np.asarray(uniforms))
    assert accepted.tolist() == some.tolist()
    assert out.tolist() == want.tolist()
    return some, want


def random_case(seqs, steps, vocab, seed, noise=0.5, drawn=True):
    gen = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn(seqs, steps + 1, vocab, generator=gen)
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits[:, :steps] + noise * torch.randn(seqs, steps, vocab, generator=gen), -1)
    if steps and drawn:
        tokens = torch.multinomial(draft.reshape(-1, vocab), 1, generator=gen).reshape(seqs, steps)
    else:
        tokens = draft.argmax(-1)
    return target, draft if drawn else None, tokens.to(torch.int32), torch.rand(seqs, steps + 1, generator=gen)


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("seqs,steps,vocab", [(1, 1, 1), (1, 0, 17), (3, 4, 2), (5, 3, 1000), (2, 1, 4095), (2, 2, 4097),
                                              (3, 16, 8192), (3, 16, 8193), (2, 70, 513), (6, 4, 32000), (2, 3, 32768), (2, 3, 32769), (4, 5, 50257), (1, 4, 151936), (200, 2, 301)])
def test_against_the_definition(cuda, seqs, steps, vocab, drawn):
    print(f"drafts seqs={seqs} steps={steps} vocab={vocab} drawn={drawn}", flush=True)
    for seed in range(3):
        target, draft, tokens, uniforms = random_case(seqs, steps, vocab, seed, drawn=drawn)
        same(cuda, target, draft, tokens, None, uniforms)
        lens = torch.randint(-1, steps + 2, (seqs,), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        same(cuda, target, draft, tokens, lens, uniforms)


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("vocab", [300, 10000, 20000])
def test_many_taken(cuda, vocab, drawn):
    """More drafted tokens than a wave has lanes, of which 0, 63, 64, 65, 128, 149 and all are taken."""
    taken, steps = [0, 63, 64, 65, 128, 149, 150], 150
    gen = torch.Generator().manual_seed(7)
    target = torch.rand(len(taken), steps + 1, vocab, generator=gen) / vocab
    draft = torch.rand(len(taken), steps, vocab, generator=gen) / vocab
    tokens = torch.randint(0, vocab, (len(taken), steps), generator=gen).to(torch.int32)
    uniforms = torch.rand(len(taken), steps + 1, generator=gen)
    at = tokens.long()[..., None]
    target[:, :steps].scatter_(2, at, 1.0)
    draft.scatter_(2, at, 0.5)
    for s, n in enumerate(taken):
        if n < steps:
            target[s, n, tokens[s, n]] = 0.0
    accepted, _ = same(cuda, target, draft if drawn else None, tokens, None, uniforms)
    assert accepted.tolist() == taken


def test_borders(cuda):
    """Exact ties: dyadic weights whose sums are exact in any order. The threshold is passed, not reached; a uniform of 0
    takes the first token that weighs anything; a product equal to the target's probability refuses."""
    target = torch.zeros(6, 2, 8)
    target[:, :, 1] = 0.25
    target[:, :, 3] = 0.5
    target[:, :, 6] = 0.25
    draft = torch.zeros(6, 1, 8)
    draft[:, :, 3] = 1.0
    tokens = torch.full((6, 1), 3, dtype=torch.int32)
    uniforms = torch.tensor([[0.5, 0.0], [0.49, 0.25], [0.5, 0.5], [0.75, 0.49], [0.1, 0.75], [0.9, 1.0]])
    some, out = same(cuda, target, draft, tokens, None, uniforms)
    assert some.tolist() == [0, 1, 0, 0, 1, 0]
    assert out[:, 0].tolist() == [1, 3, 6, 1, 3, 6] and out[1, 1] == 3 and out[4, 1] == 6


@pytest.mark.parametrize("vocab", [5000, 9000, 40000])
def test_weights_that_are_none(cuda, vocab):
    """Nothing left of the target where the draft refused: the target itself. Rows of zeros, NaN and infinities: no token.
    Tokens outside the vocabulary are refused; NaN uniforms refuse, and draw the last token that weighs anything."""
    target, draft, tokens, uniforms = random_case(8, 2, vocab, 1)
    draft[0, 0] = target[0, 0] * 2          # nothing left
    uniforms[0, 0] = 0.9
    target[1, 0] = 0                         # no weights at all
    target[2, 0, 5:4000] = float("nan")
    target[2, 0, 7] = float("inf")
    uniforms[2, 0] = 1.0
    tokens[3, 0] = vocab
    tokens[4, 0] = -1
    uniforms[5, 0] = float("nan")
    uniforms[6, 2] = float("nan")
    target[7, :, :] = -1.0
    some, out = same(cuda, target, draft, tokens, None, uniforms)
    assert some[[0, 1, 3, 4, 5, 7]].tolist() == [0] * 6 and out[1, 0] == -1 and out[7, 0] == -1
    same(cuda, target, None, tokens, None, uniforms)


def test_strided_rows(cuda):
    """Rows that stand apart, at odd addresses, and one draft row for every step."""
    target, draft, tokens, uniforms = random_case(4, 3, 3001, 7)
    wide = torch.zeros(4, 6, 3005)
    wide[:, 1:5, 3:3004] = target
    one = draft[:, :1].expand(4, 3, 3001)
    dev = wide.to(cuda)
    accepted, out = w4a16.verify_drafts(dev[:, 1:5, 3:3004], tokens.to(cuda), uniforms.to(cuda),
                                        draft=draft[:, :1].to(cuda).expand(4, 3, 3001))
    some, want = kv_oracle.verify(target.numpy(), one.numpy(), tokens.numpy(), None, uniforms.numpy())
    assert accepted.tolist() == some.tolist() and out.tolist() == want.tolist()


def test_captured(cuda):
    """In a graph, replayed with other inputs and eager work between."""
    shape = (5, 3, 40007)
    dev = [t.to(cuda) for t in random_case(*shape, 1)]
    call = lambda: w4a16.verify_drafts(dev[0], dev[2], dev[3], draft=dev[1])  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        accepted, tokens = call()
    for seed in range(2, 6):
        for to, t in zip(dev, random_case(*shape, seed)):
            to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        again = call()
        assert torch.equal(accepted, again[0]) and torch.equal(tokens, again[1])


def test_the_sampled_distribution(cuda):
    """Over many draws the first token is distributed as the target's row, whatever the draft: the counts of 40000
    sequences lie within five standard deviations of it."""
    vocab, seqs = 6, 40000
    p = torch.tensor([0.05, 0.3, 0.2, 0.02, 0.33, 0.1])
    q = torch.tensor([0.3, 0.1, 0.2, 0.2, 0.1, 0.1])
    gen = torch.Generator().manual_seed(1)
    tokens = torch.multinomial(q.expand(seqs, vocab), 1, generator=gen).to(torch.int32)
    got = [w4a16.verify_drafts(p.to(cuda).expand(n, 2, vocab), tokens[a:a + n].to(cuda),
                               torch.rand(n, 2, generator=gen).to(cuda), draft=q.to(cuda).expand(n, 1, vocab))[1][:, 0]
           for a, n in ((0, 30000), (30000, 10000))]
    share = torch.bincount(torch.cat(got).cpu().long(), minlength=vocab).double() / seqs
    assert ((share - p).abs() <= 5 * (p * (1 - p) / seqs).sqrt()).all()
