"""Beam selection over more chunks than a block's threads hold (8192: 256 FP32 words each, 512 BF16), which is by pieces of four chunks first, on the
GPU against FP64 and a stable sort; and as many chunks as are still held."""

import pytest
import torch

import test_beams
from test_beams import check

pytestmark = pytest.mark.gpu

CASES = [
    # kind, groups, beams, vocab, take: chunks a beam
    ("fp32", 1, 1024, 2048, 40),     # 8: as many as are held
    ("fp32", 1, 911, 2100, 40),      # 9: more by a few, and a last piece of one chunk
    ("fp32", 2, 600, 3600, 128),     # 15
    ("fp32", 1, 1024, 2100, 1),
    ("bf16", 1, 1024, 4096, 33),     # 8
    ("bf16", 2, 1024, 4100, 128),    # 9
    ("fp32", 1, 16, 151937, 1), ("fp32", 2, 16, 151937, 40), ("fp32", 1, 16, 151937, 128),  # 594
    ("bf16", 1, 32, 151937, 40), ("fp32", 1, 64, 128257, 8), ("bf16", 1, 64, 128257, 128),
]


@pytest.mark.parametrize("kind,groups,beams,vocab,take", CASES)
def test_against_a_sort(cuda, kind, groups, beams, vocab, take):
    print(f"by pieces {kind} groups={groups} beams={beams} vocab={vocab} take={take}", flush=True)
    for seed, spread in ((1, 3.0), (2, 0.05)):
        gen = torch.Generator().manual_seed(seed)
        logits = spread * torch.randn(groups, beams, vocab, generator=gen)
        scores = -4 * torch.rand(groups, beams, generator=gen)
        check(cuda, logits.to(torch.bfloat16) if kind == "bf16" else logits, scores, take)


@pytest.mark.parametrize("kind,beams,vocab,take", [("fp32", 600, 3600, 40), ("bf16", 1024, 4100, 128), ("fp32", 1024, 2100, 1)])
def test_equal_values(cuda, kind, beams, vocab, take):
    """More equal pieces than there is room for, and equal candidates: the lowest numbers come first."""
    test_beams.test_equal_values(cuda, beams, vocab, take, kind)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_values_that_are_none(cuda, kind):
    """Most beams out, or without a number, and most words masked, in whole pieces too: what is left is all there is."""
    beams, vocab = 1024, 2100 if kind == "fp32" else 4100
    gen = torch.Generator().manual_seed(7)
    logits, scores = torch.randn(4, beams, vocab, generator=gen), -torch.rand(4, beams, generator=gen)
    scores[0, torch.randperm(beams, generator=gen)[5:]] = -float("inf")
    logits[1, ::2, 17], logits[1, 1::4, vocab - 1] = float("nan"), float("inf")
    logits[2, :, 3:] = -float("inf")
    logits[2, :1000] = -float("inf")   # 72 candidates
    logits[3, :, :vocab - 4] = -float("inf")
    scores[3, 10:] = float("nan")      # 40, in the last chunk
    for take in (1, 128):
        check(cuda, logits.to(torch.bfloat16) if kind == "bf16" else logits, scores, take)
