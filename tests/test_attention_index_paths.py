"""Attention on the GPU where its counting is longest: more sequences than a wave has lanes whose work is cut, contexts of 100000
tokens, rows of few in pages past 2^32 bytes."""

import pytest
import torch

import w4a16
from kv_check import check
from test_kv_cache import filled, make_batch

pytestmark = pytest.mark.gpu


def attend(cuda, kv_lens, news, q_heads, heads, dim, page, fmt, window=0, **hints):
    pages = sum(-(-n // page) for n in kv_lens) + 1
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=dim + len(kv_lens))
    q = (2 * torch.randn(sum(news), q_heads, dim, generator=torch.Generator().manual_seed(q_heads))).to(torch.bfloat16)
    batch, table = make_batch(kv_lens, news, page, pages, cuda, **hints)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, window=window, return_lse=True)
    check(out, lse, cache, table, q, kv_lens, news, page, pages, dim**-0.5, window=window)


RAGGED = [1500 + 13 * i if i % 9 == 4 else 3 + 37 * i % 300 for i in range(130)]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("seqs,news,q_heads,heads,dim,window", [
    (130, 1, 2, 1, 64, 0), (130, 3, 6, 2, 128, 0), (70, 2, 4, 1, 256, 0), (65, 5, 5, 1, 64, 1200),
    (70, 40, 1, 1, 64, 0), (129, 35, 2, 1, 128, 0), (66, 18, 2, 1, 256, 0), (70, 40, 2, 2, 64, 1100),
])
def test_more_sequences_than_lanes(cuda, seqs, news, q_heads, heads, dim, window, fmt):
    print(f"index paths {fmt} seqs={seqs} news={news} heads={q_heads}/{heads} dim={dim} window={window}", flush=True)
    lens = RAGGED[:seqs]
    attend(cuda, lens, [min(n, news) for n in lens], q_heads, heads, dim, 32, fmt, window)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_more_sequences_than_lanes_of_both_kernels(cuda, fmt):
    """Decoding sequences and chunks by turns, in both halves of the count."""
    lens = RAGGED[:90]
    attend(cuda, lens, [min(n, 50) if i % 4 == 0 else 1 for i, n in enumerate(lens)], 4, 2, 64, 16, fmt, max_new=50, max_kv=max(lens))


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("news,dim", [(1, 64), (5, 128), (1, 256), (40, 64), (30, 128), (20, 256)])
def test_long_contexts(cuda, news, dim, fmt):
    print(f"index paths {fmt} 100003 tokens news={news} dim={dim}", flush=True)
    attend(cuda, [100003], [news], 3, 1, dim, 256, fmt)


@pytest.mark.parametrize("fmt,dim", [("bf16", 256), ("fp8", 128)])
def test_few_rows_at_far_offsets(cuda, fmt, dim):
    """The same rows from pages past 2^32 bytes of a cache as from near ones."""
    page, heads = 256, 8
    pages = (1 << 32) // (page * heads * dim * (2 if fmt == "bf16" else 1)) + 20
    cache = w4a16.KvCache.empty(pages, page, heads, dim, fmt, device=cuda)
    near = w4a16.KvCache.empty(8, page, heads, dim, fmt, device=cuda)
    lens = torch.tensor([700, 300, 1000], dtype=torch.int32, device=cuda)
    # the last sequence ends in the first one's second page; entry by entry the same in both
    far_table = [[pages - 1, pages - 7, pages - 5, 0], [pages - 3, pages - 2, 0, 0], [pages - 4, 1, pages - 6, pages - 7]]
    near_table = [[0, 1, 2, 0], [3, 4, 0, 0], [5, 6, 7, 1]]
    gen = torch.Generator(device=cuda).manual_seed(1)
    k, v = (torch.randn(2000, heads, dim, generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(5, 16, dim, generator=gen, device=cuda).to(torch.bfloat16)
    news = torch.tensor([0, 1, 4, 5], dtype=torch.int32, device=cuda)
    both = []
    for c, table in ((cache, far_table), (near, near_table)):
        table, first = torch.tensor(table, dtype=torch.int32, device=cuda), 0
        for s, n in enumerate(lens.tolist()):  # in turn: two of them write the shared page
            one = w4a16.KvBatch(table[s:s + 1], lens[s:s + 1], torch.tensor([0, n], dtype=torch.int32, device=cuda), n)
            c.write(k[first:first + n], v[first:first + n], one)
            first += n
        both.append(w4a16.paged_attention(q, c, w4a16.KvBatch(table, lens, news, 5, max_new=3), return_lse=True))
    assert torch.equal(both[0][0], both[1][0]) and torch.equal(both[0][1], both[1][1])
    assert both[0][1].isfinite().all()
