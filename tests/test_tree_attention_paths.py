"""Attention of drafted trees on the GPU, by the paths that a plan may take: the same sizes as test_tree_attention's under a bound of the lengths
that calls for tiles of 128 rows, sequences of few and of many rows in one call, more than 64 sequences, offsets past 32 bits, keys that are
no numbers."""

import pytest
import torch

import kv_check
import test_tree_attention as short
import tree_oracle
import w4a16
from test_kv_cache import filled, make_batch
from test_paged_attention import whole

pytestmark = pytest.mark.gpu


@pytest.fixture
def long_bound(monkeypatch):
    """Batches that may have 2^20 tokens a sequence and any number of new ones, by their bounds."""
    of = w4a16.KvBatch
    monkeypatch.setattr(w4a16, "KvBatch", lambda *a, **more: of(*a, **{**more, "max_kv": 1 << 20, "max_new": 0}))


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("case", short.CASES)
def test_wide_tiles(cuda, long_bound, case, fmt):
    short.test_against_fp64(cuda, *case, fmt)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("nodes", [40, 90])
def test_bits_of_ones_own_in_wide_tiles(cuda, long_bound, nodes, dim, fmt):
    short.test_bits_of_ones_own(cuda, nodes, dim, fmt)


def test_pages_that_are_none_in_wide_tiles(cuda, long_bound):
    short.test_pages_that_are_none(cuda, 40)


def test_captured_in_wide_tiles(cuda, long_bound):
    short.test_captured(cuda)


def check(cuda, kv_lens, news, nodes, q_heads, heads, dim, page, fmt, window=0, **hints):
    pages = sum(-(-n // page) for n in kv_lens) + 2
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=dim)
    q = (2 * torch.randn(sum(news), q_heads, dim, generator=torch.Generator().manual_seed(q_heads))).to(torch.bfloat16)
    batch, table = make_batch(kv_lens, news, page, pages, cuda, **hints)
    parents = short.random_parents(len(news), nodes, nodes, "random")
    sizes = [min(nodes, m + 2) for m in news]
    tree = w4a16.KvTree(parents.to(cuda), batch, sizes=torch.tensor(sizes, dtype=torch.int32, device=cuda))
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, window=window, return_lse=True, tree=tree)
    (seen, positions), _ = short.plan_of(parents, sizes, kv_lens, news)
    k, v, there = whole(cache, table, kv_lens, page, pages)
    seen_by = tree_oracle.visible(seen, positions, sizes, kv_lens, news, nodes, window)
    tree_oracle.check(out, lse, tree_oracle.attention(q, k, v, there, seen_by, dim**-0.5, kv_check.sizes(cache, table, kv_lens, page, pages)))


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_few_and_many_rows(cuda, dim, fmt):
    """Twelve sequences, two of them with trees of more rows than a narrow tile: two launches."""
    kv_lens = [2000 + 97 * i for i in range(12)]
    check(cuda, kv_lens, [1, 3, 40, 2, 1, 4, 2, 1, 33, 2, 1, 1], 44, 32, 8, dim, 32, fmt)


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
@pytest.mark.parametrize("longest", [40, 700])
def test_many_sequences(cuda, longest, fmt):
    """More than the 64 that are looked at at once, each with more rows than a narrow tile."""
    count = 70
    check(cuda, [longest + 3 * i for i in range(count)], [33 + i % 3 for i in range(count)], 40, 1, 1, 64, 16, fmt, max_kv=1 << 20)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
def test_parts_alike(cuda, fmt):
    """Sequences about as long as each other, in equal parts, and one that is not."""
    check(cuda, [3000, 2950, 2900], [40, 33, 40], 42, 8, 2, 128, 64, fmt, max_kv=1 << 20)
    check(cuda, [3000, 300, 2900], [40, 33, 40], 42, 8, 2, 128, 64, fmt, max_kv=1 << 20)
    check(cuda, [3000, 2950, 2900], [40, 33, 40], 42, 8, 2, 128, 64, fmt, window=700, max_kv=1 << 20)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("bound", [0, 1 << 20])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_keys_that_are_no_numbers(cuda, dim, bound, fmt):
    """At tokens of the tree and before it (behind the window's end): they reach the rows that see them and no others."""
    kv_lens, page, nodes, window, heads = [500, 260], 16, 40, 200, 2
    news = [40, 40]
    pages = sum(-(-n // page) for n in kv_lens) + 2
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=dim)
    batch, table = make_batch(kv_lens, news, page, pages, cuda, max_kv=bound)
    parents = short.random_parents(2, nodes, 5, "random")
    tree = w4a16.KvTree(parents.to(cuda), batch)
    bad = [(0, 480), (0, 262), (1, 239), (1, 21)]
    for n, (s, at) in enumerate(bad):
        place = (table[s][at // page], slice(None), at % page)
        if fmt == "bf16":
            cache.k[place][..., n] = float("nan")
        else:
            cache.k_scale[place] = float("nan")
    q = torch.randn(80, 6, dim, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, window=window, return_lse=True, tree=tree)
    (seen, positions), every = short.plan_of(parents, None, kv_lens, news)
    seen_by = tree_oracle.visible(seen, positions, every, kv_lens, news, nodes, window)
    spoiled = torch.zeros(80, dtype=torch.bool)
    for s, at in bad:
        spoiled[40 * s:40 * s + 40] |= seen_by[s][:, at]
    assert 0 < spoiled.sum() < 80
    assert torch.equal(out.isnan().all(-1).all(-1).cpu(), spoiled) and torch.equal(out.isfinite().all(-1).all(-1).cpu(), ~spoiled)
    for s, at in bad:
        place = (table[s][at // page], slice(None), at % page)
        cache.k[place] = 0
        if fmt != "bf16":
            cache.k_scale[place] = 0.0
    k, v, there = whole(cache, table, kv_lens, page, pages)
    wanted = tree_oracle.attention(q, k, v, there, seen_by, dim**-0.5, kv_check.sizes(cache, table, kv_lens, page, pages))
    fine = ~spoiled
    tree_oracle.check(out[fine.to(cuda)], lse[fine.to(cuda)], [t[fine] for t in wanted])


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_far_offsets(cuda, fmt, dim):
    """Append, attention of few and of many rows, a kept path and copied tails in pages past 2^32 bytes of a cache, as in near ones."""
    page, heads = 256, 8
    pages = (1 << 32) // (page * heads * dim * (2 if fmt == "bf16" else 1)) + 20
    far = w4a16.KvCache.empty(pages, page, heads, dim, fmt, device=cuda)
    near = w4a16.KvCache.empty(8, page, heads, dim, fmt, device=cuda)
    lens = torch.tensor([700, 300, 700], dtype=torch.int32, device=cuda)
    tables = [[pages - 1, pages - 7, pages - 5], [pages - 3, pages - 2, 0], [pages - 4, pages - 8, pages - 6]], [[0, 1, 2], [3, 4, 0], [5, 6, 7]]
    gen = torch.Generator(device=cuda).manual_seed(1)
    k, v = (torch.randn(1700, heads, dim, generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(1700, 16, dim, generator=gen, device=cuda).to(torch.bfloat16)
    rope = w4a16.Rope.of(dim, device=cuda)
    path = torch.tensor([[0, 2, 5] + [-1] * 37, [3, 4, 9] + [-1] * 37, [-1, 39] + [-1] * 38], dtype=torch.int32, device=cuda)
    source = torch.tensor([2, -1, -1], dtype=torch.int32, device=cuda)
    both = []
    for cache, table in zip((far, near), tables):
        table = torch.tensor(table, dtype=torch.int32, device=cuda)
        every = w4a16.KvBatch(table, lens, torch.tensor([0, 700, 1000, 1700], dtype=torch.int32, device=cuda), 1700)
        got = [cache.append(k, v, every, rope, q=q)]
        for m, bound in ((2, 0), (40, 0), (40, 1 << 20)):
            batch = w4a16.KvBatch(table, lens, torch.arange(4, dtype=torch.int32, device=cuda) * m, 3 * m, max_kv=bound)
            tree = w4a16.KvTree(short.random_parents(3, m, 3, "random").to(cuda), batch)
            got += w4a16.paged_attention(q[:3 * m], cache, batch, return_lse=True, tree=tree)
        cache.keep_path(batch, path)
        got += cache.read(every)
        cache.copy_tails(table, lens, source)
        got += cache.read(every)
        both.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*both))
    assert all(t.isfinite().all() for t in both[0])
    assert not torch.equal(both[0][-4], both[0][-2])
