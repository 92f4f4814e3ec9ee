"""Attention of drafted trees over the paged cache on the GPU: what the plan says of every row, and the outputs against FP64 with the
bounds that its roundings allow."""

import pytest
import torch

import kv_check
import tree_oracle
import w4a16
from test_kv_cache import filled, make_batch
from test_paged_attention import whole

pytestmark = pytest.mark.gpu


def random_parents(seqs, nodes, seed, kind):
    gen = torch.Generator().manual_seed(seed)
    at = torch.arange(nodes)
    if kind == "chain":
        return (at - 1).expand(seqs, nodes).to(torch.int32).clone()
    if kind == "star":
        return torch.where(at == 0, -1, 0).expand(seqs, nodes).to(torch.int32).clone()
    if kind == "roots":  # several, and links that are none
        p = torch.randint(-3, nodes + 3, (seqs, nodes), generator=gen)
        return p.to(torch.int32)
    return torch.where(at == 0, -1, (torch.rand(seqs, nodes, generator=gen) * at).long()).to(torch.int32)


def plan_of(parents, sizes, kv_lens, news):
    nodes = parents.shape[1]
    every = [nodes] * len(news) if sizes is None else sizes
    return tree_oracle.plan(parents.tolist(), every, kv_lens, news, nodes), every


@pytest.mark.parametrize("kind", ["chain", "star", "roots", "random"])
@pytest.mark.parametrize("nodes", [1, 2, 31, 64, 65, 128, 200, 256])
def test_plan(cuda, nodes, kind):
    """Whole trees, the last rows of growing ones, rows before the tree, sequences without nodes or with fewer tokens than nodes."""
    kv_lens = [nodes, 700, 300 + nodes, 40, 3, 0, 900]
    news = [nodes, min(5, nodes), nodes + 17, 20, 3, 2, 300]
    parents = random_parents(len(news), nodes, nodes, kind)
    for sizes in (None, [nodes, nodes, nodes, 0, -4, nodes + 9, (nodes + 1) // 2]):
        batch, _ = make_batch(kv_lens, news, 16, 200, cuda)
        tree = w4a16.KvTree(parents.to(cuda), batch, sizes=None if sizes is None else torch.tensor(sizes, dtype=torch.int32, device=cuda))
        (seen, positions), _ = plan_of(parents, sizes, kv_lens, news)
        assert torch.equal(tree.seen.cpu(), tree_oracle.bits(seen, nodes))
        assert tree.positions.tolist() == positions


def test_plan_leaves_other_rows(cuda):
    """Rows before and behind the sequences' stay; sequences whose rows are not the call's are passed over."""
    wide = torch.zeros(3, 9, dtype=torch.int32, device=cuda)
    lens = torch.tensor([9, 9, 9], dtype=torch.int32, device=cuda)
    starts = torch.tensor([2, 6, 30, 32], dtype=torch.int32, device=cuda)
    batch = w4a16.KvBatch(torch.zeros(3, 2, dtype=torch.int32, device=cuda), lens, starts, 12, padded=True)
    tree = w4a16.KvTree(wide[:, :4], batch)
    tree.positions.fill_(-77)
    tree.seen.fill_(5)
    tree.update()
    assert tree.positions.tolist() == [-77] * 2 + [5, 6, 6, 6] + [-77] * 6
    assert tree.seen[:, 0].tolist() == [5] * 2 + [1, 3, 5, 9] + [5] * 6


CASES = [
    # kv_lens, news, sizes, nodes, q heads, kv heads, dim, page, window
    ([1], [1], None, 1, 1, 1, 64, 8, 0),
    ([40], [7], None, 7, 8, 2, 128, 16, 0),
    ([300, 77, 512], [4, 1, 4], [4, 1, 3], 4, 8, 2, 128, 16, 0),             # 16 rows a tile
    ([300, 77, 512], [8, 3, 8], [20, 3, 8], 20, 8, 2, 64, 32, 0),            # growing trees, 32 rows
    ([260, 700], [5, 3], [9, 40], 40, 12, 2, 256, 32, 64),
    ([600, 333, 90], [26, 13, 20], [26, 13, 0], 26, 32, 8, 128, 16, 0),      # 104 rows; an ordinary sequence
    ([600, 333, 290], [64, 64, 40], [64, 60, 64], 64, 6, 2, 64, 64, 0),      # rows before the tree
    ([2049, 1500], [65, 33], None, 65, 16, 2, 256, 64, 0),
    ([1300, 700, 400], [251, 200, 256], [251, 256, 256], 256, 5, 1, 128, 128, 0),
    ([1300, 700, 400], [251, 200, 256], [251, 256, 256], 256, 5, 1, 64, 128, 300),
    ([9, 30, 20], [9, 5, 12], [40, 33, 12], 40, 8, 2, 128, 8, 40),           # fewer tokens than nodes
    ([5000, 3000], [16, 12], None, 16, 8, 2, 128, 64, 0),                    # cut into parts
    ([9000], [40], [64], 64, 8, 1, 64, 64, 1000),
    ([150 + i for i in range(66)], [1 + i % 3 for i in range(66)], [2 + i % 5 for i in range(66)], 6, 2, 1, 64, 32, 0),
    ([4100], [3], [100], 100, 6, 2, 128, 32, 3500),
]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("kv_lens,news,sizes,nodes,q_heads,heads,dim,page,window", CASES)
def test_against_fp64(cuda, kv_lens, news, sizes, nodes, q_heads, heads, dim, page, window, fmt):
    print(f"tree {fmt} lens={kv_lens[:4]} news={news[:4]} nodes={nodes} heads={q_heads}/{heads} dim={dim} page={page} window={window}",
          flush=True)
    pages = sum(-(-n // page) for n in kv_lens) + 2
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=dim + len(kv_lens))
    q = (2 * torch.randn(sum(news), q_heads + 1, dim, generator=torch.Generator().manual_seed(q_heads))).to(torch.bfloat16)
    for kind, hints in (("random", {"max_new": max(news), "max_kv": max(kv_lens)}), ("chain", {}), ("star", {"max_new": 1, "max_kv": 1})):
        batch, table = make_batch(kv_lens, news, page, pages, cuda, **hints)
        parents = random_parents(len(news), nodes, nodes, kind)
        tree = w4a16.KvTree(parents.to(cuda), batch, sizes=None if sizes is None else torch.tensor(sizes, dtype=torch.int32, device=cuda))
        out, lse = w4a16.paged_attention(q.to(cuda)[:, 1:], cache, batch, window=window, return_lse=True, tree=tree)
        (seen, positions), every = plan_of(parents, sizes, kv_lens, news)
        k, v, there = whole(cache, table, kv_lens, page, pages)
        seen_by = tree_oracle.visible(seen, positions, every, kv_lens, news, nodes, window)
        wanted = tree_oracle.attention(q[:, 1:], k, v, there, seen_by, dim**-0.5, kv_check.sizes(cache, table, kv_lens, page, pages))
        tree_oracle.check(out, lse, wanted)
        if kind == "chain" and all(s >= m for s, m in zip(every, news)) and all(n >= s for n, s in zip(kv_lens, every)):
            # a chain is what the ordinary attention sees, cut into other parts: the same bounds hold of both
            plain, plain_lse = w4a16.paged_attention(q.to(cuda)[:, 1:], cache, batch, window=window, return_lse=True)
            tree_oracle.check(plain, plain_lse, wanted)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("nodes", [3, 40, 90])
def test_bits_of_ones_own(cuda, nodes, dim, fmt):
    """Any bits: rows that see nothing of the tree, not even themselves, or nodes behind them (which they do not); positions anywhere,
    as far as a window counts from them. Infinities and NaN at tokens reach the rows that see them and no others."""
    kv_lens, page, window = [300, nodes, 170], 16, 128
    news = [nodes, nodes, nodes // 2 + 1]
    pages, heads, q_heads = sum(-(-n // page) for n in kv_lens) + 2, 2, 6
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=nodes)
    batch, table = make_batch(kv_lens, news, page, pages, cuda)
    tree = w4a16.KvTree(random_parents(3, nodes, 1, "random").to(cuda), batch)
    gen = torch.Generator().manual_seed(nodes)
    picks = torch.rand(sum(news), nodes, generator=gen) < 0.3
    picks[::4] = False
    seen = [torch.nonzero(p)[:, 0].tolist() for p in picks]
    positions = torch.randint(-50, 600, (sum(news),), generator=gen)
    tree.seen.copy_(tree_oracle.bits(seen, nodes))
    tree.positions.copy_(positions)
    # a few tokens of the trees that are no numbers, and one before them
    bad = [(0, 300 - nodes + nodes // 2), (1, nodes // 3), (2, 169), (0, 200)]
    for n, (s, at) in enumerate(bad):
        place = (table[s][at // page], slice(None), at % page)
        if fmt == "bf16":
            cache.v[place][..., n] = float("inf") if n % 2 else float("nan")
        else:
            cache.v_scale[place] = float("inf") if n % 2 else float("nan")
    q = torch.randn(sum(news), q_heads, dim, generator=gen).to(torch.bfloat16)
    seen_by = tree_oracle.visible(seen, positions.tolist(), [nodes] * 3, kv_lens, news, nodes, window)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, window=window, return_lse=True, tree=tree)
    spoiled = torch.zeros(sum(news), dtype=torch.bool)
    starts = [0, news[0], news[0] + news[1]]
    for s, at in bad:
        spoiled[starts[s]:starts[s] + news[s]] |= seen_by[s][:, at]
    assert 0 < spoiled.sum() < spoiled.numel()
    assert torch.equal(torch.isfinite(out.float()).all(-1).all(-1).cpu(), ~spoiled)
    # the others: as if those tokens held zeros, of which they see none
    for s, at in bad:
        place = (table[s][at // page], slice(None), at % page)
        cache.v[place] = 0
        if fmt != "bf16":
            cache.v_scale[place] = 0.0
    k, v, there = whole(cache, table, kv_lens, page, pages)
    wanted = tree_oracle.attention(q, k, v, there, seen_by, dim**-0.5, kv_check.sizes(cache, table, kv_lens, page, pages))
    fine = ~spoiled
    tree_oracle.check(out[fine.to(cuda)], lse[fine.to(cuda)], [t[fine] for t in wanted])


@pytest.mark.parametrize("many", [1, 40])
def test_pages_that_are_none(cuda, many):
    """Pages outside the cache inside the tree and before it, lengths past the table, rows of no sequence left as they were."""
    page, pages, dim, nodes = 8, 9, 64, 5 * many
    table = [[3, -5, 1, 1 << 20], [0, 8, 2, 4], [5, 6, 7, 3]]
    kv_lens, news = [30, 32, 40], [2 * many, 3, 3 * many]
    starts = [2, 2 + 2 * many, 5 + 2 * many, 5 + 5 * many]
    rows = starts[-1] + 3
    batch = w4a16.KvBatch(torch.tensor(table, dtype=torch.int32, device=cuda), torch.tensor(kv_lens, dtype=torch.int32, device=cuda),
                          torch.tensor(starts, dtype=torch.int32, device=cuda), rows, padded=True)
    cache = filled(pages, page, 1, dim, "fp8", cuda, seed=4)
    parents = random_parents(3, nodes, 3, "random")
    tree = w4a16.KvTree(parents.to(cuda), batch)
    q = torch.randn(rows, 3, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    out = torch.full((rows, 3, dim), 9.0, dtype=torch.bfloat16, device=cuda)
    _, lse = w4a16.paged_attention(q.to(cuda), cache, batch, out=out, return_lse=True, tree=tree)
    (seen, positions), every = plan_of(parents, None, kv_lens, news)
    k, v, there = whole(cache, table, kv_lens, page, pages)
    seen_by = tree_oracle.visible(seen, positions, every, kv_lens, news, nodes, 0)
    inner = slice(2, rows - 3)
    tree_oracle.check(out[inner], lse[inner], tree_oracle.attention(q[inner], k, v, there, seen_by, dim**-0.5,
                                                                    kv_check.sizes(cache, table, kv_lens, page, pages)))
    for outer in (slice(0, 2), slice(rows - 3, rows)):
        assert (out[outer] == 9).all() and (lse[outer] == float("-inf")).all()


def test_captured(cuda):
    """A step's plan and attention in a graph, replayed with other lengths, links and sizes, eager work between; two layers of it."""
    kv_lens, news, page, pages = [900, 400, 130], [20, 20, 20], 16, 100
    batch, _ = make_batch(kv_lens, news, page, pages, cuda, max_new=20, max_kv=1000)
    caches = [filled(pages, page, 2, 128, "int8", cuda, seed=n) for n in range(2)]
    q = torch.randn(60, 8, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda)
    parents, sizes = random_parents(3, 33, 1, "random").to(cuda), torch.tensor([33, 20, 0], dtype=torch.int32, device=cuda)
    tree = w4a16.KvTree(parents, batch, sizes=sizes)

    def step():
        tree.update()
        return [w4a16.paged_attention(q, c, batch, return_lse=True, tree=tree) for c in caches]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(4):
        parents.copy_(random_parents(3, 33, 9 + n, ("random", "star", "chain", "roots")[n]))
        sizes.copy_(torch.tensor([20 + n, 33 - n, 5 * n], dtype=torch.int32))
        batch.kv_lens.copy_(torch.tensor([900 - 50 * n, 300 + n, 100 + n], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(got, step()):
            assert torch.equal(a, c) and torch.equal(b, d)


def test_two_streams(cuda):
    """Two calls at once, each with a workspace of its own."""
    kv_lens, news, page, pages = [3000, 2900], [9, 7], 16, 400
    cache = filled(pages, page, 2, 128, "bf16", cuda, seed=3)
    batch, _ = make_batch(kv_lens, news, page, pages, cuda)
    q = torch.randn(16, 8, 128, device=cuda).to(torch.bfloat16)
    tree = w4a16.KvTree(random_parents(2, 12, 1, "random").to(cuda), batch)
    want = w4a16.paged_attention(q, cache, batch, tree=tree)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[w4a16.paged_attention(q, cache, batch, tree=tree, stream=s) for s in streams] for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for pair in outs for o in pair)
