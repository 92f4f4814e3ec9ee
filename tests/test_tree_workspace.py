"""The workspace of attention of drafted trees: places for the parts of what is cut, which are no more however many sequences there are. On the
CPU its bytes; on the GPU batches of which little is cut, in a workspace of exactly those bytes, against FP64."""

import ctypes

import pytest
import torch

import kv_check
import test_tree_attention as short
import tree_oracle
import w4a16
from test_kv_cache import filled, make_batch
from test_kv_refusals import batch, cache
from test_paged_attention import whole

GUARD = 1 << 16


def asked(c, b, q_heads):
    size = ctypes.c_size_t(0)
    assert w4a16.lib.w4a16_paged_tree_attention_workspace(ctypes.byref(c), ctypes.byref(b), q_heads, ctypes.byref(size)) == 0
    return size.value


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("nodes,q_heads,heads", [(256, 128, 8), (256, 32, 8), (60, 8, 8), (8, 32, 8), (1, 16, 16)])
def test_bytes(nodes, q_heads, heads, dim, fmt):
    """At most two places for each of the blocks that 256 CUs hold at once, of as many rows as a tile has: up to 4 blocks a CU and 32
    rows where no sequence has more rows, else 3 (2 above 64 values) and 128; both where the batch does not say."""
    scales = dict(k_scale=1 << 40, v_scale=1 << 41) if fmt else {}
    c = cache(format=fmt, head_dim=dim, kv_heads=heads, page_size=64, num_pages=1 << 16, **scales)
    place = 2 * 256 * (dim + 2) * 4
    few, many = place * 4 * 32, place * (3 if dim == 64 else 2) * 128
    for seqs in (1, 64, 1000, 20000):
        for columns, max_new in ((8, nodes), (64, nodes), (8192, 0)):
            need = asked(c, batch(seqs=seqs, rows=seqs * nodes, table_pages=columns, table_stride=columns, max_new=max_new), q_heads)
            most = few + many if max_new == 0 else few if nodes * q_heads // heads <= 32 else many
            assert need <= most, (seqs, columns, need, most)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("count,news,q_heads,heads,dim,longest", [
    (300, 36, 4, 4, 64, 3000),   # 1200 pairs of tiles of 128 rows, four of them cut
    (70, 40, 8, 8, 256, 2100),   # 560
    (200, 3, 32, 8, 64, 9000),   # 1600 of 16 rows, eight cut
    (200, 5, 16, 4, 128, 9000),  # 800 of 32
])
def test_little_is_cut(cuda, count, news, q_heads, heads, dim, longest, fmt):
    print(f"little is cut: {fmt} {count} x {news} heads={q_heads}/{heads} dim={dim}", flush=True)
    kv_lens = [news + 4 + i % 9 for i in range(count)]
    kv_lens[count - 3], kv_lens[7] = longest, longest // 3
    page, rows = 16, [news] * count
    pages = sum(-(-n // page) for n in kv_lens)
    of = filled(pages, page, heads, dim, fmt, cuda, seed=dim)
    q = (2 * torch.randn(sum(rows), q_heads, dim, generator=torch.Generator().manual_seed(q_heads))).to(torch.bfloat16)
    held, table = make_batch(kv_lens, rows, page, pages, cuda, max_new=news, max_kv=longest)
    parents = short.random_parents(count, news, news, "random")
    tree = w4a16.KvTree(parents.to(cuda), held)
    need = asked(of._c, held._c, q_heads)
    assert need > 0
    space = torch.full((need + GUARD,), 171, dtype=torch.uint8, device=cuda)
    out, lse = w4a16.paged_attention(q.to(cuda), of, held, return_lse=True, tree=tree, workspace=space[:need])
    assert (space[need:] == 171).all()
    (seen, positions), sizes = short.plan_of(parents, None, kv_lens, rows)
    k, v, there = whole(of, table, kv_lens, page, pages)
    seen_by = tree_oracle.visible(seen, positions, sizes, kv_lens, rows, news, 0)
    tree_oracle.check(out, lse, tree_oracle.attention(q, k, v, there, seen_by, dim**-0.5, kv_check.sizes(of, table, kv_lens, page, pages)))


@pytest.mark.gpu
@pytest.mark.parametrize("news,q_heads", [(40, 8), (4, 8)])
def test_sequences_that_overlap(cuda, news, q_heads):
    """Sequences that share rows, far more than rows can have: whatever they give, nothing is stored behind the workspace."""
    count, page, heads, dim = 401, 16, 4, 64
    starts = torch.tensor([news * (i % 2) for i in range(count + 1)], dtype=torch.int32, device=cuda)
    lens = torch.full((count,), 900, dtype=torch.int32, device=cuda)
    table = torch.arange(60, dtype=torch.int32, device=cuda).expand(count, 60).contiguous()
    held = w4a16.KvBatch(table, lens, starts, news)
    of = filled(60, page, heads, dim, "fp8", cuda, seed=1)
    tree = w4a16.KvTree(short.random_parents(count, news, 1, "chain").to(cuda), held)
    q = torch.randn(news, q_heads, dim, device=cuda).to(torch.bfloat16)
    need = asked(of._c, held._c, q_heads)
    space = torch.full((need + GUARD,), 171, dtype=torch.uint8, device=cuda)
    out = w4a16.paged_attention(q, of, held, tree=tree, workspace=space[:need])
    torch.cuda.synchronize()
    assert (space[need:] == 171).all() and out.shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
@pytest.mark.parametrize("news", [2, 33])
def test_very_many_sequences(cuda, news, fmt):
    """More than 65536 pairs, and one long sequence that is cut all the same: it, and some of the others, against FP64."""
    print(f"very many: {fmt} {news}", flush=True)
    count, page, heads, q_heads, dim, longest, held_pages = 8300, 16, 8, 8, 64, 4000, 300
    kv_lens = [news + i % 11 for i in range(count)]
    kv_lens[5000] = longest
    columns = -(-longest // page)
    table = (torch.arange(count)[:, None] * 7 + torch.arange(columns) * 11) % held_pages  # pages are shared: nothing writes
    starts = torch.arange(count + 1, dtype=torch.int32) * news
    batch_of = w4a16.KvBatch(table.to(torch.int32).to(cuda), torch.tensor(kv_lens, dtype=torch.int32, device=cuda), starts.to(cuda), count * news,
                             max_new=news, max_kv=longest)
    of = filled(held_pages, page, heads, dim, fmt, cuda, seed=2)
    parents = short.random_parents(count, news, news, "random")
    tree = w4a16.KvTree(parents.to(cuda), batch_of)
    q = (2 * torch.randn(count * news, q_heads, dim, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16)
    need = asked(of._c, batch_of._c, q_heads)
    space = torch.full((need + GUARD,), 171, dtype=torch.uint8, device=cuda)
    out, lse = w4a16.paged_attention(q.to(cuda), of, batch_of, return_lse=True, tree=tree, workspace=space[:need])
    assert (space[need:] == 171).all()
    some = [0, 1, 63, 64, 4999, 5000, 5001, 8255, 8256, count - 1]
    rows = torch.cat([torch.arange(s * news, (s + 1) * news) for s in some])
    lens, tables = [kv_lens[s] for s in some], [table[s].tolist() for s in some]
    (seen, positions), sizes = short.plan_of(parents[some], None, lens, [news] * len(some))
    k, v, there = whole(of, tables, lens, page, held_pages)
    seen_by = tree_oracle.visible(seen, positions, sizes, lens, [news] * len(some), news, 0)
    tree_oracle.check(out.cpu()[rows], lse.cpu()[rows], tree_oracle.attention(q[rows], k, v, there, seen_by, dim**-0.5,
                                                                              kv_check.sizes(of, tables, lens, page, held_pages)))
