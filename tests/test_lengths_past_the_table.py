"""Sequences whose kv_lens pass what the table holds, on the GPU: their rows stand where kv_lens puts them, in the write as in
the attention, and only the keys end with the table."""

import pytest
import torch

import kv_oracle
import w4a16
from test_kv_cache import filled
from kv_check import check

pytestmark = pytest.mark.gpu

FAR = (1 << 31) - 1  # the largest kv_lens

CASES = [
    # kv_lens, table pages, news, q heads, kv heads, dim, page, windows
    ([40, 33, 31, FAR], 4, [3, 1, 2, 4], 3, 1, 64, 8, (0, 1, 12, 40)),
    ([30, 45, 24], 3, [3, 9, 1], 4, 2, 128, 8, (0, 10, 16)),           # a table that ends inside 32 tokens
    ([50, 33], 2, [45, 2], 2, 2, 256, 16, (0, 7, 20)),                 # rows before the first token too
    ([1100, 2600, 700], 32, [5, 1, 2], 6, 2, 64, 32, (0, 600, 1590)),  # parts and their join
    ([1100, 1500], 16, [3, 2], 4, 1, 256, 64, (0, 500)),
    ([300, 222, 270], 16, [100, 70, 14], 6, 2, 64, 16, (0, 40, 200)),   # the tiled kernel, rows that see nothing beside others
    ([300, 222], 25, [100, 70], 4, 1, 128, 8, (0, 40, 150)),
    ([300, FAR], 4, [70, 60], 3, 1, 256, 64, (0, 80)),
    ([2200, 2000], 64, [150, 90], 4, 1, 128, 32, (0, 1100)),           # its parts
    ([150, 140, 99], 8, [100, 1, 3], 8, 2, 128, 16, (0, 30)),          # both kernels in a call
]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kv_lens,count,news,q_heads,heads,dim,page,windows", CASES)
def test_rows_stand_where_the_lengths_put_them(cuda, kv_lens, count, news, q_heads, heads, dim, page, windows, causal, fmt):
    print(f"past the table: {fmt} lens={kv_lens} pages={count} news={news} dim={dim} page={page} causal={causal}", flush=True)
    pages = count * len(kv_lens) + 1
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(dim)).tolist()
    table = [table[s * count:(s + 1) * count] for s in range(len(kv_lens))]
    starts = [sum(news[:s]) for s in range(len(news) + 1)]
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=dim + page)
    q = torch.randn(sum(news), q_heads, dim, generator=torch.Generator().manual_seed(q_heads)).to(torch.bfloat16)
    dev = [torch.tensor(t, dtype=torch.int32, device=cuda) for t in (table, kv_lens, starts)]
    for window in windows:
        for hints in ({}, {"max_new": max(news), "max_kv": count * page}):
            batch = w4a16.KvBatch(*dev, sum(news), **hints)
            out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, causal=causal, window=window, return_lse=True)
            check(out, lse, cache, table, q, kv_lens, news, page, pages, dim**-0.5, causal=causal, window=window)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("many", [1, 40])
def test_rows_without_keys(cuda, fmt, many):
    """A sequence without tokens, rows before the first token, lengths past the table, pages that are none; rows before
    and behind the sequences' stay as they were."""
    page, pages, dim = 8, 9, 64
    table = [[3, -5, 1, 1 << 20], [0, 8, 2, 4], [5, 6, 7, 3]]
    kv_lens, news = [30, 0, 40], [2 * many, 3, 3 * many]
    starts = [2, 2 + 2 * many, 5 + 2 * many, 5 + 5 * many]
    rows = starts[-1] + 3
    batch = w4a16.KvBatch(*(torch.tensor(t, dtype=torch.int32, device=cuda) for t in (table, kv_lens, starts)), rows, padded=True)
    cache = filled(pages, page, 1, dim, fmt, cuda, seed=4)
    q = torch.randn(rows, 3, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    out = torch.full((rows, 3, dim), 9.0, dtype=torch.bfloat16, device=cuda)
    _, lse = w4a16.paged_attention(q.to(cuda), cache, batch, out=out, return_lse=True)
    inner = slice(2, rows - 3)
    check(out[inner], lse[inner], cache, table, q[inner], kv_lens, news, page, pages, dim**-0.5)
    assert (out[:2] == 9).all() and (out[-3:] == 9).all()


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
@pytest.mark.parametrize("many", [1, 30])
def test_write_and_attention_place_rows_alike(cuda, fmt, many):
    """Twelve tokens of which four have a place: each row sees its own key, at the position that the write gave it."""
    page, heads, dim, news = 8, 1, 64, 12 * many
    room = 32 * many
    table = torch.arange(room // page, dtype=torch.int32, device=cuda)[None]
    lens = room + 8 * many
    batch = w4a16.KvBatch(table, torch.tensor([lens], dtype=torch.int32, device=cuda),
                          torch.tensor([0, news], dtype=torch.int32, device=cuda), news)
    cache = filled(room // page, page, heads, dim, fmt, cuda, seed=5)
    gen = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn(news, n, dim, generator=gen).to(torch.bfloat16) for n in (heads, heads, 2))
    cache.write(k.to(cuda), v.to(cuda), batch)
    # a window of one: the row itself, or nothing
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, window=1, return_lse=True)
    codes, scales = kv_oracle.quantise(v, fmt)
    own = kv_oracle.values(codes, scales).expand(-1, 2, -1)
    there = room - (lens - news)
    assert there == 4 * many and (out[there:] == 0).all() and (lse[there:] == float("-inf")).all()
    # a weight of 1 and an output rounded once
    assert ((out[:there].cpu().double() - own[:there]).abs() <= own[:there].abs() * 2.0**-8 * 1.001).all()
    whole, whole_lse = w4a16.paged_attention(q.to(cuda), cache, batch, return_lse=True)
    check(whole, whole_lse, cache, [list(range(room // page))], q, [lens], [news], page, room // page, dim**-0.5)


@pytest.mark.parametrize("news,q_heads", [(3, 2), (90, 2)])
@pytest.mark.parametrize("lens", [(1 << 30) - 7, 1 << 30, (1 << 30) + 100, FAR])
def test_positions_around_the_last(cuda, news, q_heads, lens):
    """Tables of more than 2^30 tokens (one page again and again): the last that are there, and lengths behind them."""
    page, dim, window, last = 65536, 64, 150, 1 << 30
    cache = w4a16.KvCache.empty(1, page, 1, dim, "bf16", device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(2)
    cache.k.normal_(generator=gen)
    cache.v.normal_(generator=gen)
    table = torch.zeros(1, (last >> 16) + 3, dtype=torch.int32, device=cuda)
    batch = w4a16.KvBatch(table, torch.tensor([lens], dtype=torch.int32, device=cuda),
                          torch.tensor([0, news], dtype=torch.int32, device=cuda), news)
    q = torch.randn(news, q_heads, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, window=window, return_lse=True)
    # the same from a place near the end on
    first = min(lens, last) - 400
    at = torch.arange(first, min(lens, last)) % page
    k, v = (t.cpu()[0, :, at].double() for t in (cache.k, cache.v))
    there = torch.ones(len(at), dtype=torch.bool)
    want, want_lse, off, lse_off = kv_oracle.attention(q, [k], [v], [there], dim**-0.5, True, window, [news], [lens - first])
    empty = want_lse == float("-inf")
    assert torch.equal(lse.cpu() == float("-inf"), empty) and (out.cpu()[empty] == 0).all()
    assert ((out.cpu().double() - want).abs() <= off).all()
    assert ((lse.cpu().double() - want_lse).abs() <= lse_off)[~empty].all()
