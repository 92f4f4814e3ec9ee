"""The weights of a BF16 cache's few rows with trees are held in two BF16 parts too, on the GPU: off by 2^-15 + 2^-23, as without trees. Few are
up to 32 rows a key head in each sequence of a call by its bound, and more over few tokens."""

import pytest
import torch

import test_tree_attention as short
import tree_oracle
import w4a16
from test_kv_cache import filled, make_batch
from test_paged_attention import whole

pytestmark = pytest.mark.gpu

HALF = 2.0**-15 + 2.0**-23


def attended(cuda, cache, kv_lens, news, nodes, q, page, pages, scale, kind, window=0, **hints):
    batch, table = make_batch(kv_lens, news, page, pages, cuda, **hints)
    parents = short.random_parents(len(news), nodes, nodes, kind)
    tree = w4a16.KvTree(parents.to(cuda), batch)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, scale=scale, window=window, return_lse=True, tree=tree)
    (seen, positions), sizes = short.plan_of(parents, None, kv_lens, news)
    k, v, there = whole(cache, table, kv_lens, page, pages)
    seen_by = tree_oracle.visible(seen, positions, sizes, kv_lens, news, nodes, window)
    wanted = tree_oracle.attention(q, k, v, there, seen_by, scale, half=HALF)
    tree_oracle.check(out, lse, wanted)
    return k, v, seen_by, wanted


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv_lens,news,nodes,q_heads,heads,window", [
    ([1], [1], 1, 1, 1, 0), ([37], [4], 9, 4, 2, 0), ([300, 33], [3, 2], 20, 8, 2, 0), ([333, 90], [5, 9], 12, 3, 1, 70),
    ([1500, 700], [16, 4], 16, 4, 2, 0), ([2100], [30], 40, 2, 2, 600), ([5000, 41, 40], [1, 4, 2], 6, 32, 8, 0),
    ([300, 70], [64, 51], 64, 2, 1, 0),  # more rows over few tokens
])
def test_against_fp64(cuda, kv_lens, news, nodes, q_heads, heads, window, dim):
    print(f"weights kv_lens={kv_lens} news={news} dim={dim}", flush=True)
    page = 32
    pages = sum(-(-n // page) for n in kv_lens) + 2
    cache = filled(pages, page, heads, dim, "bf16", cuda, seed=dim)
    q = (2 * torch.randn(sum(news), q_heads, dim, generator=torch.Generator().manual_seed(q_heads))).to(torch.bfloat16)
    for hints in ({"max_new": max(news)}, {"max_new": max(news), "max_kv": max(kv_lens)}):
        attended(cuda, cache, kv_lens, news, nodes, q, page, pages, dim**-0.5, "random", window, **hints)


@pytest.mark.parametrize("kind", ["chain", "star"])
@pytest.mark.parametrize("dim,news", [(64, 12), (64, 30), (128, 12), (128, 30), (256, 12), (256, 30), (128, 100)])
def test_values_that_cancel(cuda, dim, news, kind):
    """Values of 1 under one key and of -1 under another, in turn: a row has two weights, whose roundings add up over the
    tokens, and an output so small beside sum p|v| that its own rounding hides nothing of them. BF16 weights, worked out here,
    leave the bounds."""
    page, pages, n = 16, 40, 600
    k, v = torch.zeros(n, 1, dim), torch.ones(n, 1, dim)
    k[1::2, :, 0] = 1.0
    v[1::2] = -1.0
    q = torch.zeros(news, 1, dim)
    q[:, 0, 0] = -(torch.arange(news) + 1) / 64.0
    k, v, q = (t.to(torch.bfloat16) for t in (k, v, q))
    cache = w4a16.KvCache.empty(pages, page, 1, dim, "bf16", device=cuda)
    every, _ = make_batch([n], [n], page, pages, cuda)
    cache.write(k.to(cuda), v.to(cuda), every)
    keys, vals, seen_by, (want, _, off, _) = attended(cuda, cache, [n], [news], news, q, page, pages, 1.0, kind, max_new=news)
    weight = (q[:, 0].double() @ keys[0][0].T).exp() * seen_by[0]
    rough = weight.to(torch.bfloat16).double() @ vals[0][0] / weight.sum(-1, keepdim=True)
    assert ((rough - want[:, 0]).abs() > off[:, 0]).any()
