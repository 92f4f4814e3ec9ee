"""The weights of an INT8 or FP8 cache are held in FP16, 2^-11 of each or 2^-31 of the largest times the largest scale, on the
GPU: against FP64 with those bounds, which weights of fewer bits do not keep."""

import pytest
import torch

import kv_oracle
import w4a16
from kv_check import check, sizes
from test_kv_cache import filled, make_batch
from test_paged_attention import whole

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv_lens,news,q_heads,heads,window", [
    ([1], [1], 1, 1, 0), ([37], [1], 4, 2, 0), ([300, 33], [3, 2], 6, 2, 0), ([333, 90], [30, 2], 4, 1, 70), ([1500, 700], [1, 4], 4, 2, 0),
    ([500, 40], [130, 40], 6, 2, 0), ([900], [200], 2, 1, 150), ([3000], [70], 2, 1, 0),
])
def test_against_fp64(cuda, kv_lens, news, q_heads, heads, dim, window, fmt):
    page = 32
    pages = sum(-(-n // page) for n in kv_lens) + 2
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=dim)
    q = (2 * torch.randn(sum(news), q_heads, dim, generator=torch.Generator().manual_seed(q_heads))).to(torch.bfloat16)
    batch, table = make_batch(kv_lens, news, page, pages, cuda)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, window=window, return_lse=True)
    check(out, lse, cache, table, q, kv_lens, news, page, pages, dim**-0.5, window=window)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("news", [12, 25, 90])
def test_values_that_cancel(cuda, fmt, dim, news):
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
    cache = w4a16.KvCache.empty(pages, page, 1, dim, fmt, device=cuda)
    every, table = make_batch([n], [n], page, pages, cuda)
    cache.write(k.to(cuda), v.to(cuda), every)
    batch = w4a16.KvBatch(every.page_table, every.kv_lens, torch.tensor([0, news], dtype=torch.int32, device=cuda), news)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, scale=1.0, causal=False, return_lse=True)
    check(out, lse, cache, table, q, [n], [news], page, pages, 1.0, causal=False)
    keys, vals, there = whole(cache, table, [n], page, pages)
    coded = sizes(cache, table, [n], page, pages)
    want, _, off, _ = kv_oracle.attention(q, keys, vals, there, 1.0, False, 0, [news], [n], coded)
    weight = (q[:, 0].double() @ keys[0][0].T).exp()
    held = (weight * coded[0][1][0]).to(torch.bfloat16).double()
    rough = held @ (vals[0][0] / coded[0][1][0][:, None]) / weight.sum(-1, keepdim=True)
    assert ((rough - want[:, 0]).abs() > off[:, 0]).any()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("news", [3, 60])
@pytest.mark.parametrize("at", [0, 230])
@pytest.mark.parametrize("up", [6, 14, 18, 22, 26, 30, 34, 60])
def test_scales_far_apart(cuda, fmt, dim, news, at, up):
    """A token that weighs nothing, but whose values are 2^up times the others': what it takes from their weights."""
    page, pages, n = 16, 20, 300
    gen = torch.Generator().manual_seed(at)
    k, v = torch.zeros(n, 2, dim), torch.rand(n, 2, dim, generator=gen) * 2 - 1
    k[:, :, 1] = torch.randn(n, 2, generator=gen) / 8
    k[at, :, 0] = -100.0
    v[at] *= 2.0**up
    q = torch.zeros(news, 4, dim)
    q[:, :, :2] = 1.0
    k, v, q = (t.to(torch.bfloat16) for t in (k, v, q))
    cache = w4a16.KvCache.empty(pages, page, 2, dim, fmt, device=cuda)
    every, table = make_batch([n], [n], page, pages, cuda)
    cache.write(k.to(cuda), v.to(cuda), every)
    batch = w4a16.KvBatch(every.page_table, every.kv_lens, torch.tensor([0, news], dtype=torch.int32, device=cuda), news)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, scale=1.0, return_lse=True)
    check(out, lse, cache, table, q, [n], [news], page, pages, 1.0)
