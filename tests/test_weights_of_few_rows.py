"""The weights of a BF16 cache's few rows are held in two BF16 parts, on the GPU: a part cut to 8 bits and a rest, under 2^-7 of the
weight, rounded to 8 more (half a step, 2^-8), with a last bit of 2^-23 set: off by 2^-15 + 2^-23."""

import math

import pytest
import torch

import kv_oracle
import w4a16
from kv_check import check
from test_kv_cache import filled, make_batch
from test_paged_attention import whole

pytestmark = pytest.mark.gpu

HALF = 2.0**-15 + 2.0**-23


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv_lens,news,q_heads,heads,window", [
    ([1], [1], 1, 1, 0), ([37], [1], 4, 2, 0), ([300, 33], [3, 2], 8, 2, 0), ([333, 90], [5, 2], 3, 1, 70), ([1500, 700], [1, 4], 8, 2, 0),
    ([2100], [16], 2, 2, 600), ([5000, 1, 40], [1, 1, 1], 32, 2, 0),
])
def test_against_fp64(cuda, kv_lens, news, q_heads, heads, dim, window):
    page = 32
    pages = sum(-(-n // page) for n in kv_lens) + 2
    cache = filled(pages, page, heads, dim, "bf16", cuda, seed=dim)
    q = (2 * torch.randn(sum(news), q_heads, dim, generator=torch.Generator().manual_seed(q_heads))).to(torch.bfloat16)
    for hints in ({"max_new": max(news)}, {"max_new": max(news), "max_kv": max(kv_lens)}):
        batch, table = make_batch(kv_lens, news, page, pages, cuda, **hints)
        out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, window=window, return_lse=True)
        check(out, lse, cache, table, q, kv_lens, news, page, pages, dim**-0.5, window=window, half=HALF)


@pytest.mark.parametrize("dim,news", [(64, 12), (64, 30), (128, 12), (128, 30), (256, 12), (256, 16)])
def test_values_that_cancel(cuda, dim, news):
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
    every, table = make_batch([n], [n], page, pages, cuda)
    cache.write(k.to(cuda), v.to(cuda), every)
    batch = w4a16.KvBatch(every.page_table, every.kv_lens, torch.tensor([0, news], dtype=torch.int32, device=cuda), news, max_new=news)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, scale=1.0, causal=False, return_lse=True)
    check(out, lse, cache, table, q, [n], [news], page, pages, 1.0, causal=False, half=HALF)
    keys, vals, there = whole(cache, table, [n], page, pages)
    want, _, off, _ = kv_oracle.attention(q, keys, vals, there, 1.0, False, 0, [news], [n], half=HALF)
    weight = (q[:, 0].double() @ keys[0][0].T).exp()
    rough = weight.to(torch.bfloat16).double() @ vals[0][0] / weight.sum(-1, keepdim=True)
    assert ((rough - want[:, 0]).abs() > off[:, 0]).any()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinities_stay_what_they_are(cuda, dim, bad):
    """An infinity among V's values at tokens that every row sees, that some see, and whose weight is all but none: it is what the
    rows that see it get in that column, and nothing else changes. Of a weight under 2^-100 of the largest a part may be
    zero: the rest can be 2^-23 of it, BF16 ends at 2^-126 without denormals, and so does the exponential (in plain FP32
    weights are zero under 2^-149). Zero times an infinity is NaN: there either will do."""
    news, n = 5, 300
    for at, down in ((20, 0.0), (n - 3, 0.0), (20, 60.0), (n - 2, 60.0)):
        batch, table = make_batch([n], [news], 16, 24, cuda)
        cache = filled(24, 16, 1, dim, "bf16", cuda, seed=2)
        cache.k[:, 0, :, 0] = 0.0
        cache.k[table[0][at // 16], 0, at % 16, 0] = -down
        q = torch.randn(news, 2, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
        q[:, :, 0] = 1.0
        want = w4a16.paged_attention(q, cache, batch, scale=1.0)
        cache.v[table[0][at // 16], 0, at % 16, 5] = bad
        out = w4a16.paged_attention(q, cache, batch, scale=1.0)
        first = max(0, at - (n - news))
        assert torch.equal(out[:first], want[:first])
        got = out[first:, :, 5].cpu()
        keys = whole(cache, table, [n], 16, 24)[0][0][0]
        score = q[first:].cpu().double() @ keys.T
        hidden = torch.arange(n) > (n - news + first + torch.arange(news - first))[:, None, None]
        held = score[..., at] - score.masked_fill(hidden, float("-inf")).amax(-1) > -100 * math.log(2)
        assert (got[held].isnan() if bad != bad else got[held] == bad).all()
        assert (got[~held].isnan() | (got[~held] == bad)).all()
        rest = [d for d in range(dim) if d != 5]
        assert torch.equal(out[first:][:, :, rest], want[first:][:, :, rest])
