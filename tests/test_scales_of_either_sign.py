"""Scales that a caller fills in by itself, on the GPU: of either sign, and infinite ones of either sign."""

import pytest
import torch

import w4a16
from test_kv_cache import filled, make_batch
from kv_check import check

pytestmark = pytest.mark.gpu

NEWS = [[3], [20], [90]]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("news", NEWS)
@pytest.mark.parametrize("up", [0, 12, 40])
def test_signs(cuda, fmt, dim, news, up):
    """Half of the scales are negative, one of them 2^up times the others in size."""
    page, pages, n = 16, 25, 333
    cache = filled(pages, page, 2, dim, fmt, cuda, seed=dim)
    gen = torch.Generator().manual_seed(up)
    for scales in (cache.k_scale, cache.v_scale):
        scales *= torch.where(torch.rand(scales.shape, generator=gen) < 0.5, -1.0, 1.0).to(cuda)
    batch, table = make_batch([n], news, page, pages, cuda)
    t = 50
    cache.v_scale[table[0][t // page], :, t % page] = -(2.0**up) * cache.v_scale.abs().max()
    q = torch.randn(news[0], 4, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, return_lse=True)
    check(out, lse, cache, table, q, [n], news, page, pages, dim**-0.5)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("news,window", [([6], 0), ([6], 20), ([20], 20), ([100], 0), ([100], 20)])
@pytest.mark.parametrize("bad", [float("-inf"), float("inf"), float("nan"), -float("nan")])
def test_no_numbers(cuda, fmt, news, window, dim, bad):
    """A scale that is no number reaches the rows that see its token, whatever its sign."""
    page, pages, n = 32, 8, 170
    batch, table = make_batch([n], news, page, pages, cuda)
    cache = filled(pages, page, 2, dim, fmt, cuda, seed=8)
    q = torch.randn(news[0], 4, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    want = w4a16.paged_attention(q, cache, batch, window=window)
    places = list(range(n - 3, len(table[0]) * page)) + (list(range(0, n - news[0] - window + 1)) if window else [])
    for t in places:
        cache.v_scale[table[0][t // page], :, t % page] = bad
    out = w4a16.paged_attention(q, cache, batch, window=window)
    assert torch.equal(out[:-3], want[:-3])
    assert not out[-3:].isfinite().any()
