"""An axis of one has no stride: what a tensor says of it is not looked at (GPU)."""

import pytest
import torch

import w4a16
from test_kv_cache import filled, make_batch

pytestmark = pytest.mark.gpu


def restrided(x, axis, stride):
    """x with another stride on an axis of one."""
    strides = list(x.stride())
    strides[axis] = stride
    return x.as_strided(x.shape, strides)


@pytest.mark.parametrize("stride", [0, 1, 3, 8, 12345, (1 << 61) + 4])
@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
def test_one_row(cuda, fmt, stride):
    heads, q_heads, dim, page, pages = 2, 6, 64, 16, 8
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, n, dim, generator=gen).to(torch.bfloat16).to(cuda) for n in (q_heads, heads, heads))
    batch, _ = make_batch([100], [1], page, pages, cuda)
    caches = [filled(pages, page, heads, dim, fmt, cuda, seed=6) for _ in range(2)]
    caches[0].write(k, v, batch)
    want = w4a16.paged_attention(q, caches[0], batch)
    caches[1].write(restrided(k, 0, stride), restrided(v, 0, stride), batch)
    out = torch.zeros_like(want)
    w4a16.paged_attention(restrided(q, 0, stride), caches[1], batch, out=restrided(out, 0, stride))
    assert torch.equal(out, want)
    inplace = restrided(q.clone(), 0, stride)
    assert torch.equal(w4a16.paged_attention(inplace, caches[1], batch, out=inplace), want)
    # heads still have one
    with pytest.raises(w4a16.W4A16Error, match="strides"):
        w4a16.paged_attention(q.new_zeros(q_heads * (dim + 4)).as_strided(q.shape, (stride, dim + 4, 1)), caches[1], batch)


@pytest.mark.parametrize("stride", [0, 1, 3, 8, 12345, (1 << 61) + 4])
def test_one_head(cuda, stride):
    dim, page, pages, rows = 128, 16, 20, 40
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(rows, 1, dim, generator=gen).to(torch.bfloat16).to(cuda) for _ in range(3))
    batch, _ = make_batch([200], [rows], page, pages, cuda)
    caches = [filled(pages, page, 1, dim, "int8", cuda, seed=6) for _ in range(2)]
    caches[0].write(k, v, batch)
    want = w4a16.paged_attention(q, caches[0], batch)
    caches[1].write(restrided(k, 1, stride), restrided(v, 1, stride), batch)
    out = torch.zeros_like(want)
    w4a16.paged_attention(restrided(q, 1, stride), caches[1], batch, out=restrided(out, 1, stride))
    assert torch.equal(out, want)
    with pytest.raises(w4a16.W4A16Error, match="strides"):
        w4a16.paged_attention(q.new_zeros(rows * (dim + 4)).as_strided(q.shape, (dim + 4, stride, 1)), caches[1], batch)
