"""The paged cache on the GPU: what a write leaves (bit for bit the definition's, and nothing else touched), and what a
read gives back."""

import numpy as np
import pytest
import torch

import kv_oracle
import w4a16

pytestmark = pytest.mark.gpu


def make_batch(kv_lens, news, page, pages, cuda, seed=0, rows=None, **more):
    """A table of distinct pages in no order, and the batch over it."""
    counts = [max(1, -(-n // page)) for n in kv_lens]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    assert sum(counts) <= pages
    table = [[order.pop() for _ in range(c)] + [0] * (max(counts) - c) for c in counts]
    starts = np.concatenate([[0], np.cumsum(news)]).tolist()
    used = [row[:c] for row, c in zip(table, counts)]
    batch = w4a16.KvBatch(torch.tensor(table, dtype=torch.int32, device=cuda), torch.tensor(kv_lens, dtype=torch.int32, device=cuda),
                          torch.tensor(starts, dtype=torch.int32, device=cuda), starts[-1] if rows is None else rows, **more)
    return batch, used


def filled(pages, page, heads, dim, fmt, cuda, seed):
    """A cache that holds random codes and scales everywhere."""
    gen = torch.Generator().manual_seed(seed)
    cache = w4a16.KvCache.empty(pages, page, heads, dim, fmt, device=cuda)
    for name in ("k", "v"):
        codes, scales = kv_oracle.quantise(torch.randn(pages, heads, page, dim, generator=gen).to(torch.bfloat16), fmt)
        getattr(cache, name).view(torch.uint8).copy_(codes.view(torch.uint8))
        if scales is not None:
            getattr(cache, name + "_scale").copy_(scales)
    return cache


def held(cache, name):
    t, s = getattr(cache, name).cpu(), getattr(cache, name + "_scale")
    return t, None if s is None else s.cpu()


def awkward(x):
    """Rows of zeros, of tiny and of huge values, with an infinity and with a NaN, where there are so many."""
    flat = x.view(-1, x.shape[-1])
    for i, row in enumerate(flat[::5]):
        kind = i % 6
        if kind == 0:
            row.zero_()
        elif kind == 1:
            row.mul_(2.0**-125)  # under the least that is held
        elif kind == 2:
            row[3] = float("inf")
        elif kind == 3:
            row[row.numel() - 1] = float("nan")
        elif kind == 4:
            row.fill_(3.3e38)
        else:
            row.mul_(2.0**-110)
    return x


CASES = [
    # kv_lens, news, heads, dim, page
    ([1], [1], 1, 64, 8),
    ([9, 8, 1], [1, 8, 1], 3, 64, 8),
    ([100, 7, 33], [37, 7, 1], 8, 128, 16),
    ([130], [129], 5, 256, 64),
    ([300, 256], [44, 256], 2, 128, 256),
    ([70] * 70, [1] * 70, 2, 64, 32),  # more sequences than a wave has lanes
]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("kv_lens,news,heads,dim,page", CASES)
def test_write_and_read(cuda, kv_lens, news, heads, dim, page, fmt):
    print(f"kv {fmt} lens={kv_lens[:4]} news={news[:4]} heads={heads} dim={dim} page={page}", flush=True)
    pages = sum(-(-n // page) for n in kv_lens) + 3
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=dim + page)
    batch, table = make_batch(kv_lens, news, page, pages, cuda)
    rows = sum(news)
    # keys and values side by side in the rows of a wider tensor
    fused = awkward(torch.randn(rows, 3 * heads, dim, generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16))
    k, v = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    dev = fused.to(cuda)
    want = {}
    for name, x in (("k", k), ("v", v)):
        codes, scales = held(cache, name)
        new, new_scales = kv_oracle.quantise(x.contiguous(), fmt)
        for i, (_, at, inside) in enumerate(kv_oracle.places(table, kv_lens, news, page, pages)):
            codes.view(torch.uint8)[at, :, inside] = new[i].view(torch.uint8)
            if scales is not None:
                scales[at, :, inside] = new_scales[i]
        want[name] = codes, scales
    cache.write(dev[:, heads:2 * heads], dev[:, 2 * heads:], batch)
    for name in ("k", "v"):
        codes, scales = held(cache, name)
        assert torch.equal(codes.view(torch.uint8), want[name][0].view(torch.uint8)), name
        if scales is not None:
            assert torch.equal(scales.view(torch.int32).abs() > 0x7F800000, want[name][1].view(torch.int32).abs() > 0x7F800000)
            assert torch.equal(scales.nan_to_num(-1), want[name][1].nan_to_num(-1)), name
    # all of every sequence back: the product of code and scale, rounded once
    whole, _ = make_batch(kv_lens, kv_lens, page, pages, cuda)
    whole = w4a16.KvBatch(batch.page_table, batch.kv_lens, whole.starts, sum(kv_lens))
    got = whole and cache.read(whole)
    for name, x in zip(("k", "v"), got):
        codes, scales = want[name]
        rows_of = torch.stack([codes[at, :, inside].float() if scales is None else codes[at, :, inside].float() * scales[at, :, inside][:, None]
                               for _, at, inside in kv_oracle.places(table, kv_lens, kv_lens, page, pages)])
        rounded = rows_of.to(torch.bfloat16)
        assert torch.equal(x.cpu().isnan(), rounded.isnan())
        assert torch.equal(x.cpu().nan_to_num(0, 1e30, -1e30), rounded.nan_to_num(0, 1e30, -1e30)), name


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
def test_rows_without_a_place(cuda, fmt):
    """Positions before the first token or past the table, pages that are none, rows before and behind the sequences':
    not written; read as zeros where they are a sequence's, left as they were where they are not."""
    page, heads, dim, pages = 8, 2, 64, 6
    table = torch.tensor([[2, -1, 4], [6, 1, 1 << 30], [3, 5, 0]], dtype=torch.int32, device=cuda)
    kv_lens, news = [20, 10, 26], [18, 12, 4]
    starts = torch.tensor([2, 20, 32, 36], dtype=torch.int32, device=cuda)
    batch = w4a16.KvBatch(table, torch.tensor(kv_lens, dtype=torch.int32, device=cuda), starts, 40, padded=True)
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=3)
    before = {name: held(cache, name) for name in ("k", "v")}
    x = torch.randn(40, heads, dim, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    cache.write(x.to(cuda), (x * 2).to(cuda), batch)
    where = kv_oracle.places(table.tolist(), kv_lens, news, page, pages)
    assert sum(at < 0 for _, at, _ in where) > 12
    out = tuple(torch.full((40, heads, dim), 7.0, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    cache.read(batch, out=out)
    fresh = cache.read(batch)
    for name, rows, got, new in (("k", x, out[0].cpu(), fresh[0].cpu()), ("v", x * 2, out[1].cpu(), fresh[1].cpu())):
        codes, scales = before[name]
        n_codes, n_scales = kv_oracle.quantise(rows, fmt)
        for i, (_, at, inside) in enumerate(where):
            if at < 0:
                assert (got[2 + i] == 0).all()
                continue
            codes.view(torch.uint8)[at, :, inside] = n_codes[2 + i].view(torch.uint8)
            if scales is not None:
                scales[at, :, inside] = n_scales[2 + i]
            value = n_codes[2 + i].float() if scales is None else n_codes[2 + i].float() * n_scales[2 + i][:, None]
            assert torch.equal(got[2 + i], value.to(torch.bfloat16))
        now = held(cache, name)
        assert torch.equal(now[0].view(torch.uint8), codes.view(torch.uint8))
        assert scales is None or torch.equal(now[1], scales)
        assert (got[:2] == 7).all() and (got[36:] == 7).all()
        assert (new[:2] == 0).all() and (new[36:] == 0).all() and torch.equal(new[2:36], got[2:36])


def test_far_offsets(cuda):
    """Pages past 2^32 bytes (and values) of a cache."""
    page, heads, dim = 256, 8, 256
    pages = (1 << 32) // (page * heads * dim) + 20
    cache = w4a16.KvCache.empty(pages, page, heads, dim, "fp8", device=cuda)
    table = torch.tensor([[pages - 1, 0], [pages - 3, pages - 2]], dtype=torch.int32, device=cuda)
    batch = w4a16.KvBatch(table, torch.tensor([200, 300], dtype=torch.int32, device=cuda),
                          torch.tensor([0, 200, 500], dtype=torch.int32, device=cuda), 500)
    x = torch.randn(500, heads, dim, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(torch.bfloat16)
    cache.write(x, x.flip(0), batch)
    k, v = cache.read(batch)
    for got, rows in ((k, x), (v, x.flip(0))):
        codes, scales = kv_oracle.quantise(rows.cpu(), "fp8")
        assert torch.equal(got.cpu(), (codes.float() * scales[..., None]).to(torch.bfloat16))
    q = torch.randn(500, 16, dim, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda).to(torch.bfloat16)
    out = w4a16.paged_attention(q, cache, batch)
    small = w4a16.KvCache.empty(3, page, heads, dim, "fp8", device=cuda)
    near = w4a16.KvBatch(torch.tensor([[2, 0], [0, 1]], dtype=torch.int32, device=cuda), batch.kv_lens, batch.starts, 500)
    small.write(x, x.flip(0), near)
    assert torch.equal(out, w4a16.paged_attention(q, small, near))
