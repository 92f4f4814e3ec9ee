"""Appending turned keys and values on the GPU: what the cache holds and the queries that come back, against FP64."""

import numpy as np
import pytest
import torch

import kv_oracle
import rope_oracle
import w4a16
from test_kv_cache import filled, held, make_batch

pytestmark = pytest.mark.gpu


def places_of(kv_lens, news):
    return torch.tensor([n - m + i for n, m in zip(kv_lens, news) for i in range(m)], dtype=torch.int32)


def check_cache(cache, before, at, k, v, positions, inv_freq, interleaved, fmt):
    """The cache's rows at `at` [(sequence, page, place)], and everything else as it was."""
    some = torch.tensor([p >= 0 for _, p, _ in at])
    pages, inside = (torch.tensor([a[i] for a in at if a[1] >= 0]) for i in (1, 2))
    for name, rows in (("k", k), ("v", v)):
        codes, scales = held(cache, name)
        rest, rest_scales = before[name]
        # rows [n, heads, D] of the places that were written; the later wins where a place came twice (it does not here)
        mine = codes.view(torch.uint8).reshape(*codes.shape[:3], -1)[pages, :, inside].view(codes.dtype)
        mine_scales = None if scales is None else scales[pages, :, inside]
        if name == "v":
            want, want_scales = kv_oracle.quantise(rows[some].contiguous(), fmt)
            assert torch.equal(mine.reshape(want.shape).view(torch.uint8), want.view(torch.uint8))
            assert scales is None or torch.equal(mine_scales.nan_to_num(nan=-5.0), want_scales.nan_to_num(nan=-5.0))
        else:
            want, off = rope_oracle.turned(rows[some], positions[some], inv_freq, interleaved)
            rope_oracle.check_held(mine.reshape(want.shape), mine_scales, want, off, fmt)
        after = codes.view(torch.uint8).reshape(*codes.shape[:3], -1).clone()
        was = rest.view(torch.uint8).reshape(*rest.shape[:3], -1)
        after[pages, :, inside] = was[pages, :, inside]
        assert torch.equal(after, was)
        if scales is not None:
            scales = scales.clone()
            scales[pages, :, inside] = rest_scales[pages, :, inside]
            assert torch.equal(scales, rest_scales)


CASES = [
    # kv_lens, news, kv heads, q heads, dim, page, rotary, interleaved
    ([1], [1], 1, 1, 64, 8, 64, False),
    ([9, 8, 1], [1, 8, 1], 3, 6, 64, 8, 16, False),
    ([100, 7, 33], [37, 7, 1], 8, 32, 128, 16, 128, False),
    ([100, 7, 33], [37, 7, 1], 2, 5, 128, 16, 128, True),
    ([130], [129], 5, 5, 256, 64, 64, True),
    ([130, 40], [3, 2], 1, 16, 256, 64, 256, False),
    ([300, 256], [44, 256], 2, 3, 128, 256, 40, False),
    ([70] * 70, [1] * 70, 2, 4, 64, 32, 8, True),
    ([1000], [900], 1, 0, 128, 16, 24, False),
    ([2500, 3000], [2400, 2990], 1, 2, 64, 32, 32, False),   # a wave for all of a row's heads
]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("kv_lens,news,heads,q_heads,dim,page,rotary,interleaved", CASES)
def test_against_fp64(cuda, kv_lens, news, heads, q_heads, dim, page, rotary, interleaved, fmt):
    print(f"append {fmt} lens={kv_lens[:4]} heads={q_heads}/{heads} dim={dim} rotary={rotary} interleaved={interleaved}", flush=True)
    pages = sum(-(-n // page) for n in kv_lens) + 3
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=dim + page)
    batch, table = make_batch(kv_lens, news, page, pages, cuda)
    rope = w4a16.Rope.of(rotary, 10000.0, interleaved, device=cuda)
    gen = torch.Generator().manual_seed(rotary)
    fused = (3 * torch.randn(sum(news), q_heads + 2 * heads, dim, generator=gen)).to(torch.bfloat16)
    q, k, v = fused.split([q_heads, heads, heads], 1)
    for positions in (None, torch.randint(0, 1 << 20, (sum(news),), generator=gen).to(torch.int32)):
        before = {name: held(cache, name) for name in "kv"}
        dev = fused.to(cuda)
        dq, dk, dv = dev.split([q_heads, heads, heads], 1)
        got = cache.append(dk, dv, batch, rope, q=dq if q_heads else None, positions=None if positions is None else positions.to(cuda))
        place = places_of(kv_lens, news) if positions is None else positions
        at = kv_oracle.places(table, kv_lens, news, page, pages)
        check_cache(cache, before, at, k, v, place, rope.inv_freq.cpu(), interleaved, fmt)
        if q_heads:
            want, off = rope_oracle.turned(q, place, rope.inv_freq.cpu(), interleaved)
            rope_oracle.check_held(got.cpu(), None, want, off, "bf16")
            # in place, beside keys and values that stay as they are
            again = cache.append(dk, dv, batch, rope, q=dq, out=dq, positions=None if positions is None else positions.to(cuda))
            assert again is dq and torch.equal(dq, got)
        else:
            assert got is None
        assert torch.equal(dev[:, q_heads:].cpu(), fused[:, q_heads:])


@pytest.mark.parametrize("dim,heads", [(64, 3), (128, 8), (256, 1)])
def test_values_are_written_as_by_write(cuda, dim, heads):
    """V bit for bit what the cache's own write leaves, and K too where the positions are 0: rows of zeros, tiny and huge
    ones, infinities and NaN among them."""
    from test_kv_cache import awkward

    kv_lens, news, page, pages = [40, 61], [31, 61], 16, 9
    batch, _ = make_batch(kv_lens, news, page, pages, cuda)
    gen = torch.Generator().manual_seed(2)
    k, v = (awkward(torch.randn(sum(news), heads, dim, generator=gen).to(torch.bfloat16)).to(cuda) for _ in range(2))
    for fmt in ("bf16", "int8", "fp8"):
        one, two = (filled(pages, page, heads, dim, fmt, cuda, seed=3) for _ in range(2))
        one.write(k, v, batch)
        # at position 0 a turn is x * 1 - y * 0: an infinity makes NaN of its partner
        finite = torch.isfinite(k.float()).all(-1, keepdim=True)
        two.append(k if fmt != "bf16" else torch.where(finite, k, 1.0), v, batch, w4a16.Rope.of(dim // 2, device=cuda),
                   positions=torch.zeros(sum(news), dtype=torch.int32, device=cuda))
        if fmt == "bf16":
            one.write(torch.where(finite, k, 1.0), v, batch)
        for name in "kv":
            (a, s), (b, t) = held(one, name), held(two, name)
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) or torch.equal(a.float(), b.float())
            assert s is None or torch.equal(s.nan_to_num(nan=-5.0), t.nan_to_num(nan=-5.0))


def test_turns_past_fp32(cuda):
    """Finite keys whose turn is not: a row with an infinity (BF16), and one that is no number (8 bits)."""
    k = torch.full((1, 1, 64), 3.0e38).to(torch.bfloat16).to(cuda)
    batch, table = make_batch([1], [1], 8, 3, cuda)
    rope = w4a16.Rope(torch.full((4,), np.pi / 4, dtype=torch.float32, device=cuda), interleaved=True)
    one = torch.ones(1, dtype=torch.int32, device=cuda)
    for fmt in ("bf16", "int8", "fp8"):
        cache = filled(3, 8, 1, 64, fmt, cuda, seed=3)
        cache.append(k, k, batch, rope, positions=one)
        codes, scales = held(cache, "k")
        row = codes[table[0][0], 0, 0].float()
        if fmt == "bf16":
            assert torch.equal(row[1:8:2], torch.full((4,), float("inf"))) and torch.isfinite(row[8:]).all()
        else:
            assert (row == 0).all() and scales[table[0][0], 0, 0].isnan()


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(cuda, interleaved):
    """Positions up to 2^30 and before 0: FP64 angles."""
    positions = torch.tensor([0, 1, -1, 131071, 131072, (1 << 24) + 1, (1 << 30) - 1, -(1 << 30), 999999937], dtype=torch.int32)
    rows = positions.numel()
    batch, _ = make_batch([rows], [rows], 8, 4, cuda)
    cache = filled(4, 8, 1, 128, "bf16", cuda, seed=1)
    rope = w4a16.Rope.of(128, 1e6, interleaved, device=cuda)
    x = torch.randn(rows, 3, 128, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    got = cache.append(x.to(cuda)[:, :1], x.to(cuda)[:, 1:2], batch, rope, q=x.to(cuda), positions=positions.to(cuda))
    want, off = rope_oracle.turned(x, positions, rope.inv_freq.cpu(), interleaved)
    rope_oracle.check_held(got.cpu(), None, want, off, "bf16")


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
def test_rows_without_a_place(cuda, fmt):
    """Pages outside the cache, lengths past the table, rows before the first token: nothing written, queries turned all the same.
    Rows of no sequence: left as they were."""
    page, pages, heads, dim = 8, 9, 2, 64
    table = [[3, -5, 1, 1 << 20], [0, 8, 2, 4], [5, 6, 7, 3]]
    kv_lens, news = [30, 2, 40], [20, 5, 12]
    starts = [2, 22, 27, 39]
    rows = 42
    batch = w4a16.KvBatch(torch.tensor(table, dtype=torch.int32, device=cuda), torch.tensor(kv_lens, dtype=torch.int32, device=cuda),
                          torch.tensor(starts, dtype=torch.int32, device=cuda), rows, padded=True)
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=4)
    before = {name: held(cache, name) for name in "kv"}
    x = torch.randn(rows, 7, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    rope = w4a16.Rope.of(32, device=cuda)
    dev = x.to(cuda)
    out = torch.full((rows, 3, dim), 9.0, dtype=torch.bfloat16, device=cuda)
    got = cache.append(dev[:, 3:5], dev[:, 5:], batch, rope, q=dev[:, :3], out=out)
    assert got is out and (out[:2] == 9).all() and (out[39:] == 9).all()
    place = places_of(kv_lens, news)
    want, off = rope_oracle.turned(x[2:39, :3], place, rope.inv_freq.cpu(), False)
    rope_oracle.check_held(out[2:39].cpu(), None, want, off, "bf16")
    at = kv_oracle.places(table, kv_lens, news, page, pages)
    assert any(p < 0 for _, p, _ in at) and any(p >= 0 for _, p, _ in at)
    check_cache(cache, before, at, x[2:39, 3:5], x[2:39, 5:], place, rope.inv_freq.cpu(), False, fmt)
    fresh = cache.append(dev[:, 3:5], dev[:, 5:], batch, rope, q=dev[:, :3])
    assert (fresh[:2] == 0).all() and (fresh[39:] == 0).all() and torch.equal(fresh[2:39], out[2:39])


def test_captured_and_on_another_stream(cuda):
    """A graph with other lengths, positions and angles of each replay, eager work between; a call on a stream of its own."""
    caches = [filled(40, 16, 2, 128, "fp8", cuda, seed=1) for _ in range(2)]
    batch, _ = make_batch([60, 200], [9, 30], 16, 40, cuda)
    rope = w4a16.Rope.of(128, device=cuda)
    x = torch.randn(39, 8, 128, device=cuda).to(torch.bfloat16)
    positions = torch.zeros(39, dtype=torch.int32, device=cuda)
    call = lambda cache: cache.append(x[:, 4:6], x[:, 6:], batch, rope, q=x[:, :4], positions=positions)  # noqa: E731
    call(caches[0])
    call(caches[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(caches[0])
    for n in range(4):
        x.normal_()
        positions.random_(0, 5000)
        batch.kv_lens.copy_(torch.tensor([40 + n, 180 - 7 * n], dtype=torch.int32))
        rope.inv_freq.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        want = call(caches[1])
        assert torch.equal(got, want)
        for name in ("k", "v", "k_scale", "v_scale"):
            a, b = getattr(caches[0], name), getattr(caches[1], name)
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = caches[0].append(x[:, 4:6], x[:, 6:], batch, rope, q=x[:, :4], positions=positions, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
