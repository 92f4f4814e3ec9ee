"""Attention over the paged cache on the GPU, against FP64 with the bounds that its roundings allow (kv_oracle.py)."""

import pytest
import torch

import kv_oracle
import w4a16
from test_kv_cache import filled, held, make_batch

pytestmark = pytest.mark.gpu


def whole(cache, table, kv_lens, page, pages):
    """(keys, values, whether each token is there) of every sequence, in FP64."""
    k, v, there = [], [], []
    kc, vc = kv_oracle.values(*held(cache, "k")), kv_oracle.values(*held(cache, "v"))
    for row, n in zip(table, kv_lens):
        n = min(n, len(row) * page)
        at = [row[i // page] for i in range(n)]
        ok = torch.tensor([0 <= a < pages for a in at], dtype=torch.bool)
        safe = torch.tensor([a if 0 <= a < pages else 0 for a in at], dtype=torch.long)
        inside = torch.arange(n) % page
        k.append(kc[safe, :, inside].transpose(0, 1) if n else torch.zeros(kc.shape[1], 0, kc.shape[3], dtype=torch.float64))
        v.append(vc[safe, :, inside].transpose(0, 1) if n else torch.zeros(kc.shape[1], 0, kc.shape[3], dtype=torch.float64))
        there.append(ok)
    return k, v, there


def check(out, lse, cache, table, q, kv_lens, news, page, pages, scale, causal=True, window=0):
    k, v, there = whole(cache, table, kv_lens, page, pages)
    want, want_lse, off, lse_off = kv_oracle.attention(q, k, v, there, scale, causal, window, news, kv_lens)
    got, got_lse = out.cpu().double(), lse.cpu().double()
    assert torch.equal(got_lse == float("-inf"), want_lse == float("-inf"))
    empty = want_lse == float("-inf")
    far = ((got - want).abs() / off.clamp(min=1e-300))[~empty]
    lse_far = ((got_lse - want_lse).abs() / lse_off.clamp(min=1e-300))[~empty]
    if far.numel():
        print(f"  of what the roundings allow: out {far.max():.3f}, lse {lse_far.max():.3f}", flush=True)
        assert far.max() <= 1 and lse_far.max() <= 1
    assert (got[empty] == 0).all()


CASES = [
    # kv_lens, news, q heads, kv heads, dim, page, window
    ([1], [1], 1, 1, 64, 8, 0),
    ([37], [1], 8, 2, 128, 16, 0),
    ([1000, 3, 517], [1, 1, 1], 8, 2, 128, 16, 0),
    ([2049], [1], 6, 1, 256, 64, 0),
    ([260, 700], [5, 3], 12, 2, 64, 32, 0),          # verify rows: 30 rows a tile pair
    ([300, 90, 33], [7, 5, 1], 16, 2, 128, 8, 0),     # 56 rows
    ([129], [9], 16, 1, 256, 128, 0),                 # 144 rows
    ([31, 32, 33, 64], [31, 32, 2, 17], 4, 4, 128, 16, 0),
    ([500, 40], [130, 40], 6, 2, 64, 16, 0),
    ([700], [3], 4, 2, 128, 32, 100),
    ([400, 900], [50, 1], 5, 1, 256, 16, 33),
    ([90], [90], 2, 2, 64, 8, 1),                     # a window of the row itself
    ([3000, 800], [1, 1], 32, 2, 128, 256, 0),        # a group of sixteen
    ([150] * 66, [1] * 66, 2, 1, 64, 32, 0),          # more sequences than a wave has lanes
    ([640, 1, 300], [257, 1, 129], 7, 1, 128, 64, 0),
    ([640, 300], [200, 129], 4, 2, 256, 64, 150),
    ([70, 500], [3, 4], 4, 1, 256, 32, 37),           # windows that begin at every place of four tokens
    ([333, 90], [9, 2], 3, 1, 64, 8, 10),
    ([333, 90], [60, 2], 5, 1, 128, 8, 10),
    ([3 + 37 * i % 300 for i in range(50)], [1 + i % 3 for i in range(50)], 528, 16, 64, 32, 0),   # more tiles than
    ([3 + 37 * i % 300 for i in range(50)], [1 + i % 3 for i in range(50)], 528, 16, 64, 32, 70),  # there is room for
    ([500, 40, 700, 16], [16, 9, 16, 16], 8, 2, 64, 16, 0),   # 64 rows
    ([500, 40, 700, 16], [16, 9, 13, 16], 8, 2, 128, 16, 75),
    ([5000, 3000], [16, 12], 8, 2, 128, 64, 0),
    ([4100], [21], 6, 2, 64, 32, 3500),
]


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("kv_lens,news,q_heads,heads,dim,page,window", CASES)
def test_against_fp64(cuda, kv_lens, news, q_heads, heads, dim, page, window, fmt):
    print(f"attention {fmt} lens={kv_lens[:4]} news={news[:4]} heads={q_heads}/{heads} dim={dim} page={page} window={window}", flush=True)
    pages = sum(-(-n // page) for n in kv_lens) + 2
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=dim + len(kv_lens))
    q = (2 * torch.randn(sum(news), q_heads + 1, dim, generator=torch.Generator().manual_seed(q_heads))).to(torch.bfloat16)
    for hints in ({}, {"max_new": max(news), "max_kv": max(kv_lens)}, {"max_new": 1, "max_kv": 1}):
        batch, table = make_batch(kv_lens, news, page, pages, cuda, **hints)
        out, lse = w4a16.paged_attention(q.to(cuda)[:, 1:], cache, batch, window=window, return_lse=True)
        check(out, lse, cache, table, q[:, 1:], kv_lens, news, page, pages, dim**-0.5, window=window)


@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("scale", [0.2, -0.1, 0.0])
@pytest.mark.parametrize("news", [[3, 2], [80, 70]])
def test_every_row_sees_all(cuda, fmt, news, scale, window):
    """causal=False, and a scale of the caller's, of either sign or none."""
    kv_lens, page, pages = [333, 200], 16, 40
    cache = filled(pages, page, 2, 128, fmt, cuda, seed=9)
    batch, table = make_batch(kv_lens, news, page, pages, cuda)
    q = torch.randn(sum(news), 6, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, scale=scale, causal=False, window=window, return_lse=True)
    check(out, lse, cache, table, q, kv_lens, news, page, pages, scale, causal=False, window=window)


def test_sequences_that_decrease_or_overlap(cuda):
    """Starts that no caller should give: every access stays where it belongs, and the sequences that are whole and
    alone are right."""
    page, pages, dim = 8, 300, 64
    cache = filled(pages, page, 2, dim, "fp8", cuda, seed=4)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(0)).to(torch.int32)
    table = order[:4 * 70].reshape(4, 70).to(cuda)
    lens = torch.tensor([550, 560, 40, 555], dtype=torch.int32, device=cuda)
    q = torch.randn(40, 4, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    alone = w4a16.KvBatch(table[:1], lens[:1], torch.tensor([0, 3], dtype=torch.int32, device=cuda), 40, max_new=3, padded=True)
    want = w4a16.paged_attention(q, cache, alone)
    for starts in ([0, 3, 1, 9, 5], [0, 3, 60, 2, 40], [0, 3, -5, 20, 41], [0, 3, 3, 3, 3]):
        batch = w4a16.KvBatch(table, lens, torch.tensor(starts, dtype=torch.int32, device=cuda), 40, max_new=3, padded=True)
        out = w4a16.paged_attention(q, cache, batch)
        if starts[2] >= 3:
            assert torch.equal(out[:2], want[:2])
        cache.write(q[:, :2], q[:, 2:], batch)
        cache.read(batch)
        torch.cuda.synchronize()
        cache = filled(pages, page, 2, dim, "fp8", cuda, seed=4)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("many", [1, 40])
def test_rows_that_see_nothing(cuda, fmt, many):
    """A sequence without tokens, rows before the first token, lengths past the table, pages that are none; rows before
    and behind the sequences' stay as they were."""
    page, pages, dim = 8, 9, 64
    table = [[3, -5, 1, 1 << 20], [0, 8, 2, 4], [5, 6, 7, 3]]
    kv_lens, news = [30, 0, 40], [2 * many, 3, 3 * many]
    lens = [n if n < 32 else 32 for n in kv_lens]
    starts = [2, 2 + 2 * many, 5 + 2 * many, 5 + 5 * many]
    rows = starts[-1] + 3
    batch = w4a16.KvBatch(torch.tensor(table, dtype=torch.int32, device=cuda), torch.tensor(kv_lens, dtype=torch.int32, device=cuda),
                          torch.tensor(starts, dtype=torch.int32, device=cuda), rows, padded=True)
    cache = filled(pages, page, 1, dim, fmt, cuda, seed=4)
    q = torch.randn(rows, 3, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    out = torch.full((rows, 3, dim), 9.0, dtype=torch.bfloat16, device=cuda)
    _, lse = w4a16.paged_attention(q.to(cuda), cache, batch, out=out, return_lse=True)
    inner = slice(2, rows - 3)
    check(out[inner], lse[inner], cache, table, q[inner], lens, news, page, pages, dim**-0.5)
    assert (out[:2] == 9).all() and (out[-3:] == 9).all()


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("news,window", [([6], 0), ([6], 20), ([20], 0), ([20], 20), ([100], 0), ([100], 20)])
def test_nonfinite_values_stay_with_the_rows_that_see_them(cuda, fmt, news, window, dim):
    """Keys and values with infinities and NaN behind the last token, outside the window and at later positions change
    nothing; a row that sees one is not a number where the value is not."""
    page, pages, heads, n = 32, 8, 2, 170
    batch, table = make_batch([n], news, page, pages, cuda)
    clean = filled(pages, page, heads, dim, fmt, cuda, seed=8)
    q = torch.randn(news[0], 4, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    want = w4a16.paged_attention(q, clean, batch, window=window)
    first_bad = n - 3  # the last three tokens
    for t in range(first_bad, len(table[0]) * page):
        at, inside = table[0][t // page], t % page
        if fmt == "bf16":
            clean.k[at, :, inside] = float("nan")
            clean.v[at, :, inside, ::3] = float("inf") if t % 2 else float("nan")
        else:
            clean.k_scale[at, :, inside] = float("nan")
            clean.v_scale[at, :, inside] = float("inf") if t % 2 else float("nan")
    if window:  # and what every row has left behind
        for t in range(0, n - news[0] - window + 1):
            at, inside = table[0][t // page], t % page
            if fmt == "bf16":
                clean.v[at, :, inside] = float("nan")
            else:
                clean.v_scale[at, :, inside] = float("nan")
    out = w4a16.paged_attention(q, clean, batch, window=window)
    assert torch.equal(out[:-3], want[:-3])
    assert out[-3:].isnan().any(-1).all()


def test_an_infinite_value_reaches_its_rows_alone(cuda):
    """One value column of one BF16 token at infinity: the rows that see the token get it there and nowhere else."""
    for news, dim in ((4, 64), (70, 64), (4, 256), (70, 256), (70, 128)):
        batch, table = make_batch([100], [news], 16, 8, cuda)
        cache = filled(8, 16, 1, dim, "bf16", cuda, seed=2)
        q = torch.randn(news, 2, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
        want = w4a16.paged_attention(q, cache, batch)
        cache.v[table[0][98 // 16], 0, 98 % 16, 5] = float("inf")
        out = w4a16.paged_attention(q, cache, batch)
        assert torch.equal(out[:-2], want[:-2])
        assert (out[-2:, :, 5] == float("inf")).all()
        rest = [d for d in range(dim) if d != 5]
        assert torch.equal(out[-2:, :, rest], want[-2:, :, rest])


def test_rows_stay_apart(cuda):
    """A query of NaN spoils its own row."""
    for news in (5, 50):
        batch, _ = make_batch([300], [news], 16, 20, cuda)
        cache = filled(20, 16, 2, 128, "bf16", cuda, seed=2)
        q = torch.randn(news, 4, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
        want, want_lse = w4a16.paged_attention(q, cache, batch, return_lse=True)
        q[1, 2] = float("nan")
        out, lse = w4a16.paged_attention(q, cache, batch, return_lse=True)
        assert out[1, 2].isnan().all() and lse[1, 2].isnan()
        keep = torch.ones(news, 4, dtype=torch.bool, device=cuda)
        keep[1, 2] = False
        assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])


@pytest.mark.parametrize("kv_lens,news", [([900, 50], [1, 1]), ([400, 300], [90, 1])])
def test_layouts_and_aliases(cuda, kv_lens, news):
    """Head-major queries and outputs, the output in place of the queries, and beside them in one tensor: the same bits."""
    heads, q_heads, dim, page, pages = 2, 6, 128, 16, 80
    cache = filled(pages, page, heads, dim, "bf16", cuda, seed=6)
    batch, _ = make_batch(kv_lens, news, page, pages, cuda)
    rows = sum(news)
    q = torch.randn(rows, q_heads, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    want = w4a16.paged_attention(q, cache, batch)
    major = q.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.zeros_like(major.transpose(0, 1)).transpose(0, 1)
    assert torch.equal(w4a16.paged_attention(major, cache, batch, out=out), want)
    both = torch.zeros(rows, 2 * q_heads, dim, dtype=torch.bfloat16, device=cuda)
    both[:, :q_heads] = q
    w4a16.paged_attention(both[:, :q_heads], cache, batch, out=both[:, q_heads:])
    assert torch.equal(both[:, q_heads:], want) and torch.equal(both[:, :q_heads], q)
    w4a16.paged_attention(q, cache, batch, out=q)
    assert torch.equal(q, want)


def test_a_captured_call_reads_the_lengths_of_each_replay(cuda):
    """A step (write, attention, read) in a graph: replayed while the lengths and the table change, with eager work and
    synchronisation between; two graphs with workspaces of their own, replayed on two streams at once."""
    heads, q_heads, dim, page, pages = 2, 8, 128, 16, 200
    q = torch.randn(3, q_heads, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    kv = torch.randn(3, heads, dim, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(cuda)
    sides = []
    for seed, fmt in ((1, "fp8"), (2, "bf16")):
        cache = filled(pages, page, heads, dim, fmt, cuda, seed=seed)
        batch, _ = make_batch([900, 700, 1], [1, 1, 1], page, pages, cuda, seed=seed, max_new=1, max_kv=1000)
        cache.write(kv, kv, batch)
        w4a16.paged_attention(q, cache, batch)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.write(kv, kv, batch)
            out = w4a16.paged_attention(q, cache, batch)
            back = cache.read(batch)
        sides.append((graph, cache, batch, out, back))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        for _, _, batch, _, _ in sides:
            batch.kv_lens += torch.tensor([7, -150, 40 * step], dtype=torch.int32, device=cuda)
        torch.cuda.synchronize()
        for stream, (graph, _, _, _, _) in zip(streams, sides):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, cache, batch, out, back in sides:
            assert torch.equal(w4a16.paged_attention(q, cache, batch), out)
            assert all(torch.equal(a, b) for a, b in zip(cache.read(batch), back))


def test_on_a_stream_of_its_own(cuda):
    heads, q_heads, dim, page, pages = 2, 8, 128, 16, 200
    cache = filled(pages, page, heads, dim, "int8", cuda, seed=1)
    batch, _ = make_batch([900, 700], [3, 1], page, pages, cuda)
    q = torch.randn(4, q_heads, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    want = w4a16.paged_attention(q, cache, batch)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = w4a16.paged_attention(q, cache, batch)
    explicit = torch.empty_like(want)
    w4a16.paged_attention(q, cache, batch, out=explicit, stream=stream,
                          workspace=torch.empty(1 << 24, dtype=torch.uint8, device=cuda))
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(explicit, want)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("news", [[1, 2, 1], [50, 2, 70]])
def test_shared_pages(cuda, fmt, news):
    """Sequences that begin with the same pages, and one that holds a page twice, as against copies of the pages."""
    page, heads, dim = 16, 2, 128
    table = [[3, 1, 4, 5, 9], [3, 1, 4, 2, 6], [3, 3, 7, 8, 0]]
    flat = torch.tensor(table).flatten()
    cache = filled(10, page, heads, dim, fmt, cuda, seed=2)
    apart = w4a16.KvCache.empty(15, page, heads, dim, fmt, device=cuda)
    for name in ("k", "v", "k_scale", "v_scale"):
        if getattr(cache, name) is not None:
            bits = [getattr(c, name).view(torch.int16 if fmt == "bf16" else getattr(c, name).dtype) for c in (apart, cache)]
            bits[0].copy_(bits[1][flat.to(cuda)])
    lens = torch.tensor([78, 70, 80], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, news[0], news[0] + news[1], sum(news)], dtype=torch.int32, device=cuda)
    q = torch.randn(sum(news), 4, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    out = [w4a16.paged_attention(q, c, w4a16.KvBatch(t.to(torch.int32).to(cuda), lens, starts, sum(news)))
           for c, t in ((cache, torch.tensor(table)), (apart, torch.arange(15).reshape(3, 5)))]
    assert torch.equal(out[0], out[1])


@pytest.mark.parametrize("raw", [False, True])
def test_memory_of_a_call_on_another_stream(cuda, raw):
    """What a call allocates for a stream that is not the current one, and lets go of when it returns, is not given to
    the current stream while the call still runs."""
    heads, q_heads, dim, page, pages = 2, 8, 128, 16, 700
    cache = filled(pages, page, heads, dim, "fp8", cuda, seed=1)
    batch, _ = make_batch([5000, 4000], [60, 3], page, pages, cuda, padded=True)
    q = torch.randn(63, q_heads, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    want, want_lse = w4a16.paged_attention(q, cache, batch, return_lse=True)
    want_k, _ = cache.read(batch)
    gen = torch.Generator().manual_seed(5)
    probs = torch.rand(2, 3, 40000, generator=gen).to(cuda)
    ids = torch.randint(0, 40000, (2, 2), generator=gen, dtype=torch.int32).to(cuda)
    uniforms = torch.rand(2, 3, generator=gen).to(cuda)
    want_ids = w4a16.verify_drafts(probs, ids, uniforms)[1]
    stream, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device=cuda)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(20):
            busy @ busy
    where = stream.cuda_stream if raw else stream
    got, lse = w4a16.paged_attention(q, cache, batch, return_lse=True, stream=where)
    got_k, _ = cache.read(batch, stream=where)
    got_ids = w4a16.verify_drafts(probs, ids, uniforms, stream=where)[1]
    others = [torch.full((1 << n,), 77, dtype=torch.uint8, device=cuda) for n in range(9, 28) for _ in range(2)]
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, want_lse) and torch.equal(got_k, want_k) and torch.equal(got_ids, want_ids)
    assert all((t == 77).all() for t in others)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("news", [3, 60])
@pytest.mark.parametrize("at", [0, 100, 230])
def test_scales_far_apart(cuda, fmt, dim, news, at):
    """A token that weighs nothing, but whose values are 2^20 times the others', takes nothing from their weights."""
    page, pages, n = 16, 20, 300
    gen = torch.Generator().manual_seed(at)
    k, v = torch.zeros(n, 2, dim), torch.rand(n, 2, dim, generator=gen) * 2 - 1
    k[:, :, 1] = torch.randn(n, 2, generator=gen) / 8
    k[at, :, 0] = -64.0
    v[at] *= 2.0**20
    q = torch.zeros(news, 4, dim)
    q[:, :, :2] = 1.0
    k, v, q = (t.to(torch.bfloat16) for t in (k, v, q))
    cache = w4a16.KvCache.empty(pages, page, 2, dim, fmt, device=cuda)
    every, table = make_batch([n], [n], page, pages, cuda)
    cache.write(k.to(cuda), v.to(cuda), every)
    batch = w4a16.KvBatch(every.page_table, every.kv_lens, torch.tensor([0, news], dtype=torch.int32, device=cuda), news)
    out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, scale=1.0, return_lse=True)
    check(out, lse, cache, table, q, [n], [news], page, pages, 1.0)


def test_refusals_of_tensors(cuda):
    """FP16 is not BF16, and neither are strided values or other shapes."""
    cache = filled(8, 16, 2, 64, "bf16", cuda, seed=1)
    batch, _ = make_batch([20], [2], 16, 8, cuda)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=cuda)
    for bad in (q.half(), q[:1], q[:, :, :32], q.transpose(1, 2), q.cpu(), q.float()):
        with pytest.raises(w4a16.W4A16Error):
            w4a16.paged_attention(bad, cache, batch)
        with pytest.raises(w4a16.W4A16Error):
            w4a16.paged_attention(q, cache, batch, out=bad)
        with pytest.raises(w4a16.W4A16Error):
            cache.write(bad[:, :2], q[:, :2], batch)
    assert torch.equal(w4a16.paged_attention(q.view(torch.int16), cache, batch), w4a16.paged_attention(q, cache, batch))


def test_a_step_of_speculative_decoding(cuda):
    """The operators as a serving loop uses them: drafted tokens' keys and values appended, attended to, verified, the
    lengths cut back to what was taken, and the next step over the same pages."""
    heads, q_heads, dim, page, pages, steps, vocab = 2, 4, 64, 8, 40, 3, 500
    gen = torch.Generator().manual_seed(11)
    cache = w4a16.KvCache.empty(pages, page, heads, dim, "fp8", device=cuda)
    table = torch.randperm(pages, generator=gen)[:24].reshape(2, 12).to(torch.int32).to(cuda)
    kv_lens = torch.zeros(2, dtype=torch.int32, device=cuda)
    keys = [torch.zeros(0, heads, dim, dtype=torch.bfloat16) for _ in range(2)]
    values = [torch.zeros(0, heads, dim, dtype=torch.bfloat16) for _ in range(2)]
    starts = torch.arange(3, dtype=torch.int32, device=cuda) * (steps + 1)
    for _ in range(6):
        new_k, new_v = (torch.randn(2 * (steps + 1), heads, dim, generator=gen).to(torch.bfloat16) for _ in range(2))
        q = torch.randn(2 * (steps + 1), q_heads, dim, generator=gen).to(torch.bfloat16)
        kv_lens += steps + 1
        batch = w4a16.KvBatch(table, kv_lens, starts, 2 * (steps + 1), max_new=steps + 1, max_kv=96)
        cache.write(new_k.to(cuda), new_v.to(cuda), batch)
        out, lse = w4a16.paged_attention(q.to(cuda), cache, batch, return_lse=True)
        for s in range(2):
            keys[s] = torch.cat([keys[s], new_k[s * (steps + 1):(s + 1) * (steps + 1)]])
            values[s] = torch.cat([values[s], new_v[s * (steps + 1):(s + 1) * (steps + 1)]])
        lens = kv_lens.tolist()
        assert lens == [len(x) for x in keys]
        k64, v64 = ([kv_oracle.values(*kv_oracle.quantise(x, "fp8")).transpose(0, 1) for x in y] for y in (keys, values))
        there = [torch.ones(n, dtype=torch.bool) for n in lens]
        want, want_lse, off, lse_off = kv_oracle.attention(q, k64, v64, there, dim**-0.5, True, 0, [steps + 1] * 2, lens)
        assert ((out.cpu().double() - want).abs() <= off).all() and ((lse.cpu().double() - want_lse).abs() <= lse_off).all()
        logits = torch.randn(2, steps + 1, vocab, generator=gen)
        target = torch.softmax(logits, -1)
        draft = torch.softmax(logits[:, :steps] + 0.8 * torch.randn(2, steps, vocab, generator=gen), -1)
        drafted = torch.multinomial(draft.reshape(-1, vocab), 1, generator=gen).reshape(2, steps).to(torch.int32)
        uniforms = torch.rand(2, steps + 1, generator=gen)
        accepted, tokens = w4a16.verify_drafts(target.to(cuda), drafted.to(cuda), uniforms.to(cuda), draft=draft.to(cuda))
        some, all_tokens = kv_oracle.verify(target.numpy(), draft.numpy(), drafted.numpy(), None, uniforms.numpy())
        assert accepted.tolist() == some.tolist() and tokens.tolist() == all_tokens.tolist()
        # the token at the sequence's end and the taken ones stay
        kv_lens -= steps - accepted
        for s in range(2):
            keys[s], values[s] = (x[:len(x) - steps + int(some[s])] for x in (keys[s], values[s]))
