"""Beam search's selection on the GPU against FP64 and a stable sort, and the tables and caches of the beams that go on."""

import numpy as np
import pytest
import torch

import w4a16
from test_kv_cache import filled, held

pytestmark = pytest.mark.gpu


def best(logits, scores, take):
    """(scores, parents, tokens) of one group in FP64: descending, the lowest index first among equals."""
    x = logits.double().numpy()
    s = scores.double().numpy()
    with np.errstate(all="ignore"):
        most = x.max(-1, keepdims=True)
        lse = most + np.log(np.exp(x - most).sum(-1, keepdims=True))
        every = s[:, None] + (x - lse)
        none = ~np.isfinite(s)[:, None] | ~np.isfinite(lse) | np.isnan(x) | (x == -np.inf)
    every = np.where(none, -np.inf, every).reshape(-1)
    order = np.argsort(-every, kind="stable")[:take]
    got = every[order]
    real = got > -np.inf
    pad = take - len(order)
    parents = np.where(real, order // x.shape[-1], -1)
    tokens = np.where(real, order % x.shape[-1], -1)
    return (np.concatenate([got, np.full(pad, -np.inf)]), np.concatenate([parents, np.full(pad, -1)]),
            np.concatenate([tokens, np.full(pad, -1)]), every)


def check(cuda, logits, scores, take, ties=False):
    got = w4a16.beam_select(logits.to(cuda), scores.to(cuda), take)
    assert [tuple(t.shape) for t in got] == [(logits.shape[0], take)] * 3
    for g in range(logits.shape[0]):
        want, parents, tokens, every = best(logits[g], scores[g], take)
        mine, p, t = (x[g].cpu().numpy() for x in got)
        assert np.array_equal(p == -1, parents == -1) and np.array_equal(mine == -np.inf, want == -np.inf)
        real = parents >= 0
        # a score is off by its sum's 2^-22 and a rounding to FP32
        assert (np.abs(mine[real] - want[real]) <= 2.0**-21 + np.abs(want[real]) * 2.0**-23).all()
        # two candidates of different beams may change places where they are nearer than their sums are exact; of one beam never
        same = (p == parents) & (t == tokens)
        index = p.astype(np.int64) * logits.shape[-1] + t
        assert len(set(index[real])) == real.sum()
        for i in np.nonzero(~same)[0]:
            assert p[i] != parents[i] and abs(every[index[i]] - want[i]) <= 2.0**-20, (g, i)
        for b in set(p[real]):
            mine_of, want_of = t[p == b], tokens[parents == b]
            n = min(len(mine_of), len(want_of))
            assert np.array_equal(mine_of[:n], want_of[:n])
    return got


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab,take", [
    (1, 1, 1, 1), (1, 1, 1, 4), (2, 3, 2, 8), (3, 2, 17, 5), (1, 4, 255, 64), (2, 1, 257, 128), (1, 2, 513, 128), (5, 8, 1000, 16),
    (1, 4, 4097, 8), (2, 16, 5003, 64), (1, 64, 3001, 128), (3, 5, 32000, 10), (2, 10, 50257, 40), (1, 4, 151936, 8), (1, 1, 200000, 1),
    (40, 3, 700, 7), (1, 130, 900, 33),
])
def test_against_a_sort(cuda, groups, beams, vocab, take, kind):
    print(f"select {kind} groups={groups} beams={beams} vocab={vocab} take={take}", flush=True)
    for seed, spread in ((1, 3.0), (2, 0.05), (3, 30.0)):
        gen = torch.Generator().manual_seed(seed)
        logits = spread * torch.randn(groups, beams, vocab, generator=gen)
        scores = -10 * torch.rand(groups, beams, generator=gen)
        check(cuda, logits.to(torch.bfloat16) if kind == "bf16" else logits, scores, take)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("beams,vocab,take", [(1, 900, 64), (4, 5000, 128), (3, 40000, 33), (8, 20011, 1)])
def test_equal_values(cuda, beams, vocab, take, kind):
    """More equal candidates than there is room for: all of a row the same, a few values only, all beams alike; and the largest values in a row,
    in one chunk or at the end. The lowest numbers come first."""
    gen = torch.Generator().manual_seed(1)
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    flat = torch.zeros(1, beams, vocab)
    few = torch.randint(0, 3, (1, 1, vocab), generator=gen).float().expand(1, beams, vocab)
    rising = torch.arange(vocab).float().expand(1, beams, vocab) / 64
    falling = -rising
    lone = torch.full((1, beams, vocab), -20.0)
    lone[0, beams - 1, vocab // 2:vocab // 2 + 300] = 5.0
    for logits in (flat, few, rising, falling, lone):
        logits = logits.to(dtype)
        for scores in (torch.zeros(1, beams), -torch.arange(beams).float()[None]):
            out = w4a16.beam_select(logits.to(cuda).contiguous(), scores.to(cuda), take)
            want, parents, tokens, _ = best(logits[0], scores[0], take)
            # rows that are alike have sums that are alike, whatever they are: equal candidates are equal here too
            assert out[1][0].tolist() == parents.tolist() and out[2][0].tolist() == tokens.tolist()
            assert (np.abs(out[0][0].cpu().numpy() - want) <= 2.0**-21 + np.abs(want) * 2.0**-23).all()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_values_that_are_none(cuda, kind):
    """Masked words, beams that are out, beams with a NaN or an infinity, scores that are none, groups without any candidate."""
    gen = torch.Generator().manual_seed(4)
    logits = torch.randn(5, 6, 3001, generator=gen)
    logits[0, :, 5:] = -float("inf")           # 30 candidates
    logits[1, 0, 77] = float("nan")
    logits[1, 1, 3000] = float("inf")
    logits[1, 2, :] = -float("inf")
    logits[1, 3, :2900] = -float("inf")        # whole pieces masked
    scores = -torch.rand(5, 6, generator=gen)
    scores[2] = torch.tensor([float("nan"), -float("inf"), float("inf"), -1.0, -float("inf"), -2.0])
    scores[3] = -float("inf")
    logits[4] = float("nan")
    scores[1, 4:] = -float("inf")
    for take in (1, 40, 128):
        out = check(cuda, logits.to(torch.bfloat16) if kind == "bf16" else logits, scores, take)
        assert (out[1][3:] == -1).all() and (out[2][3:] == -1).all() and (out[0][3:] == -float("inf")).all()
        assert set(out[1][1].tolist()) <= {3, -1} and set(out[1][2].tolist()) <= {3, 5}


def test_far_scores(cuda):
    """Scores so large that logits are rounded off beside them: equal candidates, the lowest first; large logits."""
    logits = torch.randn(1, 2, 700, generator=torch.Generator().manual_seed(4))
    out = w4a16.beam_select(logits.to(cuda), torch.tensor([[-1.0e30, -1.0e30]], device=cuda), 20)
    assert out[1][0].tolist() == [0] * 20 and out[2][0].tolist() == list(range(20))
    check(cuda, 1.0e4 * logits, torch.zeros(1, 2), 20)
    check(cuda, 3.0e38 * torch.sign(logits), torch.zeros(1, 2), 20)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_strided_and_captured(cuda, kind):
    """Rows at odd addresses; a graph with other values of each replay, eager work between; a call on another stream."""
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    wide = torch.randn(3, 6, 5009, device=cuda).to(dtype)
    scores = -torch.rand(3, 4, device=cuda)
    view = wide[:, 1:5, 3:5004]
    want = w4a16.beam_select(view.contiguous(), scores, 12)
    got = w4a16.beam_select(view, scores, 12)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    workspace = torch.empty(1 << 20, dtype=torch.uint8, device=cuda)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = w4a16.beam_select(view, scores, 12, workspace=workspace)
    for n in range(4):
        wide.normal_()
        scores.uniform_(-3, 0)
        graph.replay()
        torch.cuda.synchronize()
        again = w4a16.beam_select(view, scores, 12)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = w4a16.beam_select(view, scores, 12, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, again))


def tables_of(table, lens, parents, page):
    """(new table, source) one beam after another."""
    groups, beams = len(parents), len(parents[0])
    new, source = [], []
    for g in range(groups):
        rows = table[g * beams:(g + 1) * beams]
        full = max(lens[g * beams], 0) // page
        up = [p if 0 <= p < beams else b for b, p in enumerate(parents[g])]
        keeper = {}
        for b, p in enumerate(up):
            keeper.setdefault(p, b)
        gone = [p for p in range(beams) if p not in keeper]
        for b, p in enumerate(up):
            own = p if keeper[p] == b else gone.pop(0)
            source.append(-1 if keeper[p] == b else g * beams + keeper[p])
            new.append(rows[p][:full] + rows[own][full:])
    return new, source


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("groups,beams,dim,heads,page,lens", [
    (1, 1, 64, 1, 8, [5]), (2, 4, 128, 2, 16, [37, 48]), (3, 5, 256, 1, 64, [70, 64, 1]), (1, 70, 64, 3, 8, [20]), (2, 8, 128, 8, 32, [0, 100]),
    (1, 3, 64, 2, 256, [255]), (1, 200, 64, 1, 8, [9]),
])
def test_beams_go_on(cuda, groups, beams, dim, heads, page, lens, fmt):
    """Every beam's tokens after the move are its parent's before, in pages that no two beams of a group share where they are
    to be written; the rest of the cache stays."""
    print(f"beams {fmt} groups={groups} beams={beams} dim={dim} page={page}", flush=True)
    every = [n for n in lens for _ in range(beams)]
    columns = max(lens) // page + 2
    pages = groups * beams * columns + 3
    rng = np.random.default_rng(beams)
    table = rng.permutation(pages)[:groups * beams * columns].reshape(-1, columns).astype(np.int32)
    cache = filled(pages, page, heads, dim, fmt, cuda, seed=beams)
    kv_lens = torch.tensor(every, dtype=torch.int32, device=cuda)
    dev_table = torch.from_numpy(table).to(cuda)
    for n in range(4):
        parents = [rng.integers(0, beams, beams).tolist(), list(range(beams))[::-1], [beams // 2] * beams,
                   rng.integers(-2, beams + 2, beams).tolist()][n]
        parents = [parents] * groups
        before = {name: held(cache, name) for name in "kv"}
        old = dev_table.tolist()
        new, source = w4a16.beam_tables(dev_table, kv_lens, torch.tensor(parents, dtype=torch.int32, device=cuda), page)
        want, want_source = tables_of(old, every, parents, page)
        assert new.tolist() == want and source.tolist() == want_source
        cache.copy_tails(new, kv_lens, source)
        expected = {name: [t.clone() if t is not None else None for t in before[name]] for name in "kv"}
        for s, src in enumerate(want_source):
            tail = every[s] % page
            if src >= 0 and tail:
                to, of = want[s][every[s] // page], want[src][every[s] // page]
                for name in "kv":
                    for t in expected[name]:
                        if t is not None:
                            raw = t.view(torch.uint8) if t.element_size() == 1 else t
                            raw[to, :, :tail] = raw[of, :, :tail]
        for name in "kv":
            for a, b in zip(held(cache, name), expected[name]):
                assert a is None or torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b)
        for g in range(groups):
            own = [tuple(r[every[g * beams] // page:]) for r in want[g * beams:(g + 1) * beams]]
            assert len(set(own)) == beams
        dev_table = new


def test_tables_in_wider_ones(cuda):
    """Tables whose rows stand apart, into an `out` that does too; copies of pages that are none are left out."""
    wide = torch.arange(6 * 9, dtype=torch.int32, device=cuda).reshape(6, 9)
    lens = torch.full((6,), 20, dtype=torch.int32, device=cuda)
    parents = torch.tensor([[1, 1, 2], [0, 0, 0]], dtype=torch.int32, device=cuda)
    out = torch.full((6, 7), -5, dtype=torch.int32, device=cuda)
    got, source = w4a16.beam_tables(wide[:, 2:7], lens, parents, 8, out=out[:, 1:6])
    want, want_source = tables_of(wide[:, 2:7].tolist(), [20] * 6, parents.tolist(), 8)
    assert got.tolist() == want and source.tolist() == want_source and (out[:, 0] == -5).all() and (out[:, 6] == -5).all()
    cache = filled(30, 8, 2, 64, "bf16", cuda, seed=1)
    before = held(cache, "k")[0]
    cache.copy_tails(got, lens, torch.tensor([5, 9, -7, 1 << 30, 4, 0], dtype=torch.int32, device=cuda))
    after = held(cache, "k")[0]
    # sequences 0 and 5 name another one; of their pages only those inside the cache count
    column = 20 // 8
    allowed = {want[s][column] for s in (0, 5)}
    changed = {p for p in range(30) if not torch.equal(before[p], after[p])}
    assert changed <= allowed
    one_column = torch.zeros(6, 1, dtype=torch.int32, device=cuda)
    cache.copy_tails(one_column, lens, source)  # the tails lie past the table
    assert torch.equal(held(cache, "k")[0], after)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim,heads,page", [(64, 3, 8), (128, 8, 16), (256, 1, 64)])
def test_keep_path(cuda, dim, heads, page, fmt):
    """Paths of every kind against taking all tokens first: places that are taken from and written, entries that are none."""
    kv_lens, news = [300, 90, 64, 40, 3], [200, 17, 64, 1, 5]
    columns, pages = 300 // page + 2, 5 * (300 // page + 2)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(5, columns)
    table[1, 5:7] = -3  # pages that are none
    batch = w4a16.KvBatch(table.to(cuda), torch.tensor(kv_lens, dtype=torch.int32, device=cuda),
                          torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=cuda), sum(news))
    rng = np.random.default_rng(dim)
    for width in (1, 9, 200, 256):
        path = np.full((5, width), -1, np.int32)
        for s, m in enumerate(news):
            count = int(rng.integers(0, min(width, m) + 1))
            path[s, :count] = np.sort(rng.permutation(m)[:count])
        path[2] = rng.integers(-5, 70, width)  # no path at all
        cache = filled(pages, page, heads, dim, fmt, cuda, seed=width)
        before = {name: held(cache, name) for name in "kv"}
        cache.keep_path(batch, torch.from_numpy(path).to(cuda))

        def place(s, i):
            at = kv_lens[s] - news[s] + i
            p = int(table[s, at // page]) if 0 <= at < columns * page else -1
            return (p, at % page) if p >= 0 else None

        expected = {name: [None if t is None else t.clone() for t in before[name]] for name in "kv"}
        for s, m in enumerate(news):
            for j in range(min(width, m)):
                i = int(path[s, j])
                if j < i < m and place(s, i) and place(s, j):
                    (p, at), (q, to) = place(s, i), place(s, j)
                    for name in "kv":
                        for t, u in zip(expected[name], before[name]):
                            if t is not None:
                                a, b = (x.view(torch.uint8) if x.element_size() == 1 else x for x in (t, u))
                                a[q, :, to] = b[p, :, at]
        for name in "kv":
            for a, b in zip(held(cache, name), expected[name]):
                assert a is None or torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b)


def test_the_longest_row(cuda):
    """2^31 - 1 words: the last of a lane's eight is none. All of a value but a few, so that the sum is known."""
    vocab = 2**31 - 1
    logits = torch.full((1, 1, vocab), -1.0, dtype=torch.bfloat16, device=cuda)
    some = {0: 24.0, vocab - 1: 26.0, vocab - 8: 25.0, 1 << 30: 23.0}
    for at, x in some.items():
        logits[0, 0, at] = x
    got, parents, tokens = w4a16.beam_select(logits, torch.full((1, 1), 0.5, device=cuda), 4)
    assert tokens.tolist() == [[vocab - 1, vocab - 8, 0, 1 << 30]] and parents.tolist() == [[0] * 4]
    lse = np.log((vocab - 4) * np.exp(-1.0) + sum(np.exp(x) for x in some.values()))
    want = 0.5 + np.array([26.0, 25.0, 24.0, 23.0]) - lse
    assert (np.abs(got[0].cpu().numpy() - want) <= 2.0**-21 + np.abs(want) * 2.0**-23).all()
