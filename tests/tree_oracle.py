"""Plain statements of drafted trees on the CPU: what their nodes see, attention under such masks in FP64 with the bounds that its
roundings allow, and their verification."""

import numpy as np
import torch


def links(parents, size):
    """Of each of a tree's `size` nodes those from itself up to its root."""
    ways = []
    for i in range(size):
        p = int(parents[i])
        ways.append([i] + (ways[p] if 0 <= p < i else []))
    return ways


def plan(parents, sizes, kv_lens, news, nodes):
    """(seen as sets of nodes, positions) of every row."""
    seen, positions = [], []
    for s, (n, m) in enumerate(zip(kv_lens, news)):
        size = min(max(int(sizes[s]), 0), nodes)
        ways = links(parents[s], size)
        for i in range(m):
            node = size - m + i
            seen.append(ways[node] if node >= 0 else [])
            positions.append(n - size + (len(ways[node]) - 1 if node >= 0 else node))
    return seen, positions


def bits(seen, nodes):
    """Sets of nodes as int64 words."""
    out = np.zeros((len(seen), (nodes + 63) // 64), np.uint64)
    for row, of in zip(out, seen):
        for j in of:
            row[j // 64] |= np.uint64(1 << (j % 64))
    return torch.from_numpy(out.view(np.int64))


def visible(seen, positions, sizes, kv_lens, news, nodes, window):
    """Of every sequence [rows, tokens]: whether a row sees a token."""
    out, first = [], 0
    for s, (n, m) in enumerate(zip(kv_lens, news)):
        size = min(max(int(sizes[s]), 0), nodes)
        base = n - size
        v = torch.zeros(m, n, dtype=torch.bool)
        for i in range(m):
            at = n - m + i
            position = at if at < base else min(max(positions[first + i], base), at)
            v[i, (max(0, position - window + 1) if window else 0):max(0, min(base, at + 1))] = True
            for j in seen[first + i]:
                if 0 <= base + j <= at and j < size:
                    v[i, base + j] = True
        out.append(v)
        first += m
    return out


def attention(q, k, v, there, seen_by, scale, sizes_of_codes=None, half=None):
    """FP64 attention of rows q [rows, q_heads, D] over keys and values k[s], v[s] [kv_heads, tokens, D] with there[s] [tokens] and
    seen_by[s] [rows, tokens]; and its bounds, which are kv_oracle.attention's, row by row. Rows that see nothing give zeros."""
    bf16 = torch.finfo(torch.bfloat16).eps / 2
    if half is None:
        half = bf16 if sizes_of_codes is None else torch.finfo(torch.float16).eps / 2
    group, dim = q.shape[1] // k[0].shape[0], q.shape[2]
    outs, lses, out_off, lse_off, first = [], [], [], [], 0
    for s, seen in enumerate(seen_by):
        tokens = k[s].shape[1]
        for i in range(seen.shape[0]):
            of = seen[i, :tokens] & there[s]
            x = q[first + i].double().reshape(-1, group, dim)
            keys, vals = k[s][:, of], v[s][:, of]
            if keys.shape[1] == 0:
                outs.append(torch.zeros(q.shape[1], dim, dtype=torch.float64))
                out_off.append(torch.zeros(q.shape[1], dim, dtype=torch.float64))
                lses.append(torch.full((q.shape[1],), float("-inf"), dtype=torch.float64))
                lse_off.append(torch.zeros(q.shape[1], dtype=torch.float64))
                continue
            score = torch.matmul(x, keys.transpose(-1, -2)) * scale
            score_off = (torch.matmul(x.abs(), keys.abs().transpose(-1, -2)) * abs(scale) * (dim + 8) * 2.0**-24).amax(-1)
            lse = torch.logsumexp(score, -1)
            p = (score - lse[..., None]).exp()
            out, weight = torch.matmul(p, vals), torch.matmul(p, vals.abs())
            rel = 2 * (score_off + 2.0**-21) + (keys.shape[1] + 16) * 2.0**-24
            least = 0.0
            if sizes_of_codes is not None:
                codes, scales = sizes_of_codes[s]
                most = scales[:, there[s]].amax(-1).clamp(min=2.0**-120)
                least = 2.0**-31 * p.amax(-1)[..., None] * most[:, None, None] * codes[:, of].sum(1)[:, None]
            outs.append(out.reshape(-1, dim))
            out_off.append(((weight * (half + rel[..., None]) + least) * (1 + bf16) + out.abs() * bf16).reshape(-1, dim))
            lses.append(lse.reshape(-1))
            lse_off.append((score_off + 2.0**-20 + (keys.shape[1] + 16) * 2.0**-24
                            + (lse.abs() + score.abs().amax(-1)) * 2.0**-22).reshape(-1))
        first += seen.shape[0]
    return tuple(torch.stack(t) for t in (outs, lses, out_off, lse_off))


def check(out, lse, wanted):
    want, want_lse, off, lse_off = wanted
    got, got_lse = out.cpu().double(), lse.cpu().double()
    empty = want_lse == float("-inf")
    assert torch.equal(got_lse == float("-inf"), empty) and (got[empty] == 0).all()
    far = ((got - want).abs() / off.clamp(min=1e-300))[~empty]
    lse_far = ((got_lse - want_lse).abs() / lse_off.clamp(min=1e-300))[~empty]
    if far.numel():
        print(f"  of what the roundings allow: out {far.max():.3f}, lse {lse_far.max():.3f}", flush=True)
        assert far.max() <= 1 and lse_far.max() <= 1


def verify(target, tokens, parents, sizes, uniforms):
    """The definition of the tree's verification, one sequence and one node after another, in FP64: (accepted, path, tokens)."""
    seqs, nodes, vocab = target.shape
    accepted, paths, out = [], np.full((seqs, nodes), -1, np.int64), np.full((seqs, nodes), -1, np.int64)

    def weight(w):
        return np.where((w > 0) & np.isfinite(w), w, np.float32(0)).astype(np.float32)

    for s in range(seqs):
        size = nodes if sizes is None else min(max(int(sizes[s]), 1), nodes)
        node, path = 0, [0]
        while True:
            children = [i for i in range(size) if 0 <= int(parents[s, i]) < i and int(parents[s, i]) == node]
            left, asked, following = np.float64(1), set(), None
            for i in children:
                x = int(tokens[s, i])
                if x in asked:
                    continue
                asked.add(x)
                p = np.float64(weight(target[s, node, x])) if 0 <= x < vocab else np.float64(0)
                if np.float64(uniforms[s, i]) * left < p:
                    following = i
                    break
                left = max(left - p, np.float64(0))
            if following is None:
                break
            node = following
            path.append(node)
        row = weight(target[s, node])
        rest = row.copy()
        for x in asked:
            if 0 <= x < vocab:
                rest[x] = 0
        if not rest.any():
            rest = row
        taken = len(path) - 1
        paths[s, :taken + 1] = path
        out[s, :taken] = [tokens[s, i] for i in path[1:]]
        if rest.any():
            run = np.cumsum(rest.astype(np.float64))
            with np.errstate(invalid="ignore"):
                past = np.nonzero((run > np.float64(uniforms[s, 0]) * run[-1]) & (rest > 0))[0]
            out[s, taken] = past[0] if len(past) else np.nonzero(rest)[0][-1]
        accepted.append(taken)
    return np.array(accepted), paths, out
