"""Plain statements of the paged cache, the attention over it and the draft verification, on the CPU in numpy and
FP64 torch: what the GPU tests compare with, and the bounds that their roundings allow.

A batch is given as lists: `kv_lens`, `news` and a page table (rows of page numbers)."""

import numpy as np
import torch

TOP = {"int8": 127.0, "fp8": 448.0}
DTYPE = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


def quantise(x, fmt):
    """(codes, scales) of BF16 rows [.., D] (CPU): FP32 arithmetic, each step rounded once."""
    if fmt == "bf16":
        return x.clone(), None
    f = x.float().numpy()
    top = np.float32(TOP[fmt])
    most = np.abs(f).max(-1)
    finite = np.isfinite(f).all(-1)
    held = finite & (most >= np.float32(2.0**-117))
    with np.errstate(all="ignore"):
        inverse = np.where(held, top / np.where(held, most, np.float32(1)), np.float32(0)).astype(np.float32)
        scale = np.where(held, most / top, np.where(finite, np.float32(0), np.float32("nan"))).astype(np.float32)
        code = np.where(held[..., None], np.clip(np.where(held[..., None], f, 0) * inverse[..., None], -top, top), np.float32(0))
    code = torch.from_numpy(code.astype(np.float32))
    return (code.round() if fmt == "int8" else code).to(DTYPE[fmt]), torch.from_numpy(scale)


def values(codes, scales):
    """What codes stand for, in FP64."""
    v = codes.float().double()
    return v if scales is None else v * scales.double()[..., None]


def places(table, kv_lens, news, page, pages):
    """For every row: (sequence, page or -1, place in it)."""
    out = []
    for s, (n, m) in enumerate(zip(kv_lens, news)):
        for i in range(m):
            at = n - m + i
            if 0 <= at < len(table[s]) * page and 0 <= table[s][at // page] < pages:
                out.append((s, table[s][at // page], at % page))
            else:
                out.append((s, -1, 0))
    return out


def attention(q, k, v, places_of, scale, causal, window, news, kv_lens, coded=None, half=None):
    """FP64 attention of the rows q [rows, q_heads, D] of sequences whose tokens' keys and values are
    k[s], v[s] [kv_heads, tokens, D] and places_of[s] [tokens] whether each is there. kv_lens places the rows, and may
    be more than the tokens there are. Returns (out, lse, and for each of
    them how far FP32 arithmetic with BF16 weights and a BF16 output may be off). `coded`: of an 8-bit cache, whose weights are
    FP16, the sizes of each sequence's V codes [kv_heads, tokens, D] and of their scales [kv_heads, tokens]. `half`: how far
    a weight may be off instead, relatively.

    The bounds. A score is a sum of D products: off by (D + 4) 2^-24 sum|q k| scale, and by a rounding or two of its own;
    a weight exp(s - m) by as much relatively, and 2^-21 for the exponential; both a weight and the sum of weights can
    be off by that, so an output by twice that of sum p|v|. Weights are rounded to BF16 (half a step, 2^-8, of
    sum p|v|), the output once more (2^-8 of itself); sums of n terms add n 2^-24.

    FP16 weights carry V's scales: what is rounded is exp(s - m) scale 2^6 / 2^e, where m is no more than the row's maximum
    and 2^e no more than the largest scale of the sequence's tokens for that head, 2^-120 at least (or the kernel's tile
    has not come across it yet, and both are less). Half a step of FP16 is 2^-11 of the value, or 2^-25 under 2^-14. The
    first is 2^-11 of sum p|v|. The second, less 2^6 / 2^e, is 2^-31 2^e of an exp(s - m); over the sum of weights
    exp(m) is at most the largest weight p: 2^-31 max p, max scale for each |code|."""
    bf16 = torch.finfo(torch.bfloat16).eps / 2
    if half is None:
        half = bf16 if coded is None else torch.finfo(torch.float16).eps / 2
    group = q.shape[1] // k[0].shape[0]
    outs, lses, out_off, lse_off, first = [], [], [], [], 0
    dim = q.shape[2]
    for s, m in enumerate(news):
        token = torch.arange(k[s].shape[1])
        for i in range(m):
            at = kv_lens[s] - m + i
            seen = places_of[s] & (token < kv_lens[s])
            if causal:
                seen = seen & (token <= at)
            if window:
                seen = seen & (token > at - window)
            x = q[first + i].double().reshape(-1, group, dim)  # [kv_heads, group, D]
            keys, vals = k[s][:, seen], v[s][:, seen]
            if keys.shape[1] == 0:
                shape = x.shape
                outs.append(torch.zeros(q.shape[1], dim, dtype=torch.float64))
                out_off.append(torch.zeros(q.shape[1], dim, dtype=torch.float64))
                lses.append(torch.full((q.shape[1],), float("-inf"), dtype=torch.float64))
                lse_off.append(torch.zeros(q.shape[1], dtype=torch.float64))
                continue
            score = torch.matmul(x, keys.transpose(-1, -2)) * scale
            score_off = torch.matmul(x.abs(), keys.abs().transpose(-1, -2)) * abs(scale) * (dim + 8) * 2.0**-24
            score_off = score_off.amax(-1)
            lse = torch.logsumexp(score, -1)
            p = (score - lse[..., None]).exp()
            out = torch.matmul(p, vals)
            weight = torch.matmul(p, vals.abs())
            rel = 2 * (score_off + 2.0**-21) + (keys.shape[1] + 16) * 2.0**-24
            least = 0.0
            if coded is not None:
                codes, scales = coded[s]
                most = scales[:, places_of[s]].amax(-1).clamp(min=2.0**-120)
                least = 2.0**-31 * p.amax(-1)[..., None] * most[:, None, None] * codes[:, seen].sum(1)[:, None]
            outs.append(out.reshape(-1, dim))
            out_off.append(((weight * (half + rel[..., None]) + least) * (1 + bf16) + out.abs() * bf16).reshape(-1, dim))
            lses.append(lse.reshape(-1))
            lse_off.append((score_off + 2.0**-20 + (keys.shape[1] + 16) * 2.0**-24
                            + (lse.abs() + score.abs().amax(-1)) * 2.0**-22).reshape(-1))
        first += m
    return tuple(torch.stack(t) for t in (outs, lses, out_off, lse_off))


def verify(target, draft, tokens, lens, uniforms):
    """The definition, one sequence and one token after another, in FP64."""
    seqs, rows, vocab = target.shape
    accepted, out = [], np.full((seqs, rows), -1, np.int64)

    def weight(w):
        return np.where((w > 0) & np.isfinite(w), w, np.float32(0)).astype(np.float32)

    for s in range(seqs):
        n = rows - 1 if lens is None else min(max(int(lens[s]), 0), rows - 1)
        taken, refused = 0, False
        for i in range(n):
            x = int(tokens[s, i])
            inside = 0 <= x < vocab
            q = np.float64(1.0 if draft is None else draft[s, i, x]) if inside else np.float64(0)
            with np.errstate(invalid="ignore"):
                if not (inside and np.float64(uniforms[s, i]) * q < np.float64(target[s, i, x])):
                    refused = True
                    break
            taken += 1
        row = target[s, taken]
        rest = weight(row)
        if refused and draft is not None:
            with np.errstate(invalid="ignore"):
                rest = weight((row - draft[s, taken]).astype(np.float32))
        elif refused and 0 <= int(tokens[s, taken]) < vocab:
            rest = rest.copy()
            rest[int(tokens[s, taken])] = 0
        if not rest.any():
            rest = weight(row)
        out[s, :taken] = tokens[s, :taken]
        if rest.any():
            run = np.cumsum(rest.astype(np.float64))
            with np.errstate(invalid="ignore"):
                past = np.nonzero((run > np.float64(uniforms[s, rows - 1]) * run[-1]) & (rest > 0))[0]
            out[s, taken] = past[0] if len(past) else np.nonzero(rest)[0][-1]
        accepted.append(taken)
    return np.array(accepted), out
