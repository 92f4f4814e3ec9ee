"""The decode step's operators beside the INT4 FFN: the paged KV cache (written in BF16, INT8 or FP8, and
read back), attention of new tokens over it, and the verification of drafted tokens.

A case is one call of one operator, as a serving loop makes it: one token, the few rows that a
speculative step verifies, a chunk of a prompt, or a batch of all of these.

Ranges that the cases stand for: 1 to 64 sequences (128 for the drafts), 1 to 8192 new tokens a call, 1 to 131072
cached tokens a sequence, pages of 8 to 256 tokens, heads of 64, 128 and 256 values in groups of 1 to 16 queries a
key head, caches of BF16, INT8 and FP8 (e4m3, a scale per token and head), sliding windows;
vocabularies of 1000 to 200000 words with 1 to 16 drafted tokens.
"""

import math
import os
import random
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.getcwd(), "haskell-infer-demo_amd"))

TOP = {"int8": 127.0, "fp8": 448.0}
TYPES = {"bf16": torch.bfloat16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
SMALL = 2.0**-117  # rows under it are held as zeros: the inverse of their scale would pass FP32


def listed():
    return [
        # one decode step's new token of a few sequences into the cache: latency
        dict(name="write-token", entry="write", seqs=4, new=1, kv=900, ragged=True, kv_heads=8, head_dim=128, page=16,
             cache="fp8", lens=1),
        # a chunk of two prompts into the cache
        dict(name="write-chunk", entry="write", seqs=2, new=4099, kv=6000, ragged=False, kv_heads=8, head_dim=128,
             page=64, cache="fp8", lens=2),
        # a short chunk appended and the whole sequences taken back out, as before a prefix is moved elsewhere
        dict(name="append-read", entry="append_read", seqs=3, new=37, kv=2100, ragged=True, kv_heads=4, head_dim=256,
             page=32, cache="int8", lens=3),
        # a large batch's cache taken out of its pages, to be kept or sent on
        dict(name="read-batch", entry="read", seqs=24, new=0, kv=8191, ragged=True, kv_heads=8, head_dim=128, page=16,
             cache="fp8", lens=4),
        # one user, one token: the smallest attention call
        dict(name="decode-one", entry="attention", seqs=1, new=1, kv=1337, ragged=False, q_heads=32, kv_heads=8,
             head_dim=128, page=16, cache="bf16", window=0, lens=5),
        # a decode step of a ragged batch
        dict(name="decode-batch", entry="attention", seqs=48, new=1, kv=8192, ragged=True, q_heads=32, kv_heads=8,
             head_dim=128, page=16, cache="int8", window=0, lens=6),
        # few users with long contexts, and wide heads in odd groups
        dict(name="decode-long", entry="attention", seqs=2, new=1, kv=100003, ragged=False, q_heads=24, kv_heads=4,
             head_dim=256, page=64, cache="fp8", window=0, lens=7),
        # the rows that a speculative step verifies
        dict(name="verify-rows", entry="attention", seqs=16, new=5, kv=4096, ragged=True, q_heads=32, kv_heads=8,
             head_dim=128, page=32, cache="fp8", window=0, lens=8),
        # prompts taken in chunks over what is cached already: the most work
        dict(name="chunk-long", entry="attention", seqs=2, new=4096, kv=16384, ragged=True, q_heads=32, kv_heads=8,
             head_dim=128, page=64, cache="bf16", window=0, lens=9),
        # prompts' chunks and decoding sequences in one call, narrow heads, a sliding window
        dict(name="chunk-mixed", entry="attention", seqs=9, new=1023, kv=5000, ragged=True, q_heads=20, kv_heads=4,
             head_dim=64, page=16, cache="int8", window=1500, lens=10),
        # one speculating user
        dict(name="drafts-one", entry="drafts", seqs=1, steps=4, vocab=151936, drawn=True, lens=11),
        # a speculating batch, a vocabulary whose rows start at odd addresses
        dict(name="drafts-batch", entry="drafts", seqs=64, steps=7, vocab=128257, drawn=True, lens=12),
    ]


def _log(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def draw(rng):
    entry = rng.choice(["write", "append_read", "read", "attention", "attention", "attention", "attention", "drafts"])
    lens = rng.randrange(1 << 20)
    if entry == "drafts":
        vocab = _log(rng, 1000, 200000)
        steps = _log(rng, 1, 16)
        # no more probabilities than the largest listed case holds
        seqs = max(1, min(_log(rng, 1, 128), 64 * 8 * 128257 // (vocab * (steps + 1))))
        return dict(entry=entry, seqs=seqs, steps=steps, vocab=vocab, drawn=rng.random() < 0.7, lens=lens)
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    page = rng.choice([8, 16, 32, 64, 128, 256])
    ragged = rng.random() < 0.75
    seqs = _log(rng, 1, 64)
    # no more bytes than the largest listed cases move
    most = (1 << 26) if entry in ("read", "append_read") else (1 << 27)
    kv = min(_log(rng, 1, 131072), max(1, most // (seqs * kv_heads * head_dim)))
    if entry == "write":
        # what an INT8 write leaves is looked at as the values it stands for, by append_read
        new = min(kv, max(1, _log(rng, 1, 8192) // seqs))
        return dict(entry=entry, seqs=seqs, new=new, kv=kv, ragged=ragged, kv_heads=kv_heads, head_dim=head_dim,
                    page=page, cache=rng.choice(["bf16", "fp8"]), lens=lens)
    cache = rng.choice(["bf16", "int8", "fp8"])
    if entry in ("read", "append_read"):
        new = 0 if entry == "read" else min(kv, max(1, _log(rng, 1, 8192) // seqs))
        return dict(entry=entry, seqs=seqs, new=new, kv=kv, ragged=ragged, kv_heads=kv_heads, head_dim=head_dim,
                    page=page, cache=cache, lens=lens)
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 8, 16])
    # one token, a few verified ones, or a chunk
    new = [1, rng.randint(2, 8), max(1, _log(rng, 9, 8192) // seqs)][rng.randrange(3)]
    new = min(new, kv)
    # no more products than the largest listed case, counted as the plain form pads them
    most = 2 * 4096 * 16384 * 32 * 128
    new = max(1, min(new, most // (seqs * kv * q_heads * head_dim)))
    window = _log(rng, 64, 8192) if rng.random() < 0.3 else 0
    return dict(entry=entry, seqs=seqs, new=new, kv=kv, ragged=ragged, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, cache=cache, window=window, lens=lens)


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------


def _lens(case):
    """(cached tokens with the new ones, new tokens) of every sequence: the first has the most of both."""
    rng = random.Random(case["lens"])
    kv, new = case["kv"], case["new"]
    if not case["ragged"]:
        return [kv] * case["seqs"], [new] * case["seqs"]
    kvs = [kv] + [_log(rng, max(1, kv // 8), kv) for _ in range(case["seqs"] - 1)]
    news = [new] + [rng.randint(1, new) if new else 0 for _ in range(case["seqs"] - 1)]
    if new > 16:  # a third of the sequences are decoding ones
        news[1:] = [1 if rng.random() < 0.33 else n for n in news[1:]]
    return kvs, [min(n, k) for n, k in zip(news, kvs)]


def _starts(lens):
    total, starts = 0, [0]
    for n in lens:
        total += n
        starts.append(total)
    return starts


def _rows(gen, *shape):
    """BF16 activations ~N(0, 1) whose last axis has a few wide channels, as keys have."""
    x = torch.empty(*shape, device="cuda").normal_(0.0, 1.0, generator=gen)
    x[..., :: max(1, shape[-1] // 4)] *= 4.0
    return x.to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["entry"] == "drafts":
        return _prepare_drafts(case, gen, seed)
    kvs, news = _lens(case)
    heads, dim, page, kind = case["kv_heads"], case["head_dim"], case["page"], case["cache"]
    counts = [-(-n // page) for n in kvs]
    pages = sum(counts) + 5
    # a cache that a server has been filling: pages in no order, other sequences' tokens in the rest
    state = dict(case=case)
    for name in ("k", "v"):
        codes, scales = [], []
        for at in range(0, pages, max(1, (1 << 26) // (heads * page * dim))):
            some = _rows(gen, min(pages - at, max(1, (1 << 26) // (heads * page * dim))), heads, page, dim)
            c, s = _quantise(some, kind)
            codes.append(c)
            scales.append(s)
        codes = torch.cat([c.view(torch.uint8) for c in codes]).view(TYPES[kind])
        state[name + "_cache"] = codes
        state[name + "_scale"] = torch.cat(scales) if kind != "bf16" else None
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.zeros(len(kvs), max(counts), dtype=torch.int32)
    for b, n in enumerate(counts):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    state["table"] = table.cuda()
    state["kv_lens"] = torch.tensor(kvs, dtype=torch.int32).cuda()
    state["starts"] = torch.tensor(_starts(news), dtype=torch.int32).cuda()
    state["all_starts"] = torch.tensor(_starts(kvs), dtype=torch.int32).cuda()
    state["rows"], state["all_rows"] = sum(news), sum(kvs)
    state["max_new"], state["max_kv"] = max(news), max(kvs)
    if case["entry"] == "attention":
        # the queries stand in front of the keys and values in the rows of one fused projection
        fused = _rows(gen, sum(news), case["q_heads"] + 2 * heads, dim)
        state["q"] = fused[:, : case["q_heads"]]
    elif case["entry"] != "read":
        fused = _rows(gen, sum(news), 4 * heads, dim)
        state["k"], state["v"] = fused[:, 2 * heads:3 * heads], fused[:, 3 * heads:]
    if own:
        # what a server keeps: the handle of its cache and the descriptions of its batch
        import w4a16

        state["cache"] = w4a16.KvCache(state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"])
        state["batch"] = w4a16.KvBatch(state["table"], state["kv_lens"], state["starts"], state["rows"],
                                       max_new=state["max_new"], max_kv=state["max_kv"])
        state["all"] = w4a16.KvBatch(state["table"], state["kv_lens"], state["all_starts"], state["all_rows"],
                                     max_new=state["max_kv"], max_kv=state["max_kv"])
    return state


def _prepare_drafts(case, gen, seed):
    b, n, v = case["seqs"], case["steps"], case["vocab"]
    logits = torch.empty(b, n + 1, v, device="cuda").normal_(0.0, 3.0, generator=gen)
    target = torch.softmax(logits, -1)
    # a draft model that agrees mostly
    near = logits[:, :n] + torch.empty(b, n, v, device="cuda").normal_(0.0, 0.4, generator=gen)
    draft = torch.softmax(near, -1)
    if case["drawn"]:
        tokens = torch.multinomial(draft.reshape(b * n, v), 1, generator=gen).reshape(b, n)
    else:
        tokens, draft = draft.argmax(-1), None
    rng = random.Random(case["lens"])
    lens = [n] + [rng.randint(0, n) if rng.random() < 0.3 else n for _ in range(b - 1)]
    return dict(case=case, target=target, draft=draft, tokens=tokens.to(torch.int32),
                lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                uniforms=torch.rand(b, n + 1, device="cuda", generator=gen))


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    entry = state["case"]["entry"]
    if entry == "drafts":
        return _plain_drafts(state)
    if entry in ("write", "append_read"):
        _plain_write(state)
    if entry == "write":
        return _buffers(state)
    if entry == "attention":
        return _plain_attention(state)
    return _plain_read(state)


def _run_own(state):
    import w4a16

    entry = state["case"]["entry"]
    if entry == "drafts":
        accepted, tokens = w4a16.verify_drafts(state["target"], state["tokens"], state["uniforms"],
                                               draft=state["draft"], lens=state["lens"])
        return {"accepted": accepted, "tokens": tokens}
    if entry in ("write", "append_read"):
        state["cache"].write(state["k"], state["v"], state["batch"])
    if entry == "write":
        return _buffers(state)
    if entry == "attention":
        out, lse = w4a16.paged_attention(state["q"], state["cache"], state["batch"], window=state["case"]["window"],
                                         return_lse=True)
        return {"out": out, "lse": lse}
    k, v = state["cache"].read(state["all"])
    return {"k": k, "v": v}


def _buffers(state):
    out = {"k": state["k_cache"], "v": state["v_cache"]}
    if state["k_scale"] is not None:
        out |= {"k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    return out


def _quantise(x, kind):
    """Codes and scales of rows of BF16 values: one scale a row."""
    if kind == "bf16":
        return x, None
    x = x.float()
    most = x.abs().amax(-1)
    held = most >= SMALL
    scale = torch.where(held, most / TOP[kind], 0.0)
    scaled = x * torch.where(held, TOP[kind] / most, 0.0)[..., None]
    scaled = scaled.clamp(-TOP[kind], TOP[kind])
    return (scaled.round() if kind == "int8" else scaled).to(TYPES[kind]), scale


def _places(state, starts, rows):
    """(sequence, position) of every row: a sequence's rows are its last tokens."""
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row.to(torch.int32), right=True)
    new = (starts[1:] - starts[:-1])[seq]
    return seq, (state["kv_lens"][seq] - new + row - starts[seq]).long()


def _plain_write(state):
    page = state["case"]["page"]
    seq, at = _places(state, state["starts"], state["rows"])
    pages = state["table"][seq, at // page].long()
    for name in ("k", "v"):
        codes, scale = _quantise(state[name], state["case"]["cache"])
        if scale is None:
            state[name + "_cache"][pages, :, at % page] = codes
        else:
            state[name + "_cache"].view(torch.uint8)[pages, :, at % page] = codes.view(torch.uint8)
            state[name + "_scale"][pages, :, at % page] = scale


def _values(state, name, index):
    """The FP32 values of the cache at an index of its pages (and of their tokens)."""
    values = state[name + "_cache"][index] if state["case"]["cache"] == "bf16" else \
        state[name + "_cache"].view(torch.uint8)[index].view(TYPES[state["case"]["cache"]])
    return values.float() if state[name + "_scale"] is None else values.float() * state[name + "_scale"][index][..., None]


def _plain_read(state):
    page = state["case"]["page"]
    seq, at = _places(state, state["all_starts"], state["all_rows"])
    index = (state["table"][seq, at // page].long(), slice(None), at % page)
    return {"k": _values(state, "k", index).to(torch.bfloat16), "v": _values(state, "v", index).to(torch.bfloat16)}


def _plain_attention(state):
    case = state["case"]
    heads, group, dim = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"]
    seqs, kv, new = case["seqs"], state["max_kv"], state["max_new"]
    # the pages of every sequence in order, as [sequence, head, token, value]
    table = state["table"].long()
    k, v = (_values(state, name, (table,)).permute(0, 2, 1, 3, 4).reshape(seqs, heads, -1, dim)[:, :, :kv] for name in "kv")
    starts = state["starts"].long()
    news = starts[1:] - starts[:-1]
    step = torch.arange(new, device="cuda")
    rows = (starts[:-1, None] + step).clamp(max=state["rows"] - 1)
    q = state["q"][rows].float().reshape(seqs, new, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, heads, -1, dim)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(dim**-0.5).view(seqs, heads, group, new, kv)
    place = (state["kv_lens"].long() - news)[:, None] + step
    token = torch.arange(kv, device="cuda")
    seen = token <= place[..., None]
    if case["window"]:
        seen &= token > place[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    scores.sub_(most).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(seqs, heads, -1, kv), v).view(seqs, heads, group, new, dim) / total
    lse = (most + total.log()).squeeze(-1)
    # back to rows
    row = torch.arange(state["rows"], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    at = row - starts[seq]
    out = out.permute(0, 3, 1, 2, 4)[seq, at].reshape(-1, case["q_heads"], dim)
    return {"out": out.to(torch.bfloat16), "lse": lse.permute(0, 3, 1, 2)[seq, at].reshape(-1, case["q_heads"])}


def _plain_drafts(state):
    target, draft, tokens, lens, u = (state[n] for n in ("target", "draft", "tokens", "lens", "uniforms"))
    seqs, steps = tokens.shape
    vocab = target.shape[-1]
    each = torch.arange(seqs, device="cuda")
    at = tokens.long()[..., None]
    p = target[:, :steps].gather(-1, at)[..., 0].double()
    q = torch.ones_like(p) if draft is None else draft.gather(-1, at)[..., 0].double()
    step = torch.arange(steps, device="cuda")
    taken = (u[:, :steps].double() * q < p) & (step < lens[:, None])
    accepted = taken.int().cumprod(-1).sum(-1)
    refused = accepted < lens
    # what is left of the target's row where the draft's was refused
    row = target[each, accepted]
    first = accepted.clamp(max=steps - 1)
    if draft is None:
        less = row.scatter(-1, tokens.long()[each, first][:, None], 0.0)
    else:
        less = (row - draft[each, first]).clamp(min=0.0)
    rest = torch.where(refused[:, None], less, row)
    rest = torch.where((rest.sum(-1) > 0)[:, None], rest, row)
    sums = rest.double().cumsum(-1)
    drawn = (sums <= u[:, -1:].double() * sums[:, -1:]).sum(-1).clamp(max=vocab - 1)
    place = torch.arange(steps + 1, device="cuda")
    padded = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(place < accepted[:, None], padded,
                      torch.where(place == accepted[:, None], drawn[:, None].int(), -1))
    return {"accepted": accepted.int(), "tokens": out}


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------------


def work(case):
    if case["entry"] == "drafts":
        rows = 2 if case["drawn"] else 1
        return {"bytes": 4 * case["seqs"] * (rows * case["vocab"] + 6 * case["steps"] + 3),
                "flops": 2 * rows * case["seqs"] * case["vocab"]}
    kvs, news = _lens(case)
    heads, dim = case["kv_heads"], case["head_dim"]
    token = 2 * heads * (dim * 2 if case["cache"] == "bf16" else dim + 4)  # K and V of one cached token
    plain = 4 * heads * dim  # the same in BF16
    if case["entry"] == "write":
        return {"bytes": sum(news) * (token + plain), "flops": 4 * sum(news) * heads * dim}
    if case["entry"] == "read":
        return {"bytes": sum(kvs) * (token + plain), "flops": 2 * sum(kvs) * heads * dim}
    if case["entry"] == "append_read":
        return {"bytes": sum(news) * (token + plain) + sum(kvs) * (token + plain),
                "flops": (4 * sum(news) + 2 * sum(kvs)) * heads * dim}
    window = case["window"]
    pairs = touched = 0
    for n, m in zip(kvs, news):
        old = n - m
        if window:
            full = max(0, min(m, window - old))  # the rows that the window does not cut
            pairs += full * old + full * (full + 1) // 2 + (m - full) * window
            touched += min(n, window + m - 1)
        else:
            pairs += m * old + m * (m + 1) // 2
            touched += n
    q = sum(news) * case["q_heads"]
    return {"bytes": touched * token + q * (4 * dim + 4), "flops": 4 * pairs * case["q_heads"] * dim}


# ------------------------------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------


def exact(case, seed):
    if case["entry"] == "drafts":
        return None  # whole numbers
    state = prepare(case, seed)
    kvs, news = _lens(case)
    if case["entry"] == "attention":
        return _exact_attention(state, kvs, news)
    held = {name: state[name + "_cache"].to(torch.float64) if case["cache"] == "bf16" else
            state[name + "_cache"].view(torch.uint8).view(TYPES[case["cache"]]).to(torch.float32).double() for name in "kv"}
    scale = {name: None if state[name + "_scale"] is None else state[name + "_scale"].double() for name in "kv"}
    table = state["table"].cpu()
    if case["entry"] != "read":
        first = 0
        for b, (n, m) in enumerate(zip(kvs, news)):
            at = torch.arange(n - m, n)
            pages, inside = table[b][at // case["page"]].long().cuda(), (at % case["page"]).cuda()
            for name in "kv":
                x = state[name][first:first + m].double()
                if case["cache"] != "bf16":
                    most = x.abs().amax(-1)
                    scale[name][pages, :, inside] = most / TOP[case["cache"]]
                    x = x / most.clamp(min=SMALL)[..., None] * TOP[case["cache"]]
                    if case["cache"] == "fp8":  # three bits behind the leading one, subnormals under 2^-6
                        unit = torch.exp2((torch.frexp(x)[1] - 1).clamp(min=-6).double() - 3)
                        x = (x / unit).round() * unit
                    x = x.round() if case["cache"] == "int8" else x
                held[name][pages, :, inside] = x
            first += m
    if case["entry"] == "write":
        return held | ({} if scale["k"] is None else {"k_scale": scale["k"], "v_scale": scale["v"]})
    out = {}
    for name in "kv":
        rows = []
        for b, n in enumerate(kvs):
            at = torch.arange(n)
            pages, inside = table[b][at // case["page"]].long().cuda(), (at % case["page"]).cuda()
            x = held[name][pages, :, inside]
            rows.append(x if scale[name] is None else x * scale[name][pages, :, inside][..., None])
        out[name] = torch.cat(rows)
    return out


def _exact_attention(state, kvs, news):
    case = state["case"]
    group, dim, page = case["q_heads"] // case["kv_heads"], case["head_dim"], case["page"]
    outs, lses, first = [], [], 0
    table = state["table"].long()
    for b, (n, m) in enumerate(zip(kvs, news)):
        pages = table[b, :-(-n // page)]
        whole = {}
        for name in "kv":
            x = state[name + "_cache"].view(torch.uint8 if case["cache"] != "bf16" else torch.bfloat16)[pages]
            x = x.view(TYPES[case["cache"]]).float().double()
            if state[name + "_scale"] is not None:
                x = x * state[name + "_scale"][pages].double()[..., None]
            whole[name] = x.transpose(0, 1).reshape(case["kv_heads"], -1, dim)[:, :n]
        place = torch.arange(n - m, n, device="cuda")[:, None]
        token = torch.arange(n, device="cuda")
        hidden = token > place
        if case["window"]:
            hidden |= token <= place - case["window"]
        out = torch.empty(m, case["q_heads"], dim, dtype=torch.float64, device="cuda")
        lse = torch.empty(m, case["q_heads"], dtype=torch.float64, device="cuda")
        for h in range(case["q_heads"]):
            s = state["q"][first:first + m, h].double() @ whole["k"][h // group].T / math.sqrt(dim)
            s.masked_fill_(hidden, -math.inf)
            lse[:, h] = torch.logsumexp(s, -1)
            out[:, h] = (s - lse[:, h:h + 1]).exp() @ whole["v"][h // group]
        outs.append(out)
        lses.append(lse)
        first += m
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
