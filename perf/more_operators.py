"""Operators of a step over a tree of drafted tokens, and of a beam search: appending rotated keys and values to
the paged cache, attention of a tree's tokens over it, the selection over beams and vocabulary with the
reordering of the beams' caches, and the verification of a drafted tree with its path kept in the cache.

A case is what a serving loop calls at one place of such a step. Every one of them works on what stays in
the server's hands: the cache, the table of its pages, the tree's links.

Ranges that the cases stand for: 1 to 64 sequences of 1 to 131072 cached tokens (beams: 1 to 32 groups of 1 to 64),
1 to 8192 appended rows, trees of 1 to 256 nodes, pages of 8 to 256 tokens, heads of 64, 128 and 256
values in groups of 1 to 16 queries a key head, rotations of a quarter of a head to the whole of it, caches
of BF16, INT8 and FP8 (e4m3, a scale per token and head), sliding windows; vocabularies of 1000 to 200000
words, of which 1 to 64 candidates a group are selected.
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
        # one decode step's new token of a few sequences: latency
        dict(name="append-token", entry="append", seqs=4, nodes=0, new=1, kv=900, ragged=True, q_heads=32, kv_heads=8, head_dim=128,
             page=16, cache="fp8", rotary=128, interleaved=False, base=1e6, lens=1),
        # a chunk of two prompts
        dict(name="append-chunk", entry="append", seqs=2, nodes=0, new=4099, kv=6000, ragged=False, q_heads=32, kv_heads=8,
             head_dim=128, page=64, cache="bf16", rotary=128, interleaved=False, base=1e6, lens=2),
        # the trees of a speculating batch: their masks and positions, and their rows, a quarter of each head turned
        dict(name="append-trees", entry="append", seqs=16, nodes=37, new=37, kv=9000, ragged=True, q_heads=24, kv_heads=4,
             head_dim=256, page=32, cache="int8", rotary=64, interleaved=True, base=1e7, lens=3),
        # one user's tree
        dict(name="tree-one", entry="attention", seqs=1, nodes=26, new=26, kv=1500, ragged=False, q_heads=32, kv_heads=8,
             head_dim=128, page=16, cache="bf16", window=0, lens=4),
        # a speculating batch, ragged in its lengths and trees
        dict(name="tree-batch", entry="attention", seqs=16, nodes=60, new=60, kv=8192, ragged=True, q_heads=32, kv_heads=8,
             head_dim=128, page=32, cache="fp8", window=0, lens=5),
        # the last level of trees that are being grown, over long contexts, wide heads in odd groups
        dict(name="grow-long", entry="attention", seqs=2, nodes=23, new=5, kv=100003, ragged=False, q_heads=24, kv_heads=4,
             head_dim=256, page=64, cache="int8", window=0, lens=6),
        # the widest trees, narrow heads, a sliding window
        dict(name="tree-wide", entry="attention", seqs=8, nodes=251, new=251, kv=16384, ragged=True, q_heads=32, kv_heads=4,
             head_dim=64, page=128, cache="bf16", window=4096, lens=7),
        # one user's beams
        dict(name="select-one", entry="select", groups=1, beams=4, vocab=151936, take=8, logits="bf16", lens=8),
        # the frontiers of a batch of trees, a vocabulary whose rows start at odd addresses
        dict(name="select-batch", entry="select", groups=16, beams=10, vocab=128257, take=40, logits="fp32", lens=9),
        # the beams of a batch go on from their parents: tables and the last pages of one layer
        dict(name="beams-move", entry="reorder", groups=16, beams=8, kv=3000, kv_heads=8, head_dim=128, page=64, cache="bf16", lens=10),
        # one user's tree is verified and its path kept
        dict(name="verify-one", entry="verify", seqs=1, nodes=26, vocab=151936, kv=1500, kv_heads=8, head_dim=128, page=16,
             cache="bf16", lens=11),
        # a batch's
        dict(name="verify-batch", entry="verify", seqs=24, nodes=40, vocab=100003, kv=700, kv_heads=8, head_dim=128, page=32,
             cache="fp8", lens=12),
    ]


def _log(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def draw(rng):
    entry = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "select", "select", "reorder",
                        "verify"])
    lens = rng.randrange(1 << 20)
    if entry == "select":
        vocab, beams = _log(rng, 1000, 200000), _log(rng, 1, 64)
        groups = max(1, min(_log(rng, 1, 32), 16 * 10 * 128257 // (beams * vocab)))
        return dict(entry=entry, groups=groups, beams=beams, vocab=vocab, take=_log(rng, 1, 64),
                    logits=rng.choice(["bf16", "fp32"]), lens=lens)
    heads = dict(kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128, 128, 256]), page=rng.choice([8, 16, 32, 64, 128, 256]))
    if entry == "reorder":
        groups, beams = _log(rng, 1, 32), _log(rng, 1, 16)
        kv = max(1, min(_log(rng, 1, 16384), (1 << 26) // (groups * beams * heads["kv_heads"] * heads["head_dim"])))
        # what INT8 pages hold is looked at as values, by append
        return dict(entry=entry, groups=groups, beams=beams, kv=kv, cache=rng.choice(["bf16", "fp8"]), lens=lens, **heads)
    if entry == "verify":
        vocab, nodes = _log(rng, 1000, 200000), _log(rng, 1, 256)
        seqs = max(1, min(_log(rng, 1, 64), 24 * 40 * 100003 // (vocab * nodes)))
        return dict(entry=entry, seqs=seqs, nodes=nodes, vocab=vocab, kv=_log(rng, nodes, 2000), cache=rng.choice(["bf16", "fp8"]),
                    lens=lens, **heads)
    q_heads = heads["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 6, 8, 16])
    cache, ragged, seqs = rng.choice(["bf16", "int8", "fp8"]), rng.random() < 0.75, _log(rng, 1, 64)
    # no more bytes than the largest listed cases move
    kv = min(_log(rng, 1, 131072), max(1, (1 << 27) // (seqs * heads["kv_heads"] * heads["head_dim"])))
    if entry == "append":
        nodes = rng.choice([0, _log(rng, 1, 256)])
        new = min(kv, max(1, _log(rng, 1, 8192) // seqs), nodes or 8192)
        rotary = heads["head_dim"] // rng.choice([1, 1, 2, 4])
        return dict(entry=entry, seqs=seqs, nodes=min(nodes, kv), new=new, kv=kv, ragged=ragged, q_heads=q_heads, cache=cache, rotary=rotary,
                    interleaved=rng.random() < 0.3, base=rng.choice([1e4, 5e5, 1e6, 1e7]), lens=lens, **heads)
    nodes = min(_log(rng, 1, 256), kv)
    # whole trees, or the last level of growing ones
    new = nodes if rng.random() < 0.7 else rng.randint(1, nodes)
    # no more products than the largest listed case, counted as the plain form pads them
    most = 8 * 251 * 16384 * 32 * 64
    while seqs * new * kv * q_heads * heads["head_dim"] > most and kv > nodes:
        kv = max(nodes, kv // 2)
    window = _log(rng, 256, 8192) if rng.random() < 0.3 else 0
    return dict(entry=entry, seqs=seqs, nodes=nodes, new=new, kv=kv, ragged=ragged, q_heads=q_heads, cache=cache, window=window,
                lens=lens, **heads)


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------


def _lens(case):
    """(cached tokens with the new ones, nodes of the tree, new tokens) of every sequence: the first has the most of each."""
    rng = random.Random(case["lens"])
    kv, nodes, new = case["kv"], case["nodes"], case["new"]
    kvs, sizes, news = [kv], [nodes], [new]
    for _ in range(case["seqs"] - 1):
        if case["ragged"]:
            kvs.append(_log(rng, max(1, kv // 8), kv))
            news.append(min(kvs[-1], rng.randint(1, new)))
            # a sequence without a tree now and then: a chunk of a prompt
            sizes.append(0 if not nodes or rng.random() < 0.1 else min(kvs[-1], rng.randint(news[-1], nodes)))
        else:
            kvs.append(kv)
            news.append(new)
            sizes.append(nodes)
    return kvs, sizes, news


def _starts(lens):
    total, starts = 0, [0]
    for n in lens:
        total += n
        starts.append(total)
    return starts


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _rows(gen, *shape):
    """BF16 activations ~N(0, 1) whose last axis has a few wide channels, as keys have."""
    x = torch.empty(*shape, device="cuda").normal_(0.0, 1.0, generator=gen)
    x[..., :: max(1, shape[-1] // 4)] *= 4.0
    return x.to(torch.bfloat16)


def _parents(gen, seqs, nodes):
    """Trees as a drafting loop grows them: any node before may be a node's parent, the last ones as likely as the first."""
    u = torch.rand(seqs, max(1, nodes), device="cuda", generator=gen)
    at = torch.arange(max(1, nodes), device="cuda")
    return torch.where(at == 0, -1, (u * at).long().clamp(max=at - 1)).to(torch.int32)


def _cache(gen, state, kvs, spare=5):
    """A cache that a server has been filling: pages in no order, other sequences' tokens in the rest."""
    case = state["case"]
    heads, dim, page, kind = case["kv_heads"], case["head_dim"], case["page"], case["cache"]
    counts = [n // page + 1 for n in kvs]
    pages = sum(counts) + spare
    step = max(1, (1 << 26) // (heads * page * dim))
    for name in ("k", "v"):
        codes, scales = [], []
        for at in range(0, pages, step):
            c, s = _quantise(_rows(gen, min(pages - at, step), heads, page, dim).float(), kind)
            codes.append(c)
            scales.append(s)
        state[name + "_cache"] = torch.cat([c.view(torch.uint8) for c in codes]).view(TYPES[kind])
        state[name + "_scale"] = torch.cat(scales) if kind != "bf16" else None
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    first = torch.tensor(_starts(counts)[:-1]).cuda()
    column = torch.arange(max(counts), device="cuda")
    count = torch.tensor(counts).cuda()
    state["table"] = torch.where(column < count[:, None], order[(first[:, None] + column).clamp(max=pages - 1)], 0)
    state["kv_lens"] = _ints(kvs)
    if own:
        import w4a16

        state["cache"] = w4a16.KvCache(state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"])


def _batch(state, kvs, news):
    state["starts"], state["rows"], state["max_new"], state["max_kv"] = _ints(_starts(news)), sum(news), max(news), max(kvs)
    if own:
        import w4a16

        state["batch"] = w4a16.KvBatch(state["table"], state["kv_lens"], state["starts"], state["rows"],
                                       max_new=state["max_new"], max_kv=state["max_kv"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case=case)
    if case["entry"] == "select":
        shape = (case["groups"], case["beams"], case["vocab"])
        logits = torch.empty(shape, device="cuda").normal_(0.0, 3.0, generator=gen)
        state["logits"] = logits.to(torch.bfloat16) if case["logits"] == "bf16" else logits
        # what beams of a few tokens have come to
        state["scores"] = -10.0 * torch.rand(shape[:2], device="cuda", generator=gen)
        return state
    if case["entry"] == "reorder":
        rng = random.Random(case["lens"])
        groups, beams = case["groups"], case["beams"]
        kvs = [n for g in range(groups) for n in [case["kv"] if g == 0 else _log(rng, max(1, case["kv"] // 8), case["kv"])] * beams]
        _cache(gen, state, kvs)
        # the better beams have more children
        u = torch.rand(groups, beams, device="cuda", generator=gen)
        state["parents"] = (u * u * beams).long().clamp(max=beams - 1).to(torch.int32)
        if own:
            _batch(state, kvs, [1] * len(kvs))
        return state
    if case["entry"] == "verify":
        return _prepare_verify(case, gen, state)
    kvs, sizes, news = _lens(case)
    _cache(gen, state, kvs)
    _batch(state, kvs, news)
    heads, dim = case["kv_heads"], case["head_dim"]
    # queries, keys and values stand side by side in the rows of one fused projection
    fused = _rows(gen, sum(news), case["q_heads"] + 2 * heads, dim)
    state["q"], state["k"], state["v"] = fused.split([case["q_heads"], heads, heads], 1)
    if case["nodes"]:
        state["parents"], state["sizes"] = _parents(gen, case["seqs"], case["nodes"]), _ints(sizes)
        # what a server has made once for all its layers; an append's case makes it anew
        if own:
            import w4a16

            state["tree"] = w4a16.KvTree(state["parents"], state["batch"], sizes=state["sizes"])
        else:
            state["seen"], state["depth"] = _ancestors(state["parents"])
    if case["entry"] == "append":
        half = case["rotary"] // 2
        state["inv_freq"] = (1.0 / case["base"] ** (torch.arange(half, dtype=torch.float64, device="cuda") / half)).float()
        if own:
            import w4a16

            state["rope"] = w4a16.Rope(state["inv_freq"], interleaved=case["interleaved"])
    return state


def _prepare_verify(case, gen, state):
    seqs, nodes, vocab = case["seqs"], case["nodes"], case["vocab"]
    rng = random.Random(case["lens"])
    sizes = [nodes] + [rng.randint(1, nodes) if rng.random() < 0.3 else nodes for _ in range(seqs - 1)]
    kvs = [case["kv"]] + [rng.randint(nodes, case["kv"]) for _ in range(seqs - 1)]
    _cache(gen, state, kvs)
    _batch(state, kvs, sizes)
    target = torch.empty(seqs, nodes, vocab, device="cuda").normal_(0.0, 3.0, generator=gen)
    state["target"] = torch.softmax(target, -1)
    parents = _parents(gen, seqs, nodes)
    # a node's children hold the likeliest words behind it, in their order
    like = state["target"].topk(min(16, vocab), -1).indices
    before = torch.arange(nodes, device="cuda")
    rank = ((parents[:, :, None] == parents[:, None, :]) & (before[:, None] > before)).sum(-1)
    each = torch.arange(seqs, device="cuda")[:, None]
    state["tokens"] = like[each, parents.long().clamp(min=0), rank % like.shape[-1]].to(torch.int32)
    state["parents"], state["sizes"] = parents, _ints(sizes)
    state["uniforms"] = torch.rand(seqs, nodes, device="cuda", generator=gen)
    return state


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attention": _plain_attention, "select": _plain_select, "reorder": _plain_reorder,
            "verify": _plain_verify}[state["case"]["entry"]](state)


def _run_own(state):
    import w4a16

    case = state["case"]
    if case["entry"] == "append":
        tree = state.get("tree")
        if tree is not None:
            tree.update()
        q = state["cache"].append(state["k"], state["v"], state["batch"], state["rope"], q=state["q"],
                                  positions=None if tree is None else tree.positions)
        out = {"q": q} | _buffers(state)
        return out if tree is None else out | {"seen": tree.seen, "positions": tree.positions}
    if case["entry"] == "attention":
        out, lse = w4a16.paged_attention(state["q"], state["cache"], state["batch"], window=case["window"], return_lse=True,
                                         tree=state["tree"])
        return {"out": out, "lse": lse}
    if case["entry"] == "select":
        scores, parents, tokens = w4a16.beam_select(state["logits"], state["scores"], case["take"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    if case["entry"] == "reorder":
        table, source = w4a16.beam_tables(state["table"], state["kv_lens"], state["parents"], case["page"])
        state["cache"].copy_tails(table, state["kv_lens"], source)
        return {"table": table, "source": source} | _buffers(state)
    accepted, path, tokens = w4a16.verify_tree(state["target"], state["tokens"], state["parents"], state["uniforms"],
                                               sizes=state["sizes"])
    state["cache"].keep_path(state["batch"], path)
    return {"accepted": accepted, "path": path, "tokens": tokens} | _buffers(state)


def _buffers(state):
    if state["case"]["cache"] == "int8":  # the values of the call's rows
        if own:
            k, v = state["cache"].read(state["batch"])
            return {"k": k, "v": v}
        seq, at = _places(state)
        index = (state["table"][seq, at // state["case"]["page"]].long(), slice(None), at % state["case"]["page"])
        return {name: _values(state, name, index).to(torch.bfloat16) for name in "kv"}
    out = {"k": state["k_cache"], "v": state["v_cache"]}
    if state["k_scale"] is not None:
        out |= {"k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    return out


def _quantise(x, kind):
    """Codes and scales of rows of FP32 values: one scale a row."""
    if kind == "bf16":
        return x.to(torch.bfloat16), None
    most = x.abs().amax(-1)
    held = most >= SMALL
    scale = torch.where(held, most / TOP[kind], 0.0)
    scaled = x * torch.where(held, TOP[kind] / most, 0.0)[..., None]
    scaled = scaled.clamp(-TOP[kind], TOP[kind])
    return (scaled.round() if kind == "int8" else scaled).to(TYPES[kind]), scale


def _places(state):
    """(sequence, place in its cache) of every row: a sequence's rows are its last tokens."""
    starts = state["starts"]
    row = torch.arange(state["rows"], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row.to(torch.int32), right=True)
    new = (starts[1:] - starts[:-1])[seq]
    return seq, (state["kv_lens"][seq] - new + row - starts[seq]).long()


def _values(state, name, index):
    """The FP32 values of the cache at an index of its pages (and of their tokens)."""
    values = state[name + "_cache"][index] if state["case"]["cache"] == "bf16" else \
        state[name + "_cache"].view(torch.uint8)[index].view(TYPES[state["case"]["cache"]])
    return values.float() if state[name + "_scale"] is None else values.float() * state[name + "_scale"][index][..., None]


def _ancestors(parents):
    """(which nodes [seqs, node, other] are a node itself or above it, links up to the root [seqs, node])."""
    seqs, nodes = parents.shape
    above = torch.zeros(seqs, nodes, nodes + 1, device="cuda")
    above.scatter_(-1, torch.where(parents < 0, nodes, parents).long()[..., None], 1.0)
    seen = above[..., :nodes] + torch.eye(nodes, device="cuda")
    for _ in range((nodes - 1).bit_length()):  # paths of twice the length
        seen = (torch.matmul(seen, seen) > 0).float()
    return seen > 0, seen.sum(-1).int() - 1


def _plain_tree(state):
    """(bits of the nodes that a row sees [rows, words], position of every row)."""
    seen, depth = _ancestors(state["parents"])
    nodes = state["case"]["nodes"]
    seq, at = _places(state)
    base = (state["kv_lens"] - state["sizes"])[seq]
    node = (at - base).clamp(min=0)
    words = -(-nodes // 64)
    bits = torch.zeros(seq.numel(), 64 * words, dtype=torch.bool, device="cuda")
    bits[:, :nodes] = seen[seq, node]
    bits &= (at >= base)[:, None]
    packed = (bits.view(-1, words, 64).long() << torch.arange(64, device="cuda")).sum(-1)
    return packed, torch.where(at >= base, base + depth[seq, node], at).int()


def _turned(x, state, position):
    """Rows of heads in FP32, the first values of each head turned by their position's angles."""
    rotary, half = state["case"]["rotary"], state["case"]["rotary"] // 2
    angle = position.double()[:, None, None] * state["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    x = x.float()
    if state["case"]["interleaved"]:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        first = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rotary]
        first = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((first, x[..., rotary:]), -1)


def _plain_append(state):
    case, page, more = state["case"], state["case"]["page"], {}
    seq, at = _places(state)
    position = at
    if case["nodes"]:
        more["seen"], position = _plain_tree(state)
        more["positions"] = position
    pages = state["table"][seq, at // page].long()
    for name in ("k", "v"):
        x = _turned(state["k"], state, position) if name == "k" else state["v"].float()
        codes, scale = _quantise(x, case["cache"])
        if scale is None:
            state[name + "_cache"][pages, :, at % page] = codes
        else:
            state[name + "_cache"].view(torch.uint8)[pages, :, at % page] = codes.view(torch.uint8)
            state[name + "_scale"][pages, :, at % page] = scale
    return {"q": _turned(state["q"], state, position).to(torch.bfloat16)} | _buffers(state) | more


def _plain_attention(state):
    case = state["case"]
    heads, group, dim = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["head_dim"]
    seqs, kv, new, nodes = case["seqs"], state["max_kv"], state["max_new"], case["nodes"]
    # the pages of every sequence in order, as [sequence, head, token, value]
    table = state["table"].long()
    k, v = (_values(state, name, (table,)).permute(0, 2, 1, 3, 4).reshape(seqs, heads, -1, dim)[:, :, :kv].contiguous() for name in "kv")
    starts, lens = state["starts"].long(), state["kv_lens"].long()
    news, base = starts[1:] - starts[:-1], lens - state["sizes"].long()
    step = torch.arange(new, device="cuda")
    rows = (starts[:-1, None] + step).clamp(max=state["rows"] - 1)
    q = state["q"][rows].float().reshape(seqs, new, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, heads, -1, dim)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(dim**-0.5).view(seqs, heads, group, new, kv)
    # a row sees what stands before the tree, and of the tree itself and its ancestors
    place = (lens - news)[:, None] + step
    each = torch.arange(seqs, device="cuda")[:, None]
    node = (place - base[:, None]).clamp(0, nodes - 1)
    position = torch.where(place >= base[:, None], base[:, None] + state["depth"][each, node], place)
    token = torch.arange(kv, device="cuda")
    other = token - base[:, None]
    of_tree = state["seen"][each[..., None], node[..., None], other.clamp(0, nodes - 1)[:, None]]
    before = other[:, None] < 0
    if case["window"]:
        before = before & (token > position[..., None] - case["window"])
    seen = (token <= place[..., None]) & (before | ((other >= 0)[:, None] & of_tree))
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)  # padding may see nothing
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


def _plain_select(state):
    logits, scores, take = state["logits"], state["scores"], state["case"]["take"]
    groups, beams, vocab = logits.shape
    # in 64 bits: candidates of two beams may be as near as their sums are exact
    x = logits.double()
    most = x.amax(-1, keepdim=True)
    every = (scores.double()[..., None] + (x - most - (x - most).exp().sum(-1, keepdim=True).log())).view(groups, -1)
    last = every.topk(take, -1).values[:, -1:]
    # the lowest of those that are equal to the last one
    above, equal = every > last, every == last
    room = take - above.sum(-1, keepdim=True)
    chosen = above | (equal & (equal.cumsum(-1) <= room))
    index = torch.arange(beams * vocab, device="cuda", dtype=torch.float64)
    at = -torch.where(chosen, -index, -math.inf).topk(take, -1).values  # in their order
    got = every.gather(-1, at.long())
    got, order = got.sort(dim=-1, descending=True, stable=True)
    at = at.gather(-1, order).long()
    return {"scores": got.float(), "parents": (at // vocab).int(), "tokens": (at % vocab).int()}


def _plain_reorder(state):
    case, parents, table = state["case"], state["parents"].long(), state["table"]
    groups, beams = parents.shape
    page, lens = case["page"], state["kv_lens"].view(groups, beams)
    each = torch.arange(beams, device="cuda")
    same = parents[:, :, None] == parents[:, None, :]
    keeper = torch.where(same, each, beams).amin(-1)  # the first child of a beam's parent
    keeps = keeper == each
    # the beams without children, in order: the others take their last pages
    dead = ~(parents[:, None, :] == each[:, None]).any(-1)
    gone = (~dead).int().sort(dim=-1, stable=True).indices
    nth = ((~keeps).long().cumsum(-1) - 1).clamp(min=0)
    private = torch.where(keeps, parents, gone.gather(-1, nth))
    full = lens[:, :1] // page
    column = torch.arange(table.shape[1], device="cuda")
    row = torch.where(column < full[..., None], parents[..., None], private[..., None])
    tables = table.view(groups, beams, -1)
    new = tables.gather(1, row)
    first = beams * torch.arange(groups, device="cuda")[:, None]
    source = torch.where(keeps, -1, keeper + first).int().view(-1)
    # the tokens of the pages that are not full
    new = new.view(groups * beams, -1)
    tail = (lens // page).view(-1).long()
    mine = torch.arange(groups * beams, device="cuda")
    to, of = new[mine, tail].long(), torch.where(source < 0, mine, source.long())
    held = torch.arange(page, device="cuda") < (lens.reshape(-1, 1) % page)
    come = new[of, tail].long()
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        if state[name] is not None:
            x = state[name] if state[name].dtype != torch.float8_e4m3fn else state[name].view(torch.uint8)
            where = held[:, None, :].view(held.shape[0], 1, page, *([1] * (x.dim() - 3)))
            x[to] = torch.where(where, x[come], x[to])
    return {"table": new, "source": source} | _buffers(state)


def _plain_verify(state):
    target, tokens, parents, u = (state[n] for n in ("target", "tokens", "parents", "uniforms"))
    seqs, nodes, vocab = target.shape
    each, at = torch.arange(seqs, device="cuda"), torch.arange(nodes, device="cuda")
    real = at < state["sizes"][:, None]
    # a child that comes after its siblings is asked when they were refused; a word that was refused has no weight left
    sibling = (parents[:, :, None] == parents[:, None, :]) & (at[:, None] > at) & real[:, None, :]
    again = (sibling & (tokens[:, :, None] == tokens[:, None, :])).any(-1)
    p = target[each[:, None], parents.long().clamp(min=0), tokens.long()].double()
    p = torch.where(again | ~real | (at == 0), 0.0, p)
    left = (1.0 - (sibling * p[:, None, :]).sum(-1)).clamp(min=0.0)
    taken = u.double() * left < p
    taken &= ~(sibling & taken[:, None, :]).any(-1)
    taken[:, 0] = True
    seen, depth = _ancestors(parents)
    on = (~seen | taken[:, None, :]).all(-1)
    accepted = on.sum(-1).int() - 1
    path = torch.where(on, at, nodes).sort(-1).values
    path = torch.where(path == nodes, -1, path).int()
    end = path.long().gather(-1, accepted.long()[:, None])
    # behind the last taken node: its row without its children
    row = target[each, end[:, 0]]
    child = (parents == end) & real & (at > 0)
    taken_off = torch.zeros_like(row).scatter_add_(-1, tokens.long(), child.float()) > 0
    rest = torch.where(taken_off, 0.0, row)
    rest = torch.where((rest.sum(-1) > 0)[:, None], rest, row)
    sums = rest.double().cumsum(-1)
    drawn = (sums <= u[:, :1].double() * sums[:, -1:]).sum(-1).clamp(max=vocab - 1).int()
    follow = tokens.gather(-1, torch.cat([path[:, 1:], path[:, :1]], 1).long().clamp(min=0))
    out = torch.where(at < accepted[:, None], follow, torch.where(at == accepted[:, None], drawn[:, None], -1))
    _plain_keep(state, path)
    return {"accepted": accepted, "path": path, "tokens": out} | _buffers(state)


def _plain_keep(state, path):
    """The path's tokens take the first places of the tree."""
    page = state["case"]["page"]
    base = (state["kv_lens"] - state["sizes"]).long()[:, None]
    each, at = torch.arange(path.shape[0], device="cuda")[:, None], torch.arange(path.shape[1], device="cuda")
    come = torch.where(path < 0, at, path.long()) + base
    to = at + base
    # places behind the sequence: one of its own instead, onto itself
    inside = to < state["kv_lens"][:, None]
    to, come = torch.where(inside, to, base), torch.where(inside, come, base)
    to_page, come_page = state["table"][each, to // page].long(), state["table"][each, come // page].long()
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        if state[name] is not None:
            x = state[name] if state[name].dtype != torch.float8_e4m3fn else state[name].view(torch.uint8)
            x[to_page, :, to % page] = x[come_page, :, come % page]


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------------


def work(case):
    if case["entry"] == "select":
        values = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": values * (2 if case["logits"] == "bf16" else 4) + 4 * case["groups"] * (case["beams"] + 3 * case["take"]),
                "flops": 3 * values}
    heads, dim = case["kv_heads"], case["head_dim"]
    token = 2 * heads * (dim * 2 if case["cache"] == "bf16" else dim + 4)  # K and V of one cached token
    if case["entry"] == "reorder":
        seqs = case["groups"] * case["beams"]
        # both tables; half of the beams are copied, of half a page
        return {"bytes": 8 * seqs * (case["kv"] // (2 * case["page"]) + 1) + seqs // 2 * case["page"] // 2 * token * 2, "flops": seqs}
    if case["entry"] == "verify":
        # a row of each sequence, the gathers, a few tokens of the path
        return {"bytes": case["seqs"] * (4 * case["vocab"] + 20 * case["nodes"] + 4 * token), "flops": 2 * case["seqs"] * case["vocab"]}
    kvs, sizes, news = _lens(case)
    plain = 2 * dim * sum(news)  # a head's rows in BF16
    if case["entry"] == "append":
        held = sum(news) * token * (2 if case["cache"] == "int8" else 1)  # INT8: and read back
        back = 2 * heads * plain if case["cache"] == "int8" else 0
        return {"bytes": held + back + plain * (2 * heads + 2 * case["q_heads"]) + 8 * sum(news),
                "flops": 3 * sum(news) * (heads + case["q_heads"]) * case["rotary"]}
    pairs = touched = 0
    for n, size, m in zip(kvs, sizes, news):
        old = n - max(size, m)
        if case["window"]:
            old = min(old, case["window"])
        pairs += m * (old + min(m, 6))  # a node's ancestors are few
        touched += old + max(size, m)
    q = sum(news) * case["q_heads"]
    return {"bytes": touched * token + q * (4 * dim + 4), "flops": 4 * pairs * case["q_heads"] * dim}


# ------------------------------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["entry"] == "select":
        return _exact_select(state)
    if case["entry"] == "append":
        return _exact_append(state)
    if case["entry"] == "attention":
        return _exact_attention(state)
    return None  # whole numbers, and values that are only moved


def _exact_select(state):
    out = []
    for logits, scores in zip(state["logits"], state["scores"]):
        every = torch.cat([s.double() + torch.log_softmax(row.double(), -1) for row, s in zip(logits, scores)])
        out.append(every.sort(descending=True).values[:state["case"]["take"]])
    return {"scores": torch.stack(out), "parents": None, "tokens": None}


def _links(parents):
    """Of every node the nodes from itself up to the root."""
    ways = []
    for i, p in enumerate(parents):
        ways.append([i] + (ways[p] if p >= 0 else []))
    return ways


def _exact_append(state):
    case = state["case"]
    kvs, sizes, news = _lens(case)
    position, places = [], []
    parents = state["parents"].tolist() if case["nodes"] else None
    table = state["table"].cpu()
    for s, (n, size, m) in enumerate(zip(kvs, sizes, news)):
        depth = [len(w) - 1 for w in _links(parents[s])] if size else []
        for at in range(n - m, n):
            node = at - (n - size)
            position.append(at if node < 0 else n - size + depth[node])
            places.append((int(table[s, at // case["page"]]), at % case["page"]))
    angle = torch.tensor(position, dtype=torch.float64).cuda()[:, None, None] * state["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)

    def turned(x):
        x = x.double()
        first, rest = x[..., :case["rotary"]], x[..., case["rotary"]:]
        if case["interleaved"]:
            z = torch.view_as_real(torch.view_as_complex(first.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
        else:
            z = torch.complex(*first.chunk(2, -1)) * turn
            z = torch.cat((z.real, z.imag), -1)
        return torch.cat((z, rest), -1)

    pages, inside = torch.tensor(places).cuda().unbind(1)
    out = {"q": turned(state["q"])}
    for name, x in (("k", turned(state["k"])), ("v", state["v"].double())):
        most = x.abs().amax(-1)
        if case["cache"] == "int8":  # read back
            out[name] = (x * 127 / most[..., None]).round() * (most[..., None] / 127)
            continue
        held = state[name + "_cache"]
        held = held.double() if case["cache"] == "bf16" else held.view(torch.uint8).view(TYPES[case["cache"]]).float().double()
        if case["cache"] == "fp8":  # three bits behind the leading one, subnormals under 2^-6
            scale = state[name + "_scale"].double()
            scale[pages, :, inside] = most / 448
            out[name + "_scale"] = scale
            x = x * 448 / most[..., None]
            unit = torch.exp2((torch.frexp(x)[1] - 1).clamp(min=-6).double() - 3)
            x = (x / unit).round() * unit
        held[pages, :, inside] = x
        out[name] = held
    return out | ({"seen": None, "positions": None} if case["nodes"] else {})


def _exact_attention(state):
    case = state["case"]
    kvs, sizes, news = _lens(case)
    group, dim, page = case["q_heads"] // case["kv_heads"], case["head_dim"], case["page"]
    outs, lses, first = [], [], 0
    table, parents = state["table"].long(), state["parents"].tolist()
    for s, (n, size, m) in enumerate(zip(kvs, sizes, news)):
        pages = table[s, :-(-n // page)]
        whole = {}
        for name in "kv":
            x = state[name + "_cache"].view(torch.uint8 if case["cache"] != "bf16" else torch.bfloat16)[pages]
            x = x.view(TYPES[case["cache"]]).float().double()
            if state[name + "_scale"] is not None:
                x = x * state[name + "_scale"][pages].double()[..., None]
            whole[name] = x.transpose(0, 1).reshape(case["kv_heads"], -1, dim)[:, :n]
        base = n - size
        hidden = torch.zeros(m, n, dtype=torch.bool)
        ways = _links(parents[s])
        for i, at in enumerate(range(n - m, n)):
            if at < base:
                position = at
                hidden[i, at + 1:] = True
            else:
                way = ways[at - base]
                position = base + len(way) - 1
                hidden[i, base:] = True
                hidden[i, [base + w for w in way]] = False
            if case["window"]:
                hidden[i, :max(0, min(base, position - case["window"] + 1))] = True
        hidden = hidden.cuda()
        out = torch.empty(m, case["q_heads"], dim, dtype=torch.float64, device="cuda")
        lse = torch.empty(m, case["q_heads"], dtype=torch.float64, device="cuda")
        for h in range(case["q_heads"]):
            x = state["q"][first:first + m, h].double() @ whole["k"][h // group].T / math.sqrt(dim)
            x.masked_fill_(hidden, -math.inf)
            lse[:, h] = torch.logsumexp(x, -1)
            out[:, h] = (x - lse[:, h:h + 1]).exp() @ whole["v"][h // group]
        outs.append(out)
        lses.append(lse)
        first += m
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
