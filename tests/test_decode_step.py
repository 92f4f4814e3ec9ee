"""A layer's verify step over a store of INT4 operands, on the GPU: the norm, the INT4 projections, the paged cache, the attention over
it, the store's FFN with its residuals, the vocabulary's probabilities, the drafted tokens' verification and the lengths cut back to
what was taken. Eager against the oracles, operator by operator, and the whole step in one graph against the eager one."""

import numpy as np
import pytest
import torch

import convert
import kv_check
import kv_oracle
import w4a16
from conftest import assert_parity
from oracle import oracle
from test_gpu_parity import from_dev, to_dev

pytestmark = pytest.mark.gpu

H, I, Q_HEADS, KV_HEADS, DIM, VOCAB = 512, 1024, 8, 2, 64, 1000
SEQS, DRAFTED, PAGE, COUNT = 2, 3, 8, 10
ROWS = SEQS * (DRAFTED + 1)


@pytest.fixture(scope="module")
def layer(tmp_path_factory):
    """A converted layer's directory and its artifact, and the other projections'."""
    out = str(tmp_path_factory.mktemp("int4_layer"))
    weights = {"mlpGate": oracle.synth_weight(I, H, 1), "mlpUp": oracle.synth_weight(I, H, 2), "mlpDown": oracle.synth_weight(H, I, 3)}
    convert.write_sidecar(out, {0: weights}, "/tmp/synthetic")
    gate, up, down = (oracle.quantize(weights[name]) for name in ("mlpGate", "mlpUp", "mlpDown"))
    ffn = (np.concatenate([gate[0], up[0]]), np.concatenate([gate[1], up[1]]), *down)
    shapes = {"qkv": ((Q_HEADS + 2 * KV_HEADS) * DIM, H), "out": (H, Q_HEADS * DIM), "vocab": (VOCAB, H)}
    return out, ffn, {name: (*oracle.quantize(oracle.synth_weight(n, k, 4 + i)), n, k) for i, (name, (n, k)) in enumerate(shapes.items())}


class Step:
    """What a server holds, and one step over it."""

    def __init__(self, engine, weights, norms, fmt, cuda):
        self.engine, self.weights, self.norms = engine, weights, norms
        pages = SEQS * COUNT + 3
        self.cache = w4a16.KvCache.empty(pages, PAGE, KV_HEADS, DIM, fmt, device=cuda)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:SEQS * COUNT].reshape(SEQS, COUNT)
        self.table = order.tolist()
        self.kv_lens = torch.zeros(SEQS, dtype=torch.int32, device=cuda)
        starts = torch.arange(SEQS + 1, dtype=torch.int32, device=cuda) * (DRAFTED + 1)
        self.batch = w4a16.KvBatch(order.to(torch.int32).to(cuda), self.kv_lens, starts, ROWS, max_new=DRAFTED + 1, max_kv=PAGE * COUNT)
        self.hidden = torch.zeros(ROWS, H, dtype=torch.bfloat16, device=cuda)
        self.residual = torch.zeros_like(self.hidden)
        self.drafted = torch.zeros(SEQS, DRAFTED, dtype=torch.int32, device=cuda)
        self.uniforms = torch.zeros(SEQS, DRAFTED + 1, device=cuda)

    def run(self):
        self.kv_lens += DRAFTED + 1
        self.residual.copy_(self.hidden)
        normed = w4a16.rmsnorm(self.residual, self.norms[0], 1, 1e-6)
        qkv = w4a16.gemm_int4_bf16(normed, self.weights["qkv"]).view(ROWS, -1, DIM)
        q, k, v = qkv.split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
        self.cache.write(k, v, self.batch)
        attended, lse = w4a16.paged_attention(q, self.cache, self.batch, return_lse=True)
        sublayer = w4a16.gemm_int4_bf16(attended.view(ROWS, -1), self.weights["out"])
        out = self.engine.forward_residual_norm(0, self.residual, sublayer, self.norms[1], 1, 1e-6)
        target = torch.softmax(w4a16.gemm_int4_bf16(self.residual, self.weights["vocab"]).float(), -1).view(SEQS, DRAFTED + 1, VOCAB)
        accepted, tokens = w4a16.verify_drafts(target, self.drafted, self.uniforms)
        self.kv_lens -= DRAFTED - accepted  # the token at the end stays
        return dict(qkv=qkv, attended=attended, lse=lse, sublayer=sublayer, out=out, target=target, accepted=accepted, tokens=tokens)


def inputs(step, n):
    gen = torch.Generator().manual_seed(n)
    step.hidden.copy_(torch.randn(ROWS, H, generator=gen))
    step.drafted.copy_(torch.randint(0, VOCAB, (SEQS, DRAFTED), generator=gen))
    u = torch.rand(SEQS, DRAFTED + 1, generator=gen)
    u[:, :DRAFTED] *= torch.rand(SEQS, DRAFTED, generator=gen) < 0.4  # most are taken
    step.uniforms.copy_(u)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
def test_step(cuda, layer, fmt):
    where, ffn, others = layer
    engine = w4a16.Engine(1, H, I, max_tokens=ROWS, int4_max_rows=ROWS)
    assert engine.load_quantized_ffn(where) == 0, engine.last_error()
    assert engine.routes_int4(0, ROWS, verify_rows=True)
    weights = {name: w4a16.TiledWeight.from_artifact(*w, device=cuda) for name, w in others.items()}
    norms = [oracle.bf16_bits(np.random.default_rng(s).normal(1.0, 0.2, H).astype(np.float32)) for s in (1, 2)]
    dev_norms = [to_dev(n, cuda) for n in norms]
    eager, captured = (Step(engine, weights, dev_norms, fmt, cuda) for _ in range(2))
    # once before the capture, over lengths that the steps then begin with
    inputs(captured, 99)
    captured.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = captured.run()
    captured.kv_lens.zero_()
    lens = [0, 0]
    for n in range(6):
        print(f"decode step {fmt} {n} lens={lens}", flush=True)
        for step in (eager, captured):
            inputs(step, n)
        got = eager.run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name, t in got.items():
            assert torch.equal(t, replayed[name]), name
        assert torch.equal(eager.residual, captured.residual) and torch.equal(eager.kv_lens, captured.kv_lens)
        assert all(torch.equal(a, b) for a, b in zip(eager.cache.read(eager.batch), captured.cache.read(captured.batch)))
        # the oracles, each on what the operator was given
        lens = [m + DRAFTED + 1 for m in lens]
        q, k, v = got["qkv"].cpu().split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
        for name, x in (("k", k), ("v", v)):
            codes, scales = kv_oracle.quantise(x.contiguous(), fmt)
            held, held_scales = getattr(eager.cache, name).cpu(), getattr(eager.cache, name + "_scale")
            places = kv_oracle.places(eager.table, lens, [DRAFTED + 1] * SEQS, PAGE, eager.cache.num_pages)
            for i, (_, at, inside) in enumerate(places):
                assert torch.equal(held[at, :, inside].view(torch.uint8), codes[i].view(torch.uint8))
                assert scales is None or torch.equal(held_scales.cpu()[at, :, inside], scales[i])
        kv_check.check(got["attended"], got["lse"], eager.cache, eager.table, q, lens, [DRAFTED + 1] * SEQS, PAGE, eager.cache.num_pages,
                       DIM**-0.5)
        bits = {name: from_dev(got[name].view(torch.int16)) for name in ("attended", "sublayer", "out")}
        hidden = from_dev(eager.hidden.view(torch.int16))
        p, s, rows, cols = others["out"]
        assert_parity(bits["sublayer"], oracle.gemm_bf16(bits["attended"].reshape(ROWS, -1), p, s, rows, cols), "output projection")
        mid, normed = oracle.residual_norm_bf16(hidden, bits["sublayer"], norms[1], 1, 1e-6)
        want, _, _ = oracle.ffn_bf16(normed, *ffn, H, I)
        assert_parity(bits["out"], want, "FFN", floor_div=16.0)
        assert_parity(from_dev(eager.residual.view(torch.int16)), oracle.residual_add_bf16(mid, want), "residual", floor_div=16.0)
        some, all_tokens = kv_oracle.verify(got["target"].cpu().numpy(), None, eager.drafted.cpu().numpy(), None, eager.uniforms.cpu().numpy())
        assert got["accepted"].tolist() == some.tolist() and got["tokens"].tolist() == all_tokens.tolist()
        lens = [m - DRAFTED + int(a) for m, a in zip(lens, some)]
        assert eager.kv_lens.tolist() == lens
    assert len(set(lens)) > 1 or lens[0] < 6 * (DRAFTED + 1)  # not everything was taken
    engine.close()
