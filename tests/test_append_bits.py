"""What an append does not turn stays bit for bit what it was, on the GPU: values, and keys and queries behind the turned ones, signalling
NaN and signs of zeros among them."""

import pytest
import torch

import w4a16
from test_kv_cache import filled, make_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(64, 8), (64, 64), (128, 40), (256, 128)])
def test_every_pattern(cuda, dim, rotary, interleaved):
    rows = 65536 // dim
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(rows, 1, dim).to(cuda)
    batch, table = make_batch([rows], [rows], 32, -(-rows // 32) + 2, cuda)
    cache = filled(-(-rows // 32) + 2, 32, 1, dim, "bf16", cuda, seed=1)
    x = every.view(torch.bfloat16)
    got = cache.append(x, x, batch, w4a16.Rope.of(rotary, interleaved=interleaved, device=cuda), q=x)
    pages = torch.tensor(table[0], device=cuda)
    k, v = (t.view(torch.int16)[pages, 0].reshape(-1, dim)[:rows] for t in (cache.k, cache.v))
    assert torch.equal(v, every[:, 0])
    assert torch.equal(k[:, rotary:], every[:, 0, rotary:])
    assert torch.equal(got.view(torch.int16)[:, 0, rotary:], every[:, 0, rotary:])
