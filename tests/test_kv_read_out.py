"""What KvCache.read takes as `out` on the GPU: a pair of contiguous BF16 tensors (or their bits) of the rows' shape, nothing else."""

import pytest
import torch

import w4a16
from test_kv_cache import filled, make_batch

pytestmark = pytest.mark.gpu


def test_out(cuda):
    rows, heads, dim = 3, 2, 64
    cache = filled(8, 16, heads, dim, "int8", cuda, seed=1)
    batch, _ = make_batch([20], [rows], 16, 8, cuda)
    want = cache.read(batch)
    good = torch.zeros(rows, heads, dim, dtype=torch.bfloat16, device=cuda)
    bad = [good.half(), good.float(), good.cpu(), good.view(rows, heads * dim), good.view(heads, rows, dim),
           torch.zeros(rows + 1, heads, dim, dtype=torch.bfloat16, device=cuda),
           torch.zeros(rows, heads + 1, dim, dtype=torch.bfloat16, device=cuda)[:, :heads],
           torch.zeros(heads, rows, dim, dtype=torch.bfloat16, device=cuda).transpose(0, 1), None]
    for b in bad:
        before = None if b is None else b.clone()
        for out in ((b, torch.empty_like(good)), (torch.empty_like(good), b)):
            with pytest.raises(w4a16.W4A16Error):
                cache.read(batch, out=out)
        assert b is None or torch.equal(b, before)
    for dtype in (torch.bfloat16, torch.int16, torch.uint16):
        out = tuple(torch.zeros(rows, heads, dim, dtype=dtype, device=cuda) for _ in range(2))
        assert cache.read(batch, out=out) is out
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(out, want))
