"""Tables and links whose rows are 2^32 entries and more apart, on the GPU: the library's strides are C integers, and what does not fit is refused
before it is cut off."""

import pytest
import torch

import w4a16
from test_kv_cache import filled

pytestmark = pytest.mark.gpu


def test_refused(cuda):
    far = torch.zeros((1 << 32) + 64, dtype=torch.int32, device=cuda).as_strided((2, 4), ((1 << 32) + 8, 1))
    near, lens = torch.zeros(2, 4, dtype=torch.int32, device=cuda), torch.full((2,), 5, dtype=torch.int32, device=cuda)
    starts, parents = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda), torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    cache = filled(4, 8, 1, 64, "bf16", cuda, seed=1)
    batch = w4a16.KvBatch(near, lens, starts, 2)
    for call in (lambda: w4a16.KvBatch(far, lens, starts, 2), lambda: w4a16.KvTree(far, batch),
                 lambda: w4a16.beam_tables(far, lens, parents, 8), lambda: w4a16.beam_tables(near, lens, parents, 8, out=far),
                 lambda: cache.copy_tails(far, lens, lens)):
        with pytest.raises(w4a16.W4A16Error):
            call()
    # a single row has no stride
    one = far[:1]
    w4a16.KvTree(one, w4a16.KvBatch(one, lens[:1], starts[:2], 1))
    table, source = w4a16.beam_tables(one, lens[:1], parents[:, :1].contiguous(), 8)
    assert torch.equal(table, near[:1]) and source.tolist() == [-1]
    cache.copy_tails(one, lens[:1], lens[:1])
    torch.cuda.synchronize()
