"""The scales that a KvCache takes on the GPU: FP32 [pages, kv_heads, page_size], as its codes are laid out."""

import pytest
import torch

import w4a16

pytestmark = pytest.mark.gpu


def test_shapes(cuda):
    codes = torch.zeros(4, 2, 16, 64, dtype=torch.int8, device=cuda)
    good = torch.ones(4, 2, 16, device=cuda)
    for bad in (good.view(4, 16, 2), good.flatten(), good[..., None], torch.ones(5, 2, 16, device=cuda), good.half(), good.cpu(),
                torch.ones(4, 2, 17, device=cuda)[..., :16], None):
        for scales in ((bad, good), (good, bad)):
            with pytest.raises(w4a16.W4A16Error):
                w4a16.KvCache(codes, codes.clone(), *scales)
    w4a16.KvCache(codes, codes.clone(), good, good.clone())
