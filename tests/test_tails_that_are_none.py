"""copy_tails where a page is none, on the GPU: a copy lacks its source, its destination or both, and everything stays as it was but for the
one that lacks neither."""

import pytest
import torch

from test_kv_cache import filled, held

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("source,copies", [
    ([5, 9, -7, 1 << 30, 4, 0], []),      # a page outside the cache at either end; no sequence; itself
    ([5, 2, -1, 1, 0, 3], [(13, 22)]),    # page 13 takes from page 22, and no other copy has both
    ([-1, -1, 1, 4, 3, 2], [(22, 13)]),
])
def test_what_is_copied(cuda, source, copies, fmt):
    pages, page, length = 30, 8, 20  # the last pages: 4, 13 and 22, and 31, 40 and 49, which are outside
    cache = filled(pages, page, 2, 64, fmt, cuda, seed=1)
    before = {name: held(cache, name) for name in "kv"}
    wide = torch.arange(6 * 9, dtype=torch.int32, device=cuda).reshape(6, 9)
    cache.copy_tails(wide[:, 2:7], torch.full((6,), length, dtype=torch.int32, device=cuda),
                     torch.tensor(source, dtype=torch.int32, device=cuda))
    for name in "kv":
        for was, now in zip(before[name], held(cache, name)):
            if was is None:
                continue
            want = was.clone().view(torch.uint8).reshape(*was.shape[:3], -1)
            for to, of in copies:
                want[to, :, :length % page] = want[of, :, :length % page]
            assert torch.equal(now.view(torch.uint8).reshape(want.shape), want)
