"""Attention of batches whose sequences have more rows than their trees, or no tree, under a window that is shorter than the rows: each tile of
rows begins at its own window. On the GPU against FP64, by either kernel, cut and whole."""

import pytest
import torch

from test_tree_attention_paths import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv_lens,news,nodes,q_heads,heads,window,hints", [
    ([700, 450], [300, 200], 40, 2, 1, 100, {}),                        # narrow tiles, one after another
    ([1500, 900, 41], [700, 520, 41], 40, 4, 2, 100, {}),               # wide ones
    ([1500, 900, 41], [700, 520, 41], 40, 4, 2, 97, {"max_kv": 1 << 20}),
    ([5000], [600], 8, 2, 1, 260, {"max_kv": 1 << 20}),                 # cut into parts, most of them behind no row's window
])
def test_against_fp64(cuda, kv_lens, news, nodes, q_heads, heads, dim, window, hints, fmt):
    print(f"windows {fmt} lens={kv_lens} news={news} dim={dim} window={window} {hints}", flush=True)
    check(cuda, kv_lens, news, nodes, q_heads, heads, dim, 32, fmt, window=window, **hints)
