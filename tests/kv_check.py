"""Attention's outputs against FP64, each cache format with the bounds of its own roundings (kv_oracle.py)."""

import torch

import kv_oracle
from test_kv_cache import held
from test_paged_attention import whole


def sizes(cache, table, kv_lens, page, pages):
    """Of an 8-bit cache's sequences the sizes of their V codes and scales; None of a BF16 one."""
    codes, scales = held(cache, "v")
    if scales is None:
        return None
    out = []
    for row, n in zip(table, kv_lens):
        token = torch.arange(min(n, len(row) * page))
        at = torch.tensor(row, dtype=torch.long)[token // page]
        at = torch.where((at >= 0) & (at < pages), at, 0)
        out.append((codes.float().double().abs()[at, :, token % page].transpose(0, 1),
                    scales.double().abs()[at, :, token % page].transpose(0, 1)))
    return out


def check(out, lse, cache, table, q, kv_lens, news, page, pages, scale, causal=True, window=0, half=None):
    k, v, there = whole(cache, table, kv_lens, page, pages)
    coded = sizes(cache, table, kv_lens, page, pages)
    want, want_lse, off, lse_off = kv_oracle.attention(q, k, v, there, scale, causal, window, news, kv_lens, coded, half)
    got, got_lse = out.cpu().double(), lse.cpu().double()
    empty = want_lse == float("-inf")
    assert torch.equal(got_lse == float("-inf"), empty)
    assert (got[empty] == 0).all()
    far = ((got - want).abs() / off.clamp(min=1e-300))[~empty]
    lse_far = ((got_lse - want_lse).abs() / lse_off.clamp(min=1e-300))[~empty]
    if far.numel():
        print(f"  of what the roundings allow: out {far.max():.3f}, lse {lse_far.max():.3f}", flush=True)
        assert far.max() <= 1 and lse_far.max() <= 1
